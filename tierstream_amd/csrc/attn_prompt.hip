// Attention over packed sequences and its gradients, a wave a row: the running maximum and sum of its softmax, a key at a time.
#include "attn_device.hpp"

namespace tsa {
namespace op {
namespace {

template <class T>
struct Row {
  float v[2];
  __device__ __forceinline__ Row(const tsa_heads& h, uint64_t t, uint32_t head, uint32_t dim) {
    const u16* p = row_of<u16>(h, t, head);
    for (int k = 0; k < 2; ++k) v[k] = threadIdx.x + 64 * k < dim ? T::up(p[threadIdx.x + 64 * k]) : 0.0f;
  }
  __device__ __forceinline__ float dot(const Row& o) const { return lanes_sum(v[0] * o.v[0] + v[1] * o.v[1]); }
};
template <class T>
__device__ __forceinline__ void put(const tsa_heads& h, uint64_t t, uint32_t head, uint32_t dim, const float (&v)[2], float by) {
  u16* p = const_cast<u16*>(row_of<u16>(h, t, head));
  for (int k = 0; k < 2; ++k)
    if (threadIdx.x + 64 * k < dim) p[threadIdx.x + 64 * k] = T::down(v[k] * by);
}

template <class T>
__global__ __launch_bounds__(64) void attend_kernel(tsa_attend_args a) {
  const uint32_t r = blockIdx.x, h = blockIdx.y, kept = h / (a.q.heads / a.k.heads);
  const uint32_t i = sequence_of(a.first, a.sequences, r);
  if (i >= a.sequences) return;
  const Span q = span_of(a.first, i, a.tokens), k = span_of(a.k_first ? a.k_first : a.first, i, a.k_tokens);
  if (r < q.begin || r >= q.begin + q.count) return;
  const int64_t keys = a.causal ? int64_t(k.count) - q.count + (r - q.begin) + 1 : k.count;
  const Row<T> x(a.q, r, h, a.head_dim);
  float o[2] = {0, 0}, top = -INFINITY, sum = 0;
  for (int64_t j = 0; j < keys; ++j) {
    const float score = x.dot(Row<T>(a.k, k.begin + j, kept, a.head_dim)) * a.scale;
    const Row<T> v(a.v, k.begin + j, kept, a.head_dim);
    const float next = fmaxf(top, score), keep = top == -INFINITY ? 0.0f : expf(top - next), w = score == -INFINITY ? 0.0f : expf(score - next);
    sum = sum * keep + w;
    for (int e = 0; e < 2; ++e) o[e] = o[e] * keep + w * v.v[e];
    top = next;
  }
  put<T>(a.out, r, h, a.head_dim, o, sum == 0 ? 0.0f : 1.0f / sum);
  if (a.lse && threadIdx.x == 0) a.lse[uint64_t(h) * a.tokens + r] = sum == 0 ? -INFINITY : top + logf(sum);
}

// p and ds of row r and key j.
template <class T>
__device__ __forceinline__ float2 pair_of(const tsa_attend_grad_args& g, const Row<T>& q, const Row<T>& k, const Row<T>& v, const Row<T>& out,
                                          const Row<T>& dout, float lse) {
  const float score = q.dot(k) * g.f.scale, p = lse == -INFINITY ? 0.0f : expf(score - lse);
  return {p, p * (dout.dot(v) - dout.dot(out)) * g.f.scale};
}

template <class T>
__global__ __launch_bounds__(64) void queries_kernel(tsa_attend_grad_args g) {
  const tsa_attend_args& a = g.f;
  const uint32_t r = blockIdx.x, h = blockIdx.y, kept = h / (a.q.heads / a.k.heads);
  const uint32_t i = sequence_of(a.first, a.sequences, r);
  if (i >= a.sequences) return;
  const Span q = span_of(a.first, i, a.tokens), k = span_of(a.k_first ? a.k_first : a.first, i, a.k_tokens);
  if (r < q.begin || r >= q.begin + q.count) return;
  const int64_t keys = a.causal ? int64_t(k.count) - q.count + (r - q.begin) + 1 : k.count;
  const Row<T> x(a.q, r, h, a.head_dim), out(a.out, r, h, a.head_dim), dout(g.dout, r, h, a.head_dim);
  const float lse = a.lse[uint64_t(h) * a.tokens + r];
  float o[2] = {0, 0};
  for (int64_t j = 0; j < keys; ++j) {
    const Row<T> key(a.k, k.begin + j, kept, a.head_dim), v(a.v, k.begin + j, kept, a.head_dim);
    const float2 w = pair_of(g, x, key, v, out, dout, lse);
    for (int e = 0; e < 2; ++e) o[e] += w.y * key.v[e];
  }
  put<T>(g.dq, r, h, a.head_dim, o, 1.0f);
}

template <class T>
__global__ __launch_bounds__(64) void keys_kernel(tsa_attend_grad_args g) {
  const tsa_attend_args& a = g.f;
  const uint32_t r = blockIdx.x, kept = blockIdx.y, group = a.q.heads / a.k.heads;
  const int32_t* k_first = a.k_first ? a.k_first : a.first;
  const uint32_t i = sequence_of(k_first, a.sequences, r);
  if (i >= a.sequences) return;
  const Span q = span_of(a.first, i, a.tokens), k = span_of(k_first, i, a.k_tokens);
  if (r < k.begin || r >= k.begin + k.count) return;
  const Row<T> key(a.k, r, kept, a.head_dim), v(a.v, r, kept, a.head_dim);
  float dk[2] = {0, 0}, dv[2] = {0, 0};
  const int64_t from = a.causal ? int64_t(r - k.begin) - (int64_t(k.count) - q.count) : 0;  // the first query that sees it
  for (uint32_t h = kept * group; h < (kept + 1) * group; ++h)
    for (int64_t t = from < 0 ? 0 : from; t < q.count; ++t) {
      const uint64_t row = q.begin + t;
      const Row<T> x(a.q, row, h, a.head_dim), out(a.out, row, h, a.head_dim), dout(g.dout, row, h, a.head_dim);
      const float2 w = pair_of(g, x, key, v, out, dout, a.lse[uint64_t(h) * a.tokens + row]);
      for (int e = 0; e < 2; ++e) dk[e] += w.y * x.v[e], dv[e] += w.x * dout.v[e];
    }
  put<T>(g.dk, r, kept, a.head_dim, dk, 1.0f);
  put<T>(g.dv, r, kept, a.head_dim, dv, 1.0f);
}

}  // namespace
}  // namespace op

int launch_attend(const tsa_attend_args& a, hipStream_t stream) {
  const dim3 grid(a.tokens, a.q.heads);
  if (a.type == TSA_BF16) hipLaunchKernelGGL(op::attend_kernel<op::Bf16>, grid, dim3(64), 0, stream, a);
  else hipLaunchKernelGGL(op::attend_kernel<op::F16>, grid, dim3(64), 0, stream, a);
  return int(hipGetLastError());
}

uint64_t attend_backward_workspace(const tsa_attend_args&) { return 0; }

int launch_attend_backward(const tsa_attend_grad_args& g, void*, hipStream_t stream) {
  const dim3 queries(g.f.tokens, g.f.q.heads), keys(g.f.k_tokens, g.f.k.heads);
  const bool bf = g.f.type == TSA_BF16;
  if (g.dq.p && g.f.tokens) {
    if (bf) hipLaunchKernelGGL(op::queries_kernel<op::Bf16>, queries, dim3(64), 0, stream, g);
    else hipLaunchKernelGGL(op::queries_kernel<op::F16>, queries, dim3(64), 0, stream, g);
  }
  if (g.dk.p && g.f.k_tokens) {
    if (bf) hipLaunchKernelGGL(op::keys_kernel<op::Bf16>, keys, dim3(64), 0, stream, g);
    else hipLaunchKernelGGL(op::keys_kernel<op::F16>, keys, dim3(64), 0, stream, g);
  }
  return int(hipGetLastError());
}

}  // namespace tsa
