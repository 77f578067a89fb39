// Attention of new tokens over the pages of their requests: one wave a query row, the running maximum and sum of its softmax, a key at
// a time.
#include "attn_device.hpp"

namespace tsa {
namespace op {
namespace {

template <class T>
__global__ __launch_bounds__(64) void cached_kernel(tsa_cache c, tsa_attend_cached_args a) {
  const uint32_t lane = threadIdx.x, r = blockIdx.x, h = blockIdx.y, kept = h / (a.q.heads / c.kv_heads), nb = c.head_dim / 32;
  const uint32_t i = sequence_of(a.first, a.requests, r);
  if (i >= a.requests) return;
  const Span rows = span_of(a.first, i, a.tokens);
  if (r < rows.begin || r >= rows.begin + rows.count) return;
  const int64_t end = min(int64_t(a.ends[i]), int64_t(a.width) * kPage);
  const int64_t keys = end - rows.count + (r - rows.begin) + 1;
  const u16* q = row_of<u16>(a.q, r, h);
  float x[2], o[2] = {0, 0}, top = -INFINITY, sum = 0;
  for (int k = 0; k < 2; ++k) x[k] = lane + 64 * k < c.head_dim ? T::up(q[lane + 64 * k]) * a.scale : 0.0f;
  for (int64_t j = 0; j < keys; ++j) {
    const uint32_t page = uint32_t(a.table[i * a.table_stride + j / kPage]), row = uint32_t(j % kPage);
    if (page >= c.n_pages) continue;
    const unsigned char* p = static_cast<const unsigned char*>(c.pages) + (uint64_t(page) * c.kv_heads + kept) * (72 * c.head_dim);
    const u16* scales = reinterpret_cast<const u16*>(p + nb * 1024);
    float k[2] = {0, 0}, v[2] = {0, 0}, score = 0;
    for (uint32_t e = 0; e < 2; ++e) {
      const uint32_t d = lane + 64 * e, b = d / 32, in = d % 16, shift = d % 32 >= 16 ? 4 : 0;
      if (d >= c.head_dim) continue;
      k[e] = float(int((p[(row * 4 + in / 4) * nb * 4 + b * 4 + in % 4] >> shift) & 15) - 8) * F16::up(scales[row * nb + b]);
      v[e] = float(int((p[nb * 1280 + (b * kPage + row) * 16 + in] >> shift) & 15) - 8) * F16::up(scales[(kPage + row) * nb + b]);
      score += x[e] * k[e];
    }
    score = lanes_sum(score);
    const float next = fmaxf(top, score), keep = top == -INFINITY ? 0.0f : expf(top - next), w = score == -INFINITY ? 0.0f : expf(score - next);
    sum = sum * keep + w;
    for (int e = 0; e < 2; ++e) o[e] = o[e] * keep + w * v[e];
    top = next;
  }
  u16* out = const_cast<u16*>(row_of<u16>(a.out, r, h));
  for (int k = 0; k < 2; ++k)
    if (lane + 64 * k < c.head_dim) out[lane + 64 * k] = T::down(sum > 0 ? o[k] / sum : sum == 0 ? 0.0f : sum);
}

}  // namespace
}  // namespace op

uint64_t attend_cached_workspace(const tsa_cache&, const tsa_attend_cached_args&) { return 0; }

int launch_attend_cached(const tsa_cache& c, const tsa_attend_cached_args& a, void*, hipStream_t stream) {
  const dim3 grid(a.tokens, a.q.heads);
  if (a.type == TSA_BF16) hipLaunchKernelGGL(op::cached_kernel<op::Bf16>, grid, dim3(64), 0, stream, c, a);
  else hipLaunchKernelGGL(op::cached_kernel<op::F16>, grid, dim3(64), 0, stream, c, a);
  return int(hipGetLastError());
}

}  // namespace tsa
