// The choice of experts: top_k of each row's logits with softmax weights, and the logits' gradient. One wave per row: the
// row's logits stay in registers (at most 1024 = 16 a lane), the k maxima are found one after the other. A step is a
// wave-wide maximum of order-preserving 32-bit keys, six register moves, and the lowest id that has it, one ballot per
// register: nothing goes through memory. One row of 256: 4.8 us, a launch and two memory latencies; 8191 rows of 128 in 16 bits,
// 8 of them: 9.0 us, the steps' arithmetic (2.6 MB in all), and 5.8 for the gradient (4.9 MB).
#include "op_device.hpp"

namespace tsa {
namespace op {
namespace {

constexpr uint32_t kRouteWaves = 4;

// Ascending keys for ascending values; 0 for a masked one (-infinity, NaN). -0 and 0 are equal.
__device__ __forceinline__ uint32_t key_of(float v) {
  if (!(v > -INFINITY)) return 0;
  const uint32_t b = __builtin_bit_cast(uint32_t, v + 0.0f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key) {
  return __builtin_bit_cast(float, key & 0x80000000u ? key & 0x7FFFFFFFu : ~key);
}

__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
  for (int s = 1; s < 64; s <<= 1) {
    const uint32_t o = __shfl_xor(v, s, 64);
    v = o > v ? o : v;
  }
  return v;
}
__device__ __forceinline__ float wave_sum(float v) {
  for (int s = 1; s < 64; s <<= 1) v += __shfl_xor(v, s, 64);
  return v;
}

// exp(v - best), 1 at the best itself (also where both are infinite)
__device__ __forceinline__ float rise(uint32_t key, uint32_t best) {
  return key == 0 ? 0.0f : key == best ? 1.0f : expf(value_of(key) - value_of(best));
}

template <uint32_t kPer>
__device__ __forceinline__ void load_keys(const tsa_route_args& a, uint64_t row, uint32_t lane, uint32_t (&key)[kPer]) {
#pragma unroll
  for (uint32_t i = 0; i < kPer; ++i) {
    const uint32_t e = 64 * i + lane;
    key[i] = e < a.n_experts ? key_of(load_as_float(a.logits, row * a.logits_stride + e, a.type)) : 0;
  }
}

template <uint32_t kPer>
__global__ __launch_bounds__(64 * kRouteWaves) void route_kernel(tsa_route_args a) {
  const uint32_t lane = threadIdx.x & 63u;
  const uint64_t step = uint64_t(gridDim.x) * kRouteWaves;
  for (uint64_t row = uint64_t(blockIdx.x) * kRouteWaves + (threadIdx.x >> 6); row < a.rows; row += step) {
    uint32_t key[kPer];
    load_keys<kPer>(a, row, lane, key);
    uint32_t best = 0, mine = 0;
    int32_t id = -1;
    float all = 0.0f;
    for (uint32_t j = 0; j < a.top_k; ++j) {
      uint32_t top = 0;
#pragma unroll
      for (uint32_t i = 0; i < kPer; ++i) top = key[i] > top ? key[i] : top;
      top = wave_max(top);
      if (j == 0) {
        best = top;
        if (!a.renorm) {
#pragma unroll
          for (uint32_t i = 0; i < kPer; ++i) all += rise(key[i], best);
          all = wave_sum(all);
        }
      }
      if (top == 0) break;
      bool found = false;
#pragma unroll
      for (uint32_t i = 0; i < kPer; ++i) {
        const uint64_t has = __ballot(key[i] == top);
        if (!found && has) {
          found = true;
          const uint32_t l = uint32_t(__builtin_ctzll(has));
          if (lane == l) key[i] = 0;
          if (lane == j) id = int32_t(64 * i + l), mine = top;
        }
      }
    }
    const float e = rise(mine, best);
    const float sum = a.renorm ? wave_sum(e) : all;
    if (lane < a.top_k) {
      a.ids[row * a.top_k + lane] = id;
      a.weights[row * a.top_k + lane] = id < 0 ? 0.0f : a.scale * (e / sum);
    }
  }
}

// With p the normalised exponentials (over the chosen or over all) and w = scale p: d logit_i = scale p_i (d w_i - sum_j
// p_j d w_j), where d w_i is 0 for what was not chosen. The chosen ones' terms reach their lanes through LDS.
template <uint32_t kPer>
__global__ __launch_bounds__(64 * kRouteWaves) void route_backward_kernel(tsa_route_args a, const float* dweights,
                                                                          void* dlogits, uint64_t stride) {
  __shared__ float pull_s[kRouteWaves][64 * kPer];
  __shared__ uint32_t key_s[kRouteWaves][64 * kPer];
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
  const uint64_t step = uint64_t(gridDim.x) * kRouteWaves;
  const uint64_t rounds = (a.rows + step - 1) / step;
  for (uint64_t it = 0; it < rounds; ++it) {  // (every wave takes part in the barriers)
    const uint64_t row = it * step + uint64_t(blockIdx.x) * kRouteWaves + wave;
    const bool on = row < a.rows;
    uint32_t key[kPer];
    uint32_t best = 0;
#pragma unroll
    for (uint32_t i = 0; i < kPer; ++i) key[i] = 0;
    if (on) load_keys<kPer>(a, row, lane, key);
#pragma unroll
    for (uint32_t i = 0; i < kPer; ++i) {
      best = key[i] > best ? key[i] : best;
      key_s[wave][64 * i + lane] = key[i];
      pull_s[wave][64 * i + lane] = 0.0f;
    }
    best = wave_max(best);
    __syncthreads();
    const int32_t id = on && lane < a.top_k ? a.ids[row * a.top_k + lane] : -1;
    const bool chosen = id >= 0 && uint32_t(id) < a.n_experts;
    const float dw = chosen ? dweights[row * a.top_k + lane] : 0.0f;
    const float e = chosen ? rise(key_s[wave][id], best) : 0.0f;
    float sum = 0.0f;
    if (a.renorm) {
      sum = e;
    } else {
#pragma unroll
      for (uint32_t i = 0; i < kPer; ++i) sum += rise(key[i], best);
    }
    sum = wave_sum(sum);
    const float inv = sum > 0.0f ? 1.0f / sum : 0.0f;
    const float mean = wave_sum(e * inv * dw);
    __syncthreads();
    if (chosen) {
      pull_s[wave][id] = a.renorm ? a.scale * (e * inv) * (dw - mean) : dw;
    }
    __syncthreads();
    if (on)
#pragma unroll
      for (uint32_t i = 0; i < kPer; ++i) {
        const uint32_t x = 64 * i + lane;
        if (x >= a.n_experts) continue;
        const float pull = pull_s[wave][x];
        const float d = a.renorm ? pull : key[i] == 0 ? 0.0f : a.scale * (rise(key[i], best) * inv) * (pull - mean);
        store_float(dlogits, row * stride + x, a.type, d);
      }
    __syncthreads();
  }
}

uint32_t route_grid(uint32_t rows) {
  const uint64_t b = (uint64_t(rows) + kRouteWaves - 1) / kRouteWaves;
  return uint32_t(b < 65536 ? b : 65536);
}

}  // namespace
}  // namespace op

#define TSA_BY_EXPERTS(n, CALL)      \
  do {                               \
    if ((n) <= 64) { CALL(1); }      \
    else if ((n) <= 128) { CALL(2); } \
    else if ((n) <= 256) { CALL(4); } \
    else if ((n) <= 512) { CALL(8); } \
    else { CALL(16); }               \
  } while (0)

int launch_route(const tsa_route_args& a, hipStream_t stream) {
  if (a.rows == 0) return 0;
#define CALL(P) \
  hipLaunchKernelGGL(op::route_kernel<P>, dim3(op::route_grid(a.rows)), dim3(64 * op::kRouteWaves), 0, stream, a)
  TSA_BY_EXPERTS(a.n_experts, CALL);
#undef CALL
  return int(hipGetLastError());
}

int launch_route_backward(const tsa_route_args& a, const float* dweights, void* dlogits, uint64_t stride,
                          hipStream_t stream) {
  if (a.rows == 0) return 0;
#define CALL(P)                                                                                                       \
  hipLaunchKernelGGL(op::route_backward_kernel<P>, dim3(op::route_grid(a.rows)), dim3(64 * op::kRouteWaves), 0, stream, \
                     a, dweights, dlogits, stride)
  TSA_BY_EXPERTS(a.n_experts, CALL);
#undef CALL
  return int(hipGetLastError());
}

}  // namespace tsa
