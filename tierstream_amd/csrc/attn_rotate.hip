// Rotary positions: pairs (a, b) of a head's values become (a cos - b sin, a sin + b cos) of position x frequency. Read once and
// written once; what bounds it is memory. The angle of a pair is the same for every head of a token, so a workgroup takes whole
// tokens: a thread each makes the sine and cosine of one pair (in 64 bits down to an eighth of a turn, where short power series
// give 32), they go to LDS, and every head reads them from there. No table of all positions is read. Pieces of 8 values a lane, a piece of
// each half where the halves are pairs.
// Measured: 8191 tokens of 36 heads of 128, 64 of them turned, 33.7 us (302 MB with the gradient's in 67: 4.5 TB/s, a large copy reaches
// 4.9); one token of 40 heads 2.9, a launch and two memory latencies.
#include "op_device.hpp"
// (behind the HIP runtime's own header)
#include "attn_launch.hpp"

namespace tsa {
namespace op {
namespace {

constexpr uint32_t kRotateThreads = 256, kRotateTable = 1024;  // pairs whose turns a workgroup holds (8 KiB)

// cos and sin of t turns. sin and cos of |f| <= pi / 4 by their power series: the first terms left out are below 2e-9.
__device__ __forceinline__ float2 turn(double t) {
  t -= rint(t);
  const double k = rint(4.0 * t);
  const float f = float((t - 0.25 * k) * 6.283185307179586), s = f * f;
  const float sn = f + f * s * (-1.0f / 6 + s * (1.0f / 120 + s * (-1.0f / 5040 + s * (1.0f / 362880))));
  const float cs = 1.0f + s * (-0.5f + s * (1.0f / 24 + s * (-1.0f / 720 + s * (1.0f / 40320 - s * (1.0f / 3628800)))));
  switch (int(k) & 3) {
    case 0: return {cs, sn};
    case 1: return {-sn, cs};
    case 2: return {-cs, -sn};
    default: return {sn, -cs};
  }
}

template <uint32_t kType, int N>
struct Values {
  float v[N];
  __device__ __forceinline__ void load(const void* p, uint64_t at) {
    if constexpr (kType == TSA_F32) {
      const f32x4* g = reinterpret_cast<const f32x4*>(static_cast<const float*>(p) + at);
#pragma unroll
      for (int i = 0; i < N; i += 4) {
        const f32x4 w = g[i / 4];
#pragma unroll
        for (int j = 0; j < 4; ++j) v[i + j] = w[j];
      }
    } else {
      const bits8 w = *reinterpret_cast<const bits8*>(static_cast<const u16*>(p) + at);
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = kType == TSA_BF16 ? Bf16::up(w[i]) : F16::up(w[i]);
    }
  }
  __device__ __forceinline__ void store(void* p, uint64_t at) const {
    if constexpr (kType == TSA_F32) {
      f32x4* g = reinterpret_cast<f32x4*>(static_cast<float*>(p) + at);
#pragma unroll
      for (int i = 0; i < N; i += 4) g[i / 4] = f32x4{v[i], v[i + 1], v[i + 2], v[i + 3]};
    } else {
      bits8 w;
#pragma unroll
      for (int i = 0; i < N; ++i) w[i] = kType == TSA_BF16 ? Bf16::down(v[i]) : F16::down(v[i]);
      *reinterpret_cast<bits8*>(static_cast<u16*>(p) + at) = w;
    }
  }
};

struct RotateShape {
  uint32_t per_head, turned;  // pieces of a head, the turned ones first
  uint32_t items;             // pieces of a token
  uint32_t tokens;            // of a workgroup
};

// kVector: pieces are 8 values (in halves: 8 of each half), 16-byte aligned; otherwise a pair, and behind the pairs a value.
template <uint32_t kType, bool kVector, bool kInterleaved>
__global__ __launch_bounds__(kRotateThreads) void rotate_kernel(tsa_rotary r, tsa_rotate_args a, RotateShape s) {
  __shared__ float2 turn_s[kRotateTable];
  __shared__ int32_t position_s[kRotateThreads];
  const uint32_t token0 = blockIdx.x * s.tokens, here = min(s.tokens, a.tokens - token0);
  const float amplitude = float(r.amplitude);
  for (uint32_t i = threadIdx.x; i < here * r.pairs; i += kRotateThreads) {
    const uint32_t t = i / r.pairs, p = i - t * r.pairs;
    const int32_t position = a.positions[token0 + t];
    const float2 w = turn(double(position) * r.turns[p]);
    turn_s[i] = {amplitude * w.x, a.backward ? -amplitude * w.y : amplitude * w.y};
    if (p == 0) position_s[t] = position;
  }
  __syncthreads();
  const uint32_t half = r.pairs, rotated = 2 * r.pairs, heads0 = a.x[0].heads;
  for (uint32_t i = threadIdx.x; i < here * s.items; i += kRotateThreads) {
    const uint32_t t = i / s.items, in = i - t * s.items;
    uint32_t head = in / s.per_head;
    const uint32_t piece = in - head * s.per_head;
    if (position_s[t] < 0) continue;
    const bool second = head >= heads0;
    if (second) head -= heads0;
    const tsa_heads& x = a.x[second];
    const tsa_heads& y = a.y[second];
    const uint64_t from = uint64_t(token0 + t) * x.token_stride + uint64_t(head) * x.head_stride;
    const uint64_t to = uint64_t(token0 + t) * y.token_stride + uint64_t(head) * y.head_stride;
    const float2* w = turn_s + t * r.pairs;
    if constexpr (kVector) {
      if (piece >= s.turned) {
        const uint32_t at = rotated + 8 * (piece - s.turned);
        if (x.p == y.p) continue;
        Values<kType, 8> v;
        v.load(x.p, from + at);
        v.store(y.p, to + at);
      } else if constexpr (kInterleaved) {
        Values<kType, 8> v;
        v.load(x.p, from + 8 * piece);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float2 c = w[4 * piece + k];
          const float p = v.v[2 * k], q = v.v[2 * k + 1];
          v.v[2 * k] = p * c.x - q * c.y;
          v.v[2 * k + 1] = p * c.y + q * c.x;
        }
        v.store(y.p, to + 8 * piece);
      } else {
        Values<kType, 8> p, q;
        p.load(x.p, from + 8 * piece);
        q.load(x.p, from + half + 8 * piece);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const float2 c = w[8 * piece + k];
          const float u = p.v[k], v = q.v[k];
          p.v[k] = u * c.x - v * c.y;
          q.v[k] = u * c.y + v * c.x;
        }
        p.store(y.p, to + 8 * piece);
        q.store(y.p, to + half + 8 * piece);
      }
    } else {
      if (piece >= s.turned) {
        const uint32_t at = rotated + piece - s.turned;
        if (x.p != y.p) store_float(y.p, to + at, kType, load_as_float(x.p, from + at, kType));
        continue;
      }
      const uint32_t first = kInterleaved ? 2 * piece : piece, other = kInterleaved ? 2 * piece + 1 : piece + half;
      const float2 c = w[piece];
      const float u = load_as_float(x.p, from + first, kType), v = load_as_float(x.p, from + other, kType);
      store_float(y.p, to + first, kType, u * c.x - v * c.y);
      store_float(y.p, to + other, kType, u * c.y + v * c.x);
    }
  }
}

bool pieces_aligned(const tsa_heads& h, uint32_t type) {
  const uint64_t size = type == TSA_F32 ? 4 : 2;
  return h.heads == 0 || (reinterpret_cast<uintptr_t>(h.p) % 16 == 0 && h.token_stride * size % 16 == 0 && h.head_stride * size % 16 == 0);
}

template <uint32_t kType, bool kVector>
void rotate(const tsa_rotary& r, const tsa_rotate_args& a, const RotateShape& s, hipStream_t stream) {
  const dim3 grid((a.tokens + s.tokens - 1) / s.tokens), block(kRotateThreads);
  if (r.interleaved) hipLaunchKernelGGL((rotate_kernel<kType, kVector, true>), grid, block, 0, stream, r, a, s);
  else hipLaunchKernelGGL((rotate_kernel<kType, kVector, false>), grid, block, 0, stream, r, a, s);
}

}  // namespace
}  // namespace op

int launch_rotate(const tsa_rotary& r, const tsa_rotate_args& a, hipStream_t stream) {
  using namespace op;
  // Pieces of 8 values where every piece starts 16-byte aligned; any other layout goes pair by pair.
  bool vector = (r.interleaved ? r.pairs % 4 : r.pairs % 8) == 0 && a.head_dim % 8 == 0;
  for (int i = 0; i < 2; ++i) vector = vector && pieces_aligned(a.x[i], a.type) && pieces_aligned(a.y[i], a.type);
  RotateShape s;
  s.turned = !vector ? r.pairs : r.interleaved ? r.pairs / 4 : r.pairs / 8;
  s.per_head = s.turned + (a.head_dim - 2 * r.pairs) / (vector ? 8 : 1);
  s.items = (a.x[0].heads + a.x[1].heads) * s.per_head;
  // as many tokens as give every thread a piece, and whose turns have room
  s.tokens = kRotateThreads / s.items;
  if (s.tokens < 1) s.tokens = 1;
  if (s.tokens > kRotateTable / r.pairs) s.tokens = kRotateTable / r.pairs;
#define CALL(T)                                              \
  if (vector) rotate<T, true>(r, a, s, stream);              \
  else rotate<T, false>(r, a, s, stream);
  if (a.type == TSA_F32) { CALL(TSA_F32) }
  else if (a.type == TSA_BF16) { CALL(TSA_BF16) }
  else { CALL(TSA_F16) }
#undef CALL
  return int(hipGetLastError());
}

}  // namespace tsa
