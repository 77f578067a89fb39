// Device parts the model operators share: the two 16-bit types with their matrix instruction, activations, 4-bit blocks,
// and the 64 x 64 tile that takes any stride and alignment.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "op_launch.hpp"

namespace tsa {
namespace op {

typedef uint16_t u16;
typedef uint16_t bits4 __attribute__((ext_vector_type(4)));
typedef uint16_t bits8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

// v_mfma_f32_16x16x32: lane l holds row (a) or column (b) l % 16 at k = 8 (l / 16) + 0..7, and of the result column
// l % 16 at rows 4 (l / 16) + 0..3. Products of 16-bit values are exact in 32 bits; sums are kept in 32.
struct Bf16 {
  typedef __bf16 v8 __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ f32x4 mfma(bits8 a, bits8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
  }
  // c += a b, c in the accumulator registers and staying where it is (for loops whose accumulators fill them).
  static __device__ __forceinline__ void mfma_in_place(f32x4& c, bits8 a, bits8 b) {
    asm("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
  }
  static __device__ __forceinline__ float up(u16 v) { return __builtin_bit_cast(float, uint32_t(v) << 16); }
  static __device__ __forceinline__ u16 down(float v) { return __builtin_bit_cast(u16, (__bf16)v); }
};
struct F16 {
  typedef _Float16 v8 __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ f32x4 mfma(bits8 a, bits8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
  }
  // c += a b, c in the accumulator registers and staying where it is (for loops whose accumulators fill them).
  static __device__ __forceinline__ void mfma_in_place(f32x4& c, bits8 a, bits8 b) {
    asm("v_mfma_f32_16x16x32_f16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
  }
  static __device__ __forceinline__ float up(u16 v) { return float(__builtin_bit_cast(_Float16, v)); }
  static __device__ __forceinline__ u16 down(float v) { return __builtin_bit_cast(u16, (_Float16)v); }
};

// A product's result on its way to be the operand of the next one. bf16 has the range of 32 bits: it is rounded where it is made.
// Half precision ends at 65504 and has fewer bits below 6e-5, so such a value stays in 32 bits until the largest of its row is
// known, and is rounded as what a power of two leaves of it (fit_kernel).
template <class T>
struct Held {
  typedef u16 type;
  static __device__ __forceinline__ u16 of(float v) { return T::down(v); }
};
template <>
struct Held<F16> {
  typedef float type;
  static __device__ __forceinline__ float of(float v) { return v; }
};
template <class T>
using held = typename Held<T>::type;

// The larger of two sizes, infinities and NaN left out.
__device__ __forceinline__ float peak(float top, float v) {
  const float a = fabsf(v);
  return a < INFINITY && a > top ? a : top;
}
// 2^-e and 2^e with the largest value `top` x 2^-e in [2^14, 2^15): 39 powers of two below it, half precision still has all its
// bits for 29 of them.
struct Fit {
  float down, up;
  explicit __device__ __forceinline__ Fit(float top) {
    const int x = int(__builtin_bit_cast(uint32_t, top) >> 23) - 127 - 14, e = x < -100 ? -100 : x;  // (113 at most)
    down = __builtin_bit_cast(float, uint32_t(127 - e) << 23);
    up = __builtin_bit_cast(float, uint32_t(127 + e) << 23);
  }
};

// 1 / (1 + exp(-v)) with the hardware's exponential and reciprocal: a few units of the last place of 32 bits for |v| below
// about 8, an absolute error below that beyond.
__device__ __forceinline__ float sigmoid(float v) { return __builtin_amdgcn_rcpf(1.0f + __expf(-v)); }

// Phi(v) = (1 + erf(v / sqrt 2)) / 2 by formula 7.1.26 of Abramowitz and Stegun's Handbook of Mathematical Functions (erf to
// 1.5e-7), with the exponential that the slope needs too.
struct Normal {
  float phi, density;  // density without its factor 1 / sqrt(2 pi)
};
__device__ __forceinline__ Normal normal(float v) {
  const float x = fabsf(v) * 0.70710678f, e = __expf(-x * x);
  const float t = __builtin_amdgcn_rcpf(1.0f + 0.3275911f * x);
  const float tail = 0.5f * t * e * (0.254829592f + t * (-0.284496736f + t * (1.421413741f + t * (-1.453152027f + t * 1.061405429f))));
  return {v < 0.0f ? tail : 1.0f - tail, e};
}

// act(v). The tanh form is v / (1 + exp(-2 z)), the same function as v (1 + tanh z) / 2 without the difference of
// nearly equal numbers at large negative z.
__device__ __forceinline__ float activate(uint32_t act, float v) {
  switch (act) {
    case TSA_ACT_SILU: return v * sigmoid(v);
    case TSA_ACT_GELU: return v * normal(v).phi;
    case TSA_ACT_GELU_TANH: return v * sigmoid(1.5957691f * (v + 0.044715f * v * v * v));
    case TSA_ACT_RELU: return v > 0.0f ? v : (v == v ? 0.0f : v);
    default: return v;
  }
}
// act'(v)
__device__ __forceinline__ float slope(uint32_t act, float v) {
  switch (act) {
    case TSA_ACT_SILU: {
      const float s = sigmoid(v);
      return s * (1.0f + v * (1.0f - s));
    }
    case TSA_ACT_GELU: {
      const Normal p = normal(v);
      return p.phi + v * p.density * 0.39894228f;
    }
    case TSA_ACT_GELU_TANH: {
      const float s = sigmoid(1.5957691f * (v + 0.044715f * v * v * v));
      return s + v * s * (1.0f - s) * 1.5957691f * (1.0f + 0.134145f * v * v);
    }
    case TSA_ACT_RELU: return v > 0.0f ? 1.0f : 0.0f;
    default: return 1.0f;
  }
}

__device__ __forceinline__ float load_as_float(const void* p, uint64_t i, uint32_t type) {
  if (type == TSA_F32) return static_cast<const float*>(p)[i];
  const u16 v = static_cast<const u16*>(p)[i];
  return type == TSA_BF16 ? Bf16::up(v) : F16::up(v);
}
__device__ __forceinline__ void store_float(void* p, uint64_t i, uint32_t type, float v) {
  if (type == TSA_F32) static_cast<float*>(p)[i] = v;
  else static_cast<u16*>(p)[i] = type == TSA_BF16 ? Bf16::down(v) : F16::down(v);
}

// ---- loads straight to LDS ----
static __device__ const u32x4 kZeroPiece = {0, 0, 0, 0};  // what a load past the end of a row or a sum reads

// 64 lanes x 16 bytes to LDS at `at` (the same in every lane) in lane order.
__device__ __forceinline__ void load_to_lds(const void* g, uint32_t at) {
  asm volatile(
      "s_mov_b32 m0, %1\n\t"
      "s_nop 0\n\t"
      "global_load_lds_dwordx4 %0, off"
      :
      : "v"(g), "s"(at)
      : "memory", "m0");
}
__device__ __forceinline__ uint32_t lds_offset(const void* p) {
  return uint32_t(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) const char*)p));
}

// ---- the 64 x 64 tile for any stride ----------------------------------------------------------------------------------
// A matrix operand: element (r, k) at base + r rs + k ks, rows through `map` if there is one; zero outside rows x n.
struct Operand {
  const u16* base = nullptr;
  uint64_t rs = 0, ks = 1;
  uint32_t rows = 0, n = 0;
  const uint32_t* map = nullptr;
  __device__ __forceinline__ bits8 load8(uint32_t r, uint32_t k) const {
    bits8 v = {0, 0, 0, 0, 0, 0, 0, 0};
    if (r >= rows) return v;
    const u16* p = base + uint64_t(map ? map[r] : r) * rs;
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i)
      if (k + i < n) v[i] = p[uint64_t(k + i) * ks];
    return v;
  }
};

// Rows of 4-bit blocks: the values 8 at a time without their scale (whole numbers -8..7, exact in either type).
template <class T>
struct Q4Operand {
  const unsigned char* base = nullptr;
  uint64_t row_bytes = 0;
  uint32_t rows = 0, n = 0;
  __device__ __forceinline__ bits8 load8(uint32_t r, uint32_t k) const {
    bits8 v = {0, 0, 0, 0, 0, 0, 0, 0};
    if (r >= rows || k >= n) return v;
    const unsigned char* p = base + r * row_bytes + uint64_t(k / 32) * kQ4Bytes + 2 + (k & 15u);
    const uint32_t shift = k & 16u ? 4 : 0;
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) v[i] = T::down(float(int((p[i] >> shift) & 15u) - 8));
    return v;
  }
  __device__ __forceinline__ float scale(uint32_t r, uint32_t k) const {
    if (r >= rows || k >= n) return 0.0f;
    const unsigned char* p = base + r * row_bytes + uint64_t(k / 32) * kQ4Bytes;
    return F16::up(u16(p[0] | p[1] << 8));
  }
};

struct TileMemory {
  u16 a[64][40], b[64][40];  // 32 values a row, 8 of padding
  float scale[64];
};

// acc[i][j] += the products of rows a0.. of `a` and rows b0.. of `b` over all k, by 256 threads: wave w covers a's rows
// 32 (w & 1).. and b's 32 (w >> 1)..; lane l's values are a-rows 16 i + 4 (l / 16) + 0..3, b-row 16 j + l % 16 of them.
template <class T, bool kQ4, class A, class B>
__device__ __forceinline__ void tile64(const A& a, uint32_t a0, const B& b, uint32_t b0, uint32_t n, TileMemory& m,
                                       f32x4 (&acc)[2][2]) {
  const uint32_t t = threadIdx.x, lane = t & 63u, wave = t >> 6;
  const uint32_t ar = (wave & 1u) * 32 + (lane & 15u), br = (wave >> 1) * 32 + (lane & 15u), kq = (lane >> 4) * 8;
  for (uint32_t k = 0; k < n; k += 32) {
    const bits8 va = a.load8(a0 + t / 4, k + (t & 3u) * 8), vb = b.load8(b0 + t / 4, k + (t & 3u) * 8);
    __syncthreads();  // the last step's reads are done
    *reinterpret_cast<bits8*>(&m.a[t / 4][(t & 3u) * 8]) = va;
    *reinterpret_cast<bits8*>(&m.b[t / 4][(t & 3u) * 8]) = vb;
    if constexpr (kQ4)
      if (t < 64) m.scale[t] = a.scale(a0 + t, k);
    __syncthreads();
#pragma unroll
    for (uint32_t i = 0; i < 2; ++i) {
      const bits8 fa = *reinterpret_cast<const bits8*>(&m.a[ar + 16 * i][kq]);
#pragma unroll
      for (uint32_t j = 0; j < 2; ++j) {
        const bits8 fb = *reinterpret_cast<const bits8*>(&m.b[br + 16 * j][kq]);
        if constexpr (kQ4) {  // 32 values are one block: its sum in whole steps, then the scale in 32 bits
          const f32x4 c = T::mfma(fa, fb, f32x4{0, 0, 0, 0});
          const float* s = &m.scale[(wave & 1u) * 32 + 16 * i + (lane >> 4) * 4];
#pragma unroll
          for (uint32_t r = 0; r < 4; ++r) acc[i][j][r] += s[r] * c[r];
        } else {
          acc[i][j] = T::mfma(fa, fb, acc[i][j]);
        }
      }
    }
  }
}

// f(a-row, b-row, value) for every value of a wave's part of the tile.
template <class F>
__device__ __forceinline__ void each64(const f32x4 (&acc)[2][2], F&& f) {
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
#pragma unroll
  for (uint32_t i = 0; i < 2; ++i)
#pragma unroll
    for (uint32_t j = 0; j < 2; ++j)
#pragma unroll
      for (uint32_t r = 0; r < 4; ++r)
        f((wave & 1u) * 32 + 16 * i + (lane >> 4) * 4 + r, (wave >> 1) * 32 + 16 * j + (lane & 15u), acc[i][j][r]);
}

}  // namespace op
}  // namespace tsa
