// Device parts the attention operators share.
#pragma once

#include "op_device.hpp"
// (behind the HIP runtime's own header)
#include "attn_launch.hpp"

namespace tsa {
namespace op {

// Heads of 16-bit values whose pieces of 8 start 16-byte aligned.
inline bool vector_heads(const tsa_heads& h) {
  return reinterpret_cast<uintptr_t>(h.p) % 16 == 0 && h.token_stride % 8 == 0 && h.head_stride % 8 == 0;
}

// Sums that stay at the largest number where they would pass it.
__device__ __forceinline__ uint32_t add_sat(uint32_t a, uint32_t b) { return __builtin_elementwise_add_sat(a, b); }

// A sequence's rows inside its array, whatever `first` holds.
struct Span {
  uint32_t begin, count;
};
__device__ __forceinline__ Span span_of(const int32_t* first, uint32_t i, uint32_t rows) {
  if (!first) return {0, rows};
  const int64_t b = first[i], e = first[i + 1], begin = b < 0 ? 0 : b, end = e > int64_t(rows) ? int64_t(rows) : e;
  return begin < end ? Span{uint32_t(begin), uint32_t(end - begin)} : Span{0, 0};
}

// The sequence of row r: the last i with first[i] <= r; n where r lies behind the last one.
__device__ __forceinline__ uint32_t sequence_of(const int32_t* first, uint32_t n, uint32_t r) {
  if (!first) return 0;
  if (int64_t(first[n]) <= int64_t(r)) return n;
  uint32_t lo = 0, hi = n;
  while (hi - lo > 1) {
    const uint32_t mid = (lo + hi) / 2;
    if (int64_t(first[mid]) <= int64_t(r)) lo = mid;
    else hi = mid;
  }
  return lo;
}

template <class T>
__device__ __forceinline__ const T* row_of(const tsa_heads& h, uint64_t token, uint32_t head) {
  return static_cast<const T*>(h.p) + token * h.token_stride + head * h.head_stride;
}

// 64 lanes x 4 bytes to LDS at `at` (the same in every lane) in lane order.
__device__ __forceinline__ void load_words_to_lds(const void* g, uint32_t at) {
  asm volatile(
      "s_mov_b32 m0, %1\n\t"
      "s_nop 0\n\t"
      "global_load_lds_dword %0, off"
      :
      : "v"(g), "s"(at)
      : "memory", "m0");
}

}  // namespace op
}  // namespace tsa
