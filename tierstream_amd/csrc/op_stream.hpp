// Products of weights with few rows of x: bound by the bytes of the weights, which cross memory once and go
// straight to registers in the layout the matrix instruction takes, without LDS.
//
// The result column of v_mfma_f32_16x16x32 (operand b) is a weight row, the result row (operand a) a row of x: lane l holds
// weight row l % 16 at 8 values of each 32, and of the result the x rows 4 (l / 16) + 0..3. The order of the 32 values
// inside a step is free as long as both operands use the same, so a 4-bit lane takes the 4 bytes 4 (l / 16).. of a block
// in one load: values 4 (l / 16) + 0..3 from their low halves, 16 more from their high ones.
//
// The waves of a workgroup take turns along the row in chunks of 128 values, each with the next chunk's loads in flight
// while it multiplies this one's, and add up through LDS. x is read from the caches, or if it is one row from LDS.
//
// One row through 4096 x 28672 (235 MB of 16-bit weights): 43 us, 5.5 TB/s; two experts of 4096 x 14336: gate and up (470 MB) 83 us,
// 5.7 TB/s, down (235 MB) 49 us, 4.8. A lane keeps one row, so an instruction reads 64 bytes of each of 16; a second chunk in
// flight, twice or half the waves, or another first chunk in every workgroup gives the same or up to 10 % less.
#pragma once

#include "op_device.hpp"

namespace tsa {
namespace op {

constexpr uint32_t kChunk = 128;  // values of a weight row per chunk: 4 steps

// 16-byte accesses at any element's alignment (the hardware takes them at every address).
typedef bits8 bits8_any __attribute__((aligned(2)));
typedef bits4 bits4_any __attribute__((aligned(2)));
typedef __attribute__((address_space(1))) const bits8_any gbits8_t;
typedef __attribute__((address_space(1))) const bits4_any gbits4_t;

__device__ __forceinline__ bits8 load_bits8(const u16* p) {
  return *reinterpret_cast<gbits8_t*>(reinterpret_cast<uintptr_t>(p));
}
// Weights are read once: past the caches.
__device__ __forceinline__ bits8 load_stream(const u16* p) {
  return __builtin_nontemporal_load(reinterpret_cast<gbits8_t*>(reinterpret_cast<uintptr_t>(p)));
}
// The first `left` of 8 values (0 or fewer: none), zeros behind them.
__device__ __forceinline__ bits8 load_end(const u16* p, int left) {
  bits8 v = {0, 0, 0, 0, 0, 0, 0, 0};
  if (left >= 8) return load_bits8(p);
#pragma unroll
  for (int i = 0; i < 7; ++i)
    if (i < left) v[i] = p[i];
  return v;
}

// 16-bit weight rows: base at row 0, `stride` values apart, at any alignment.
template <class T>
struct Rows16 {
  struct Chunk {
    bits8 v[4];
  };
  const u16* p;  // this lane's row at its first value
  uint32_t n;
  Rows16() = default;
  __device__ __forceinline__ Rows16(const void* base, uint64_t stride, uint32_t row, uint32_t n_) : n(n_) {
    p = static_cast<const u16*>(base) + row * stride + (threadIdx.x & 48u) / 2;
  }
  // The chunk at k; kTail: the row may end inside it (zeros from there on).
  template <bool kTail>
  __device__ __forceinline__ void load(Chunk& c, uint32_t k) const {
    const uint32_t q = (threadIdx.x & 48u) / 2;
#pragma unroll
    for (int s = 0; s < 4; ++s)
      c.v[s] = !kTail || k + 32 * s + q + 8 <= n ? load_stream(p + k + 32 * s) : load_end(p + k + 32 * s, int(n) - int(k + 32 * s + q));
  }
  // Values of x for the step at k, from its row.
  template <bool kTail>
  static __device__ __forceinline__ bits8 x_at(const u16* row, uint32_t k, uint32_t n) {
    const uint32_t at = k + (threadIdx.x & 48u) / 2;
    return !kTail || at + 8 <= n ? load_bits8(row + at) : load_end(row + at, int(n) - int(at));
  }
  template <int R, int CT>
  static __device__ __forceinline__ void multiply(const Chunk (&c)[R], int s, const bits8 (&x)[CT], f32x4 (&acc)[R][CT]) {
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int t = 0; t < CT; ++t) acc[r][t] = T::mfma(x[t], c[r].v[s], acc[r][t]);
  }
};

// 4-bit halves as 16-bit floating values, offset so that it takes a byte permutation: bf16 holds 16 + q as 0x4180 + 8 q, half
// precision as 0x4C00 + 64 q. The offset's part of the sum, 24 to the value q - 8, is taken off with a product of x and -24
// (exact in either type; 16 is the least power of two above all q, so that it cancels few bits).
template <class T>
struct HalfBytes;
template <>
struct HalfBytes<Bf16> {
  static constexpr u16 kMinus = 0xC1C0;  // -24
  static __device__ __forceinline__ bits8 unpack(uint32_t v) {
    const uint32_t lo = ((v << 3) & 0x78787878u) | 0x80808080u, hi = ((v >> 1) & 0x78787878u) | 0x80808080u;
    const u32x4 r = {__builtin_amdgcn_perm(0x41414141u, lo, 0x04010400u), __builtin_amdgcn_perm(0x41414141u, lo, 0x04030402u),
                     __builtin_amdgcn_perm(0x41414141u, hi, 0x04010400u), __builtin_amdgcn_perm(0x41414141u, hi, 0x04030402u)};
    return __builtin_bit_cast(bits8, r);
  }
};
template <>
struct HalfBytes<F16> {
  static constexpr u16 kMinus = 0xCE00;  // -24
  // 16 + q as 0x4C00 + 64 q: the byte pair (0x4C + q / 4, 64 (q % 4)) by shifting the half byte over the pair
  static __device__ __forceinline__ bits8 unpack(uint32_t v) {
    const uint32_t lo = v & 0x0F0F0F0Fu, hi = (v >> 4) & 0x0F0F0F0Fu;
    const u32x4 r = {(__builtin_amdgcn_perm(0, lo, 0x0C010C00u) << 6) | 0x4C004C00u,
                     (__builtin_amdgcn_perm(0, lo, 0x0C030C02u) << 6) | 0x4C004C00u,
                     (__builtin_amdgcn_perm(0, hi, 0x0C010C00u) << 6) | 0x4C004C00u,
                     (__builtin_amdgcn_perm(0, hi, 0x0C030C02u) << 6) | 0x4C004C00u};
    return __builtin_bit_cast(bits8, r);
  }
};

// Rows of 4-bit blocks back to back (n / 32 blocks each), 4-byte aligned at the base. A step is one block: its products
// are summed in whole steps of the scale, which is applied to the sum in 32 bits.
template <class T>
struct RowsQ4 {
  struct Chunk {
    uint32_t v[4];
    u16 scale[4];
  };
  const unsigned char* p;  // this lane's row, first block
  uint32_t n;
  RowsQ4() = default;
  __device__ __forceinline__ RowsQ4(const void* base, uint64_t, uint32_t row, uint32_t n_) : n(n_) {
    p = static_cast<const unsigned char*>(base) + uint64_t(row) * (n_ / kQ4Block * kQ4Bytes);
  }
  struct __attribute__((packed, aligned(2))) Word {
    uint32_t v;
  };
  typedef __attribute__((address_space(1))) const Word gword_t;
  typedef __attribute__((address_space(1))) const u16 ghalf_t;
  __device__ __forceinline__ void load_block(Chunk& c, int s, uint32_t k) const {
    const uintptr_t b = reinterpret_cast<uintptr_t>(p) + (k / kQ4Block) * kQ4Bytes;
    c.scale[s] = *reinterpret_cast<ghalf_t*>(b);
    c.v[s] = reinterpret_cast<gword_t*>(b + 2 + (threadIdx.x & 48u) / 4)->v;
  }
  template <bool kTail>
  __device__ __forceinline__ void load(Chunk& c, uint32_t k) const {
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      if (kTail) c.scale[s] = 0, c.v[s] = 0;
      if (!kTail || k + 32 * s < n) load_block(c, s, k + 32 * s);
    }
  }
  template <bool kTail>
  static __device__ __forceinline__ bits8 x_at(const u16* row, uint32_t k, uint32_t n) {
    if (kTail && k >= n) return bits8{0, 0, 0, 0, 0, 0, 0, 0};
    const uintptr_t at = reinterpret_cast<uintptr_t>(row + k + (threadIdx.x & 48u) / 4);
    const bits4 lo = *reinterpret_cast<gbits4_t*>(at), hi = *reinterpret_cast<gbits4_t*>(at + 32);
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  }
  template <int R, int CT>
  static __device__ __forceinline__ void multiply(const Chunk (&c)[R], int s, const bits8 (&x)[CT], f32x4 (&acc)[R][CT]) {
    constexpr u16 m = HalfBytes<T>::kMinus;
    bits8 w[R];
#pragma unroll
    for (int r = 0; r < R; ++r) w[r] = HalfBytes<T>::unpack(c[r].v[s]);
#pragma unroll
    for (int t = 0; t < CT; ++t) {
      const f32x4 off = T::mfma(x[t], bits8{m, m, m, m, m, m, m, m}, f32x4{0, 0, 0, 0});
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const f32x4 sum = T::mfma(x[t], w[r], off);
        const float scale = F16::up(c[r].scale[s]);
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[r][t][i] += scale * sum[i];
      }
    }
  }
};

// acc[r][t] += chunks wave, wave + waves, .. below n_chunks. at(c, w, row) gives chunk c's weight rows w[r], this lane's x
// row of each tile (operand a: lane l gives row l % 16; with one row in all, every lane gives it; null for none) and
// returns its first value k. The next chunk's x is loaded with its weights: loads return in order, so one issued later
// would wait for all of them.
template <class W, int R, int CT, bool kTail, class At>
__device__ __forceinline__ void stream_chunks(uint32_t n_chunks, uint32_t wave, uint32_t waves, At&& at, f32x4 (&acc)[R][CT]) {
  struct Step {
    typename W::Chunk c[R];
    bits8 x[4][CT];
  };
  auto load = [&](Step& b, uint32_t c) {
    W w[R];
    const u16* row[CT];
    const uint32_t k = at(c, w, row);
#pragma unroll
    for (int r = 0; r < R; ++r) w[r].template load<kTail>(b.c[r], k);
#pragma unroll
    for (int s = 0; s < 4; ++s)
#pragma unroll
      for (int t = 0; t < CT; ++t)
        b.x[s][t] = row[t] ? W::template x_at<kTail>(row[t], k + 32 * s, w[0].n) : bits8{0, 0, 0, 0, 0, 0, 0, 0};
  };
  auto multiply = [&](const Step& b) {
#pragma unroll
    for (int s = 0; s < 4; ++s) W::template multiply<R, CT>(b.c, s, b.x[s], acc);
  };
  uint32_t c = wave;
  if (c >= n_chunks) return;
  Step now;
  load(now, c);
  for (; c + waves < n_chunks; c += waves) {
    Step next;
    load(next, c + waves);
    multiply(now);
    now = next;
  }
  multiply(now);
}

// The same for one row of x that lies in LDS from `row` on, chunk after chunk: stage() puts it there and meets the other waves,
// behind the first chunk's loads. (From the caches a row of x is as many loads as one of weights: 46.5 us for 43.2, 4096 x 28672;
// down of two experts of 14336 x 4096 53.4 for 48.8.)
template <class T, int R, bool kTail, class At, class Stage>
__device__ __forceinline__ void stream_one(uint32_t n_chunks, uint32_t wave, uint32_t waves, uint32_t row, At&& at, Stage&& stage, f32x4 (&acc)[R][1]) {
  typedef Rows16<T> W;
  struct Step {
    typename W::Chunk c[R];
    uint32_t x;
  };
  typedef __attribute__((address_space(3))) const bits8 lds_bits8_t;
  auto load = [&](Step& b, uint32_t c) {
    W w[R];
    const uint32_t k = at(c, w);
    b.x = row + c * (kChunk * 2);
#pragma unroll
    for (int r = 0; r < R; ++r) w[r].template load<kTail>(b.c[r], k);
  };
  auto multiply = [&](const Step& b) {
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const bits8 x[1] = {*reinterpret_cast<lds_bits8_t*>(b.x + (threadIdx.x & 48u) + 64 * s)};
      W::template multiply<R, 1>(b.c, s, x, acc);
    }
  };
  uint32_t c = wave;
  Step now;
  if (c < n_chunks) load(now, c);
  stage();
  if (c >= n_chunks) return;
  for (; c + waves < n_chunks; c += waves) {
    Step next;
    load(next, c + waves);
    multiply(now);
    now = next;
  }
  multiply(now);
}
// A row of n values to LDS by all threads, zeros behind it up to whole chunks.
__device__ __forceinline__ void stage_row(u16* to, const u16* row, uint32_t n) {
  for (uint32_t i = threadIdx.x * 8; i < (n + kChunk - 1) / kChunk * kChunk; i += blockDim.x * 8)
    *reinterpret_cast<bits8*>(to + i) = load_end(row + i, int(n) - int(i));
}
constexpr uint32_t kStagedBytes = 64 * 1024;  // of x, at most: two workgroups a CU
inline uint64_t staged_bytes(uint32_t n) { return uint64_t(n + kChunk - 1) / kChunk * kChunk * 2; }

// The waves' sums added in their order: part[wave][i][lane], i over the wave's V vectors; thread (wave, lane) calls
// f(i, lane, sum) for i = wave, wave + waves, ... of `use` vectors.
template <int V, class F>
__device__ __forceinline__ void join_waves(f32x4* part, const f32x4 (&v)[V], uint32_t wave, uint32_t waves, F&& f) {
  const uint32_t lane = threadIdx.x & 63u;
#pragma unroll
  for (int i = 0; i < V; ++i) part[(wave * V + i) * 64 + lane] = v[i];
  __syncthreads();
  f([&](uint32_t i) {
    f32x4 s = part[i * 64 + lane];
    for (uint32_t w = 1; w < waves; ++w) s += part[(w * V + i) * 64 + lane];
    return s;
  });
}

// ---- one row of x, 4-bit rows through LDS ----
//
// A 4-bit lane's own loads are 2 and 4 bytes, 16 lines an instruction: 1.1 TB/s. Here a wave fills LDS of its own in 16-byte
// pieces (load_to_lds), a stage of 9 KiB at a time with the next one in flight: 1024 / R values of 16 rows of R parts, laid
// out as [8 blocks][row][144 bytes], and x's values of the stage behind it. Two blocks are 9 words: the first one's half
// bytes are the words q and q + 1 shifted by 16 bits, the second one's word q + 5 (q = lane / 16), the scales the low half of
// word 0 and the high half of word 4. A row's 36 words put 16 rows x 4 lanes on all banks. All 16 rows of operand a are the
// one row of x, so every result row is the same and one accumulator a part is kept. Eight experts of 7168 x 2048: gate and up
// (132 MB) 29 us, 4.6 TB/s, down (66 MB) 24 us, 2.8: bound by the stages' latency, but with a third buffer (fewer waves fit)
// both together take 68 us for 53, and loads past the caches, which split the lines that two pieces share, 56.
template <int R>
struct Q4Stage {
  static constexpr uint32_t kValues = 1024 / R, kGroups = 4 / R, kXLoads = 2 / R, kLoads = 9 + kXLoads;
  static constexpr uint32_t kBytes = kLoads * 1024, kBuffers = 2;
};

// Adds stages wave, wave + waves, .. below n_stages to acc. at(s, base, x) gives the stage's parts' first row of the tile,
// the row of x, and returns its first value k; rows: the tile's rows (up to 16), n: values of a row, a multiple of 256.
// Addresses are 16-byte aligned. lds: this wave's 2 x kBytes.
template <class T, int R, class At>
__device__ __forceinline__ void stream_q4(uint32_t n_stages, uint32_t wave, uint32_t waves, uint32_t rows, uint32_t n, uint32_t lds,
                                          At&& at, float (&acc)[R]) {
  typedef Q4Stage<R> S;
  const uint32_t lane = threadIdx.x & 63u, q = lane >> 4, row_bytes = n / kQ4Block * kQ4Bytes;
  const auto issue = [&](uint32_t s, uint32_t to) {
    const char* base[R];
    const u16* x;
    const uint32_t k = at(s, base, x);
#pragma unroll
    for (uint32_t l = 0; l < 9; ++l) {
      const uint32_t p = l * 64 + lane, piece = p % 9, row = p / 9 % (16 * R), g = p / (9 * 16 * R);
      const uint32_t r = (row & 15u) < rows ? row & 15u : rows - 1;
      const uint64_t off = uint64_t(r) * row_bytes + (k + (k + 256 * g < n ? 256 * g : 0)) / 256 * 144 + piece * 16;
      load_to_lds((R == 1 || row < 16 ? base[0] : base[R - 1]) + off, to + l * 1024);
    }
#pragma unroll
    for (uint32_t l = 0; l < S::kXLoads; ++l) {
      const uint32_t v = k + l * 512 + lane * 8;
      load_to_lds(v < n ? static_cast<const void*>(x + v) : &kZeroPiece, to + (9 + l) * 1024);
    }
  };
  typedef __attribute__((address_space(3))) const uint32_t lds_word_t;
  typedef __attribute__((address_space(3))) const bits4 lds_bits4_t;
  const auto add = [&](uint32_t from) {
    for (uint32_t g = 0; g < S::kGroups; ++g)
#pragma unroll
      for (uint32_t pair = 0; pair < 4; ++pair) {
        bits8 x[2];
        f32x4 off[2];
        constexpr u16 m = HalfBytes<T>::kMinus;
#pragma unroll
        for (uint32_t b = 0; b < 2; ++b) {
          const uint32_t xa = from + 9216 + (g * 256 + pair * 64 + b * 32 + q * 4) * 2;
          const bits4 lo = *reinterpret_cast<lds_bits4_t*>(xa), hi = *reinterpret_cast<lds_bits4_t*>(xa + 32);
          x[b] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
          off[b] = T::mfma(x[b], bits8{m, m, m, m, m, m, m, m}, f32x4{0, 0, 0, 0});
        }
#pragma unroll
        for (uint32_t r = 0; r < R; ++r) {
          lds_word_t* w = reinterpret_cast<lds_word_t*>(from + ((g * R + r) * 16 + (lane & 15u)) * 144 + pair * 36);
          const uint32_t w0 = w[q], w1 = w[q + 1], w5 = w[q + 5], s0 = w[0], s1 = w[4];
          const f32x4 even = T::mfma(x[0], HalfBytes<T>::unpack(__builtin_amdgcn_alignbit(w1, w0, 16)), off[0]);
          const f32x4 odd = T::mfma(x[1], HalfBytes<T>::unpack(w5), off[1]);
          acc[r] += F16::up(u16(s0)) * even[0];
          acc[r] += F16::up(u16(s1 >> 16)) * odd[0];
        }
      }
  };
  if (wave >= n_stages) return;
  issue(wave, lds);
  uint32_t now = 0;
  for (uint32_t s = wave; s < n_stages; s += waves) {
    if (s + waves < n_stages) {
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the reads of the buffer that is filled now
      issue(s + waves, lds + (now ^ 1) * S::kBytes);
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"(S::kLoads) : "memory");
    } else {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }
    add(lds + now * S::kBytes);
    now ^= 1;
  }
}

constexpr uint32_t kQ4Waves = 7;  // what LDS holds
// Waves per workgroup: enough for 4 a CU. Eight 24.8 MB experts, gate and up (1024 workgroups): 32 us with one wave each, 37 with
// two, 44 with four; down (448 workgroups): 39, 29, 25.5 and 27.6 us with one, two, three and four.
inline uint32_t q4_waves(uint64_t workgroups, uint64_t stages) {
  uint64_t w = (1024 + workgroups - 1) / workgroups;
  if (w > kQ4Waves) w = kQ4Waves;
  return uint32_t(w < stages ? w : stages);
}

// The waves' sums added in their order, by wave 0: lanes 0..15 call f(acc of the tile's row lane).
template <int R, class F>
__device__ __forceinline__ void join_q4(float* part, const float (&acc)[R], uint32_t wave, uint32_t waves, F&& f) {
  const uint32_t lane = threadIdx.x & 63u;
  if (lane < 16)
#pragma unroll
    for (int r = 0; r < R; ++r) part[(wave * R + r) * 16 + lane] = acc[r];
  __syncthreads();
  if (wave != 0 || lane >= 16) return;
  float s[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    s[r] = part[r * 16 + lane];
    for (uint32_t w = 1; w < waves; ++w) s[r] += part[(w * R + r) * 16 + lane];
  }
  f(s);
}

// The registers of CT tiles of x bound the waves of a workgroup.
constexpr uint32_t most_waves(int CT) { return CT == 1 ? 16 : CT == 2 ? 8 : 4; }

// Waves per workgroup: enough that the launch has about 8 a CU (256 CUs), at least 2 chunks each, a power of two.
inline uint32_t stream_waves(uint64_t workgroups, uint64_t chunks, uint32_t most) {
  uint32_t w = 4;
  while (w < most && workgroups * w < 2048) w *= 2;
  while (w > 1 && w * 2 > chunks) w /= 2;
  return w;
}
inline uint32_t chunks_of(uint32_t n) { return (n + kChunk - 1) / kChunk; }

}  // namespace op
}  // namespace tsa
