// Attention of new tokens over the pages of their requests, keys and values of 4 bits.
//
// A workgroup takes 16 query rows that share a kept head (a request's new tokens x the heads of its group) and a stretch of the
// request's pages; its four waves take pages in turn, each with the running maximum and sum of its softmax, and join at the end. All
// requests' pages are cut into equal shares, as many as workgroups work at once, so that no request's length sets the time (cut into runs
// of one request each, a few more runs than workgroups took twice the time); what falls into several is joined by a second
// launch. The cuts follow on the device from the lengths, of which the host needs to know none.
//
// A page is one contiguous piece per head and goes straight to LDS, one page ahead. Scores are S^T = K Q^T and outputs O^T = V^T P^T
// by v_mfma_f32_16x16x32: then a lane's column is its query row in both, its scores are what the second product takes as its other
// operand, and nothing is exchanged between lanes but the maximum. Half bytes become 16-bit numbers with their bits put behind a fixed
// exponent, exactly; the offset is taken off by the product's own accumulator (keys) and by a product with a constant (values). A key
// block's scale multiplies its 32-value product in 32 bits; a value's scale multiplies its probability, and the product is rounded to half
// precision whatever the type: once for half precision; for bf16 both factors are rounded before, which takes half the instructions and
// leaves a fifth of the error of one rounding to bf16. Their ranges are kept by powers of two: probabilities go up to 2^11, a block's scales
// up to 2^4 by what the largest so far in the wave's pages asks for. A scale below 2^-15 of the largest of its block keeps fewer
// bits, and so does a probability below 2^-17 of its row's largest. Values are read transposed, by ds_read_b64_tr_b4.
//
// Measured, 128 values a head: 64 requests of 1023..8191 tokens, 180 MB of pages, 46 us and 4.5 for the joining launch (3.9 TB/s; the
// loads alone take 36); four of up to 131071, three new tokens each, 371 MB, 75 to 81 and 6 (4.6 to 4.9 TB/s; 70); one of 4097 tokens, 9 and 4. What bounds
// it: the rate of the loads, and for short shares the way to the first page (lengths, then the table and queries, then the page) and the joining
// of the waves, 10 us or so together. The registers leave three workgroups a CU at 96 and 128 values a head: one spilled value costs 3 us.
#include <cmath>
#include <limits>

#include "attn_device.hpp"

namespace tsa {
namespace op {
namespace {

constexpr uint32_t kWaves = 4, kRows = 16;  // waves and query rows of a workgroup
// Workgroups of a CU that the registers leave room for, and of the chip.
constexpr uint32_t per_cu(uint32_t head_dim) { return head_dim <= 64 ? 4 : 3; }
constexpr uint32_t groups(uint32_t head_dim) { return 256 * per_cu(head_dim); }

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef int i32x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) i32x2 lds_i32x2_t;
typedef __attribute__((address_space(3))) const u32x4 lds_words_t;
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) const u32x2 lds_two_words_t;
typedef __attribute__((address_space(3))) const uint32_t lds_word_t;
typedef __attribute__((address_space(3))) u16 lds_half_t;

struct CachedShape {
  uint32_t group;     // query heads of a kept one
  uint32_t shares;    // workgroups of a kept head, at most
  float c;            // |scale| / ln 2, more than 0: masked scores are -inf before it
  uint32_t flip;      // the sign bits of two queries where the scale is negative
  bool aligned;       // q and out in pieces of 8
};

// ---- who does what --------------------------------------------------------------------------------------------------------
// All requests' tiles of 16 query rows, one behind the other, each with the rounds that its pages make for four waves (one at least), are one row
// of rounds. It is cut into equal shares, a workgroup each, wherever the cuts fall (cut by pages, a wave more had the last one alone). A tile inside one share is written at once; a share's piece of any
// other is left in the workspace: at place 0 of the share where it begins with the share, at place 1 where it begins inside. For each
// tile that begins in it a share also leaves where its pieces are.

// Request i's new tokens, the tokens it ends with, its tiles and their pages, of which the waves take one each a round.
struct Request {
  uint32_t first, fresh, tiles, pages;
  int32_t end;
  Request() = default;
  __device__ __forceinline__ Request(const tsa_attend_cached_args& a, uint32_t i, uint32_t group) {
    const Span s = span_of(a.first, i, a.tokens);
    first = s.begin, fresh = s.count;
    tiles = (fresh * group + kRows - 1) / kRows;
    end = max(0, min(a.ends[i], int32_t(a.width * kPage)));  // (width is below 2^25)
    pages = (uint32_t(end) + kPage - 1) / kPage;
  }
  __device__ __forceinline__ uint32_t rounds() const { return pages ? (pages + kWaves - 1) / kWaves : 1; }
};

struct Place {
  uint32_t share, all;  // rounds of a share and of all
  uint32_t at;          // first round of the tile
  uint32_t request, tile;
  Request r;
};
struct PlaceMemory {
  uint32_t pages[kWaves];
  Place found;
};
// Where a tile's pieces are: its rounds of all, and the rounds of a share. end 0: it is whole.
struct Pieces {
  uint32_t at, end, share;
};
// A request's first place in a list of all tiles that no tiles need to be counted for: it leaves one empty now and then. A request has
// fresh * group / 16 tiles, and one more at most.
__device__ __forceinline__ uint32_t tile_place(uint32_t request, uint32_t first, uint32_t group) { return request + uint32_t(uint64_t(first) * group / kRows); }

__device__ __forceinline__ uint32_t lanes_up_to(uint32_t v) {
#pragma unroll
  for (uint32_t s = 1; s < 64; s <<= 1) {
    const uint32_t o = __shfl_up(v, s, 64);
    if ((threadIdx.x & 63u) >= s) v = add_sat(v, o);
  }
  return v;
}

// The tile that holds the first round of share `want`. By the whole workgroup; false: there is none. Of requests that follow each
// other all rounds are below 2^31; spans that overlap (first not ascending) may have more than 32 bits count, which the sums keep to: then
// there is none either.
__device__ __forceinline__ bool find_place(const tsa_attend_cached_args& a, const CachedShape& s, uint32_t want, PlaceMemory& m, Place& out) {
  const uint32_t t = threadIdx.x, lane = t & 63u, wave = t >> 6, per = (a.requests + 64 * kWaves - 1) / (64 * kWaves);
  const uint32_t i0 = min(t * per, a.requests), i1 = min(i0 + per, a.requests);
  uint32_t pages = 0;
  Request r;  // (the last one stays: with up to 256 requests none is read twice)
  for (uint32_t i = i0; i < i1; ++i) {
    r = Request(a, i, s.group);
    pages = add_sat(pages, r.tiles * r.rounds());  // (a request's own are below 2^31)
  }
  const uint32_t upto = lanes_up_to(pages);
  if (lane == 63) m.pages[wave] = upto;
  __syncthreads();
  Place p = {};
  uint32_t page0 = upto - pages;
#pragma unroll
  for (uint32_t w = 0; w < kWaves; ++w) {
    p.all = add_sat(p.all, m.pages[w]);
    if (w < wave) page0 += m.pages[w];
  }
  if (p.all >> 31) return false;
  const uint32_t even = p.all / s.shares + (p.all % s.shares != 0);
  p.share = even;
  const uint64_t page = uint64_t(want) * p.share;  // (past all of them, perhaps by far)
  if (page >= p.all) return false;
  if (page >= page0 && page < page0 + pages) {
    for (uint32_t i = i0; i < i1; ++i) {
      if (i1 - i0 > 1) r = Request(a, i, s.group);
      const uint32_t have = r.tiles * r.rounds();
      if (page < page0 + have) {
        p.request = i;
        p.tile = uint32_t(page - page0) / r.rounds();
        p.at = page0 + p.tile * r.rounds();
        p.r = r;
        m.found = p;
        break;
      }
      page0 += have;
    }
  }
  __syncthreads();
  // (the same in every lane, which the compiler is to know)
  struct Words { uint32_t w[sizeof(Place) / 4]; } words = __builtin_bit_cast(Words, m.found);
#pragma unroll
  for (uint32_t& w : words.w) w = __builtin_amdgcn_readfirstlane(w);
  out = __builtin_bit_cast(Place, words);
  return true;
}

// ---- numbers of 4 bits ----------------------------------------------------------------------------------------------------
// The half bytes 0, 4, 1, 5, 2, 6, 3, 7 of a word as 16-bit numbers, each with an offset that its place in the word suits: keys in bf16
// n + 128, in half precision n + 16; values, whose products with probabilities are rounded already, n + 1024 where they lie in the low bits and n + 64
// where they lie four higher, which leaves one shift a word.
// The constants are kept in registers: as literals each would take an instruction of its own.
struct Numbers16 {  // keys, bf16
  uint32_t mask = 0x000F000Fu, one = 0x43004300u;
  __device__ __forceinline__ Numbers16() { asm("" : "+s"(mask), "+v"(one)); }
  __device__ __forceinline__ bits8 of(uint32_t x) const {
    return __builtin_bit_cast(bits8, u32x4{(x & mask) | one, ((x >> 4) & mask) | one, ((x >> 8) & mask) | one, ((x >> 12) & mask) | one});
  }
};
struct NumbersHalf {  // values
  uint32_t low = 0x000F000Fu, high = 0x00F000F0u, one_low = 0x64006400u, one_high = 0x54005400u;
  __device__ __forceinline__ NumbersHalf() { asm("" : "+s"(low), "+s"(high), "+v"(one_low), "+v"(one_high)); }
  __device__ __forceinline__ bits8 of(uint32_t x) const {
    const uint32_t y = x >> 8;
    return __builtin_bit_cast(bits8, u32x4{(x & low) | one_low, (x & high) | one_high, (y & low) | one_low, (y & high) | one_high});
  }
};
// Keys beside queries of half precision: three shifts a word more than with the values' offsets (long requests 83 us for 82), but a score is what is
// left of a sum in which the offset outweighs it a few times, not some hundred times, and what 32 bits lose of it grows with that: of scores around 900
// the worst row was off by 0.0034, now 0.0004, which is its own rounding.
struct KeysHalf {
  uint32_t mask = 0x03C003C0u, one = 0x4C004C00u;
  __device__ __forceinline__ KeysHalf() { asm("" : "+s"(mask), "+v"(one)); }
  __device__ __forceinline__ bits8 of(uint32_t x) const {
    return __builtin_bit_cast(bits8, u32x4{((x << 6) & mask) | one, ((x << 2) & mask) | one, ((x >> 2) & mask) | one, ((x >> 6) & mask) | one});
  }
};
// What stands for 0 at the eight places, less.
template <class N>
constexpr bits8 kZero = {0xC308, 0xC308, 0xC308, 0xC308, 0xC308, 0xC308, 0xC308, 0xC308};
template <>
constexpr bits8 kZero<KeysHalf> = {0xCE00, 0xCE00, 0xCE00, 0xCE00, 0xCE00, 0xCE00, 0xCE00, 0xCE00};
template <>
constexpr bits8 kZero<NumbersHalf> = {0xE408, 0xE408, 0xD480, 0xD480, 0xE408, 0xE408, 0xD480, 0xD480};

// The larger of a value in the four lanes of a column.
__device__ __forceinline__ float column_max(float v) {
  v = fmaxf(v, __shfl_xor(v, 16, 64));
  return fmaxf(v, __shfl_xor(v, 32, 64));
}
__device__ __forceinline__ float column_sum(float v) {
  v += __shfl_xor(v, 16, 64);
  return v + __shfl_xor(v, 32, 64);
}

// Keeps what stands before it in the program before what stands behind it.
__device__ __forceinline__ void in_order() { __builtin_amdgcn_sched_barrier(0); }

// ---- the pages --------------------------------------------------------------------------------------------------------------
// A page of a head in memory, and in LDS, where the scales have room for whole loads.
template <int NB>
struct Page {
  static constexpr uint32_t kBytes = 2304 * NB, kKeyScalesAt = 1024 * NB, kValueScalesAt = 1152 * NB, kValuesAt = 1280 * NB;
  static constexpr uint32_t kScaleLoads = (NB + 1) / 2, kKeyLoads = NB + 2 * kScaleLoads, kValueLoads = NB;  // (all scales come with the keys)
  static constexpr uint32_t kKeyScales = 1024 * NB, kScaleRoom = 256 * kScaleLoads, kValueScales = kKeyScales + kScaleRoom,  // (two pages' of the values)
                            kValues = kValueScales + 2 * kScaleRoom, kRoom = kValues + 1024 * NB;
};

// kMany loads of 64 x 16 (64 x 4) bytes to LDS, behind each other there as in memory: the instruction's offset counts for both.
template <uint32_t kMany>
__device__ __forceinline__ void pieces_to_lds(const void* g, uint32_t at) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(g), "s"(at) : "memory", "m0");
  if constexpr (kMany > 1) asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off offset:1024" ::"v"(g), "s"(at) : "memory", "m0");
  if constexpr (kMany > 2) asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off offset:2048" ::"v"(g), "s"(at) : "memory", "m0");
  if constexpr (kMany > 3) asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off offset:3*1024" ::"v"(g), "s"(at) : "memory", "m0");
}
template <uint32_t kMany>
__device__ __forceinline__ void words_to_lds(const void* g, uint32_t at) {
  static_assert(kMany <= 2);
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off" ::"v"(g), "s"(at) : "memory", "m0");
  if constexpr (kMany > 1) asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off offset:256" ::"v"(g), "s"(at) : "memory", "m0");
}
__device__ __forceinline__ void reads_done() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }
template <int N>
__device__ __forceinline__ void loads_left() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }

// The scales of four tokens, from LDS.
template <int NB>
struct Scales {
  uint32_t w[2 * NB];
  Scales() = default;
  explicit __device__ __forceinline__ Scales(uint32_t lds) {
    if constexpr (NB % 2 == 0) {
#pragma unroll
      for (int i = 0; i < NB / 2; ++i) {
        const u32x4 v = reinterpret_cast<lds_words_t*>(lds)[i];
#pragma unroll
        for (int k = 0; k < 4; ++k) w[4 * i + k] = v[k];
      }
    } else {  // (8-byte aligned)
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        const u32x2 v = reinterpret_cast<lds_two_words_t*>(lds)[i];
        w[2 * i] = v[0], w[2 * i + 1] = v[1];
      }
    }
  }
  __device__ __forceinline__ float at(uint32_t token, uint32_t block) const {
    const uint32_t i = token * NB + block;
    return F16::up(u16(w[i / 2] >> (16 * (i & 1u))));
  }
};

// The powers of two that take the values' scales of a wave's pages to 2^4 and below, a block's each.
template <int NB>
struct ScaleRange {
  uint32_t down[NB];  // the bits of 2^(1 - e), for a largest scale of 2^e and above when it was last followed
  uint32_t most[NB];  // the bits of the largest scale that this holds for
  __device__ __forceinline__ ScaleRange() {
#pragma unroll
    for (int b = 0; b < NB; ++b) down[b] = 127u << 23, most[b] = 0;
  }
  __device__ __forceinline__ float up(int b) const { return __builtin_bit_cast(float, (254u << 23) - down[b]); }
  // A token's scales; whether the page has larger ones than those so far.
  __device__ __forceinline__ bool passed(const uint32_t (&scale)[NB]) const {
    bool over = false;
#pragma unroll
    for (int b = 0; b < NB; ++b) over = over || size(scale[b]) > most[b];
    return __any(over);
  }
  // Takes them in: what an output of the old range is multiplied by.
  __device__ __forceinline__ float follow(int b, uint32_t scale) {
    uint32_t top = size(scale);
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) top = max(top, uint32_t(__shfl_xor(int(top), s, 64)));
    top = __builtin_amdgcn_readfirstlane(top);
    const uint32_t e = __builtin_bit_cast(uint32_t, F16::up(u16(top))) >> 23;  // (of 32 bits: biased by 127)
    const bool more = top > most[b];
    const float before = up(b);
    down[b] = __builtin_amdgcn_readfirstlane(more ? (255u - e) << 23 : down[b]);
    most[b] = __builtin_amdgcn_readfirstlane(more ? uint32_t(F16::down(fminf(__builtin_bit_cast(float, (e + 3u) << 23), 65504.0f))) : most[b]);
    return before * __builtin_bit_cast(float, down[b]);
  }
  __device__ __forceinline__ u16 fit(int b, uint32_t scale) const { return F16::down(F16::up(u16(scale)) * __builtin_bit_cast(float, down[b])); }

 private:
  static __device__ __forceinline__ uint32_t size(uint32_t scale) {
    const uint32_t s = scale & 0x7FFFu;
    return s < 0x7C00u ? s : 0;  // (no number stays none)
  }
};

template <class T, int NB>
__global__ __launch_bounds__(64 * kWaves, per_cu(32 * NB)) void cached_kernel(tsa_cache c, tsa_attend_cached_args a, CachedShape s, float* parts, float2* stats, Pieces* pieces) {
  typedef Page<NB> P;
  constexpr bool kHalf = std::is_same_v<T, F16>;
  constexpr uint32_t D = 32 * NB;
  __shared__ __attribute__((aligned(16))) unsigned char page_s[kWaves][P::kRoom];
  __shared__ __attribute__((aligned(16))) u16 query_s[kRows][D + 4];  // (rows apart by banks)
  __shared__ float2 stat_s[kWaves][kRows];
  __shared__ PlaceMemory place_s;
  constexpr uint32_t kOutRow = D + 4;  // (rows apart by banks)
  static_assert(P::kRoom >= kRows * kOutRow * 4, "a wave's outputs take its page's place");
  Place at;
  const uint32_t kept = blockIdx.x % c.kv_heads, share = blockIdx.x / c.kv_heads;
  if (!find_place(a, s, share, place_s, at)) return;
  const uint32_t from = share * at.share, upto = min(from + at.share, at.all);  // this share's rounds
  const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4;
  const uint32_t lds = __builtin_amdgcn_readfirstlane(lds_offset(page_s[wave]));
  typedef std::conditional_t<kHalf, KeysHalf, Numbers16> KeyNumbers;
  const KeyNumbers keys;
  const NumbersHalf values;
  const bits8 zero = kZero<NumbersHalf>;
  Request r = at.r;
  while (true) {  // the share's tiles
    const uint32_t x = at.tile * kRows + (lane & 15u);
    const bool on = x < r.fresh * s.group;
    const uint32_t token = on ? x / s.group : 0;
    const int32_t limit = on ? r.end - int32_t(r.fresh) + int32_t(token) + 1 : 0;  // keys that this row attends to
    const int32_t whole = r.end - int32_t(r.fresh) + 1;                            // keys that every row attends to

    // The queries, once for all waves (each by itself, value by value, took 9 us), on their way with the list of pages. Pieces of 8 where
    // they start 16-byte aligned.
    constexpr uint32_t kPieces = kRows * D / 8;
    static_assert(kPieces <= 64 * kWaves, "a piece a thread");
    bits8 piece = {0, 0, 0, 0, 0, 0, 0, 0};
    uint32_t t = threadIdx.x;
    asm volatile("" : "+v"(t));  // (what follows from it is made again for each tile: kept over the pages' loop, it took the last registers)
    const uint32_t piece_row = t / (D / 8), piece_at = t % (D / 8) * 8;
    if (const uint32_t y = at.tile * kRows + piece_row; t < kPieces && y < r.fresh * s.group) {
      const u16* p = row_of<u16>(a.q, r.first + y / s.group, kept * s.group + y % s.group) + piece_at;
      if (s.aligned) {
        piece = *reinterpret_cast<const bits8*>(p);
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) piece[k] = p[k];
      }
    }
    const uint32_t begin = (max(from, at.at) - at.at) * kWaves, end = min(r.pages, (upto - at.at) * kWaves);
    const int32_t* table = a.table + uint64_t(at.request) * a.table_stride;
    // Half a page to LDS, keys with all scales or values. While the keys of one are multiplied its values are on their way, and while these are
    // the next page's keys: one buffer is enough for that (the values' scales, read to the end, have two), and three or four workgroups fit a CU.
    auto page_at = [&](uint32_t page) { return static_cast<const unsigned char*>(c.pages) + (uint64_t(page) * c.kv_heads + kept) * P::kBytes; };
    auto fetch_keys = [&](uint32_t page, uint32_t scales) {
      const unsigned char *at = page_at(page), *words = at + P::kKeyScalesAt + lane * 4;
      pieces_to_lds<NB>(at + lane * 16, lds);
      if constexpr (NB % 2 == 0) {
        words_to_lds<NB / 2>(words, lds + P::kKeyScales);
        words_to_lds<NB / 2>(words + (P::kValueScalesAt - P::kKeyScalesAt), scales);
      } else {
#pragma unroll
        for (uint32_t i = 0; i < P::kScaleLoads; ++i) {  // (what the last half load is too much stays in its room)
          const uint32_t from = min(i * 256 + lane * 4, 128u * NB - 4);
          load_words_to_lds(at + P::kKeyScalesAt + from, lds + P::kKeyScales + i * 256);
          load_words_to_lds(at + P::kValueScalesAt + from, scales + i * 256);
        }
      }
    };
    auto fetch_values = [&](uint32_t page) { pieces_to_lds<NB>(page_at(page) + P::kValuesAt + lane * 16, lds + P::kValues); };
    // this wave's pages, 64 in the lanes at a time (a load in the loop would wait for the pages behind it), absent ones left out
    uint32_t ids = 0, p = begin + wave, turn = 0;
    auto page_here = [&]() {
      for (; p < end; p += kWaves, ++turn) {
        if (turn % 64 == 0) {
          const uint64_t mine = uint64_t(p) + lane * kWaves;
          ids = mine < end ? uint32_t(table[mine]) : ~0u;
        }
        const uint32_t page = uint32_t(__builtin_amdgcn_readlane(ids, turn % 64));
        if (page < c.n_pages) return page;
      }
      return ~0u;
    };
    uint32_t page = page_here();
    uint32_t value_scales = lds + P::kValueScales, next_scales = value_scales + P::kScaleRoom;
    if (t < kPieces) {
      const u32x4 w = __builtin_bit_cast(u32x4, piece) ^ s.flip;
      *reinterpret_cast<uint2*>(&query_s[piece_row][piece_at]) = uint2{w[0], w[1]};
      *reinterpret_cast<uint2*>(&query_s[piece_row][piece_at + 4]) = uint2{w[2], w[3]};
    }
    if (p < end) {
      fetch_keys(page, value_scales);
      fetch_values(page);
    }
    __syncthreads();
    // this row's, in the order of the keys' half bytes
    bits8 q[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      const bits4 lo = *reinterpret_cast<const bits4*>(&query_s[lane & 15u][32 * b + 4 * g]), hi = *reinterpret_cast<const bits4*>(&query_s[lane & 15u][32 * b + 16 + 4 * g]);
      q[b] = bits8{lo[0], lo[2], hi[0], hi[2], lo[1], lo[3], hi[1], hi[3]};
    }

    f32x4 o[2 * NB];
#pragma unroll
    for (int i = 0; i < 2 * NB; ++i) o[i] = f32x4{0, 0, 0, 0};
    float top = -INFINITY, total = 0.0f;
    ScaleRange<NB> range;

    while (p < end) {
      const int32_t key0 = int32_t(p * kPage);
      const bool edge = key0 + int32_t(kPage) > whole;
      p += kWaves, ++turn;
      page = page_here();  // the next one
      const bool more = p < end;
      loads_left<P::kValueLoads>();
      // Tokens that not every row attends to must not reach the others through 0 x NaN: behind the last key the values' scales become 0;
      // before it one that is no number becomes 0 and its key's scale NaN, which reaches only the rows that attend to it.
      if (edge && key0 + int32_t(lane) >= whole) {
#pragma unroll
        for (uint32_t b = 0; b < NB; ++b) {
          lds_half_t* const scale = reinterpret_cast<lds_half_t*>(value_scales + (lane * NB + b) * 2);
          const bool none = (*scale & 0x7C00u) == 0x7C00u;
          if (none) *reinterpret_cast<lds_half_t*>(lds + P::kKeyScales + (lane * NB + b) * 2) = 0x7E00;
          if (none || key0 + int32_t(lane) >= r.end) *scale = 0;
        }
      }

      // the values' scales, a token's a lane, into their range and the order of a lane's eight
      uint32_t mine[NB];
      const uint32_t place = (lane & 32u) | (lane >> 2 & 3u) << 3 | (lane >> 4 & 1u) << 2 | (lane & 3u);
#pragma unroll
      for (int b = 0; b < NB; ++b) mine[b] = reinterpret_cast<lds_half_t*>(value_scales + lane * 2 * NB)[b];
      const bool moved = range.passed(mine);
      float by[NB];
#pragma unroll
      for (int b = 0; b < NB; ++b) by[b] = 1.0f;
      if (moved) {
#pragma unroll
        for (int b = 0; b < NB; ++b) by[b] = range.follow(b, mine[b]);
      }
#pragma unroll
      for (int b = 0; b < NB; ++b) reinterpret_cast<lds_half_t*>(value_scales)[64 * b + place] = range.fit(b, mine[b]);

      // scores: tile j holds tokens 16 j + 4 g + 0..3 of this lane's row
      f32x4 score[4], off[NB];
      bits8 key_zero = kZero<KeyNumbers>;
      asm volatile("" : "+v"(key_zero));  // (what takes the offsets off is made again for each page: kept, it took 16 registers)
#pragma unroll
      for (int b = 0; b < NB; ++b) off[b] = T::mfma(key_zero, q[b], f32x4{0, 0, 0, 0});
      typedef uint32_t row_words __attribute__((ext_vector_type(NB)));
      row_words words[4];
      Scales<NB> scale[4];
      auto read = [&](uint32_t j) {
        const uint32_t key = lds + (16 * j + (lane & 15u)) * 16 * NB + g * 4 * NB;
        if constexpr (NB == 3) {  // (4-byte aligned)
#pragma unroll
          for (int b = 0; b < NB; ++b) words[j][b] = reinterpret_cast<lds_word_t*>(key)[b];
        } else {
          words[j] = *reinterpret_cast<__attribute__((address_space(3))) const row_words*>(key);
        }
        scale[j] = Scales<NB>(lds + P::kKeyScales + (16 * j + 4 * g) * 2 * NB);
      };
      // (reads are kept a step ahead: left to itself the compiler puts each in front of its use, and the wave waits out every one)
      read(0);
#pragma unroll
      for (uint32_t j = 0; j < 4; ++j) {
        if (j + 1 < 4) read(j + 1);
        in_order();
        f32x4 sum = {0, 0, 0, 0};
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          const f32x4 v = T::mfma(keys.of(words[j][b]), q[b], off[b]);
#pragma unroll
          for (uint32_t k = 0; k < 4; ++k) sum[k] = __builtin_fmaf(scale[j].at(k, b), v[k], sum[k]);
        }
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k) score[j][k] = sum[k];
      }
      if (edge) {
        asm volatile("" : "+v"(score[0]), "+v"(score[1]), "+v"(score[2]), "+v"(score[3]));  // (kept out of the other pages' way)
        const int32_t left = limit - key0 - int32_t(4 * g);
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j)
#pragma unroll
          for (uint32_t k = 0; k < 4; ++k)
            if (int32_t(16 * j + k) >= left) score[j][k] = -INFINITY;
      }

      reads_done();
      if (more) fetch_keys(page, next_scales);

      // the running maximum: followed only where it is passed by 2^8 (probabilities are then up to 2^8, and go to half
      // precision another 2^3 larger: times a scale they stay below 2^15, and small ones keep their bits)
      float most = -INFINITY;
#pragma unroll
      for (uint32_t j = 0; j < 4; ++j)
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k) most = fmaxf(most, score[j][k]);
      most *= s.c;
      const bool grown = __any(most > top + 8.0f);
      float keep = 1.0f;
      if (grown) {
        const float up = fmaxf(column_max(most), top);
        keep = top == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(top - up);
        top = up;
        total *= keep;
      }
      const float base = top == -INFINITY ? 0.0f : top - 3.0f;
#pragma unroll
      for (uint32_t j = 0; j < 4; ++j)
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k) {
          score[j][k] = __builtin_amdgcn_exp2f(__builtin_fmaf(score[j][k], s.c, -base));
          total += score[j][k];
        }

      half8 weight[2];  // probabilities
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 8; ++i) weight[t][i] = _Float16(score[2 * t + i / 4][i % 4]);
      // row i of the transposed read is lane i's token, of both halves of a block: a word of the result holds, in the order of Numbers, the
      // lane's eight tokens of one column
      const uint32_t i16 = lane & 15u, e = ((i16 & 3u) << 1) | ((i16 >> 2) & 1u);
      const uint32_t row = (e < 4 ? 4 * g + e : 16 + 4 * g + e - 4) * 16 + 8 * (i16 >> 3);

      if (grown || moved) {
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          o[2 * b] *= keep * by[b];
          o[2 * b + 1] *= keep * by[b];
        }
      }
      if (more) loads_left<P::kKeyLoads>();
      else loads_left<0>();
      // outputs, 32 tokens a step; a lane's eight are tiles 2 t and 2 t + 1
      i32x2 value[2 * NB];
      half8 by_scale[2 * NB];
      auto read_value = [&](uint32_t i) {
        const uint32_t t = i / NB, b = i % NB;
        value[i] = __builtin_amdgcn_ds_read_tr4_b64_v2i32(reinterpret_cast<lds_i32x2_t*>(lds + P::kValues + b * 1024 + t * 512 + row));
        by_scale[i] = *reinterpret_cast<__attribute__((address_space(3))) const half8*>(value_scales + (64 * b + 32 * t + 8 * g) * 2);
      };
      read_value(0);
#pragma unroll
      for (uint32_t i = 0; i < 2 * NB; ++i) {
        if (i + 1 < 2 * NB) read_value(i + 1);
        in_order();
        const uint32_t b = i % NB;
        half8 w;
        if constexpr (kHalf) {
#pragma unroll
          for (uint32_t k = 0; k < 8; ++k) w[k] = _Float16(__builtin_fmaf(score[2 * (i / NB) + k / 4][k % 4], float(by_scale[i][k]), 0.0f));
        } else {
          w = weight[i / NB] * by_scale[i];
        }
        const bits8 p16 = __builtin_bit_cast(bits8, w);
#pragma unroll
        for (uint32_t h = 0; h < 2; ++h) o[2 * b + h] = F16::mfma(zero, p16, o[2 * b + h]);
#pragma unroll
        for (uint32_t h = 0; h < 2; ++h) o[2 * b + h] = F16::mfma(values.of(uint32_t(value[i][h])), p16, o[2 * b + h]);
      }
      reads_done();
      if (more) fetch_values(page);
      const uint32_t other = value_scales;
      value_scales = next_scales, next_scales = other;
    }

    // the waves' parts together
    t = threadIdx.x;
    asm volatile("" : "+v"(t));
    const uint32_t row = t & 15u, quarter = (t >> 4) & 3u;
    total = column_sum(total);
    if ((t & 63u) < kRows) stat_s[wave][row] = {top, total};
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __syncthreads();  // every wave is done with its pages
    float best = -INFINITY, sum = 0.0f;
#pragma unroll
    for (uint32_t w = 0; w < kWaves; ++w) best = fmaxf(best, stat_s[w][row].x);
    const float base = best == -INFINITY ? 0.0f : best;
#pragma unroll
    for (uint32_t w = 0; w < kWaves; ++w) {
      const float2 st = stat_s[w][row];
      sum += st.y * __builtin_amdgcn_exp2f(st.x - base);
    }
    const bool whole_tile = at.at >= from && at.at + r.rounds() <= upto;
    const float by = __builtin_amdgcn_exp2f(top - base) * (!whole_tile ? 1.0f : sum == 0.0f ? 0.0f : 1.0f / sum);
    float* mine = reinterpret_cast<float*>(page_s[wave]) + row * kOutRow;
#pragma unroll
    for (int i = 0; i < 2 * NB; ++i)
#pragma unroll
      for (uint32_t k = 0; k < 4; ++k)  // column 4 g + k of the tile: byte (4 g + k) / 2 of the half block, low half bytes first
        mine[32 * (i / 2) + 8 * (i % 2) + (4 * quarter + k) / 2 + 16 * (k & 1u)] = o[i][k] * (by * range.up(i / 2));
    __syncthreads();
    const uint32_t part = (2 * share + (at.at > from)) * c.kv_heads + kept;
    if (t == 0 && at.at >= from)
      pieces[uint64_t(tile_place(at.request, r.first, s.group) + at.tile) * c.kv_heads + kept] = {at.at, whole_tile ? 0 : at.at + r.rounds(), at.share};
    if (!whole_tile && t < kRows) stats[part * kRows + t] = {best, sum};
    for (uint32_t i = t; i < kRows * D / 4; i += 64 * kWaves) {
      const uint32_t y = at.tile * kRows + i / (D / 4), d = i % (D / 4) * 4;
      if (y >= r.fresh * s.group) break;
      f32x4 v = {0, 0, 0, 0};
#pragma unroll
      for (uint32_t w = 0; w < kWaves; ++w) v += *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(page_s[w]) + i / (D / 4) * kOutRow + d);
      if (!whole_tile) {
        reinterpret_cast<f32x4*>(parts)[uint64_t(part) * (kRows * D / 4) + i] = v;
        continue;
      }
      u16* out = const_cast<u16*>(row_of<u16>(a.out, r.first + y / s.group, kept * s.group + y % s.group)) + d;
      const bits4 w = {T::down(v[0]), T::down(v[1]), T::down(v[2]), T::down(v[3])};
      if (s.aligned) {
        *reinterpret_cast<bits4*>(out) = w;
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) out[k] = w[k];
      }
    }
    at.at += r.rounds();
    if (at.at >= upto) break;
    ++at.tile;
    while (at.tile >= r.tiles) {
      if (++at.request >= a.requests) return;  // (lengths that change meanwhile)
      r = Request(a, at.request, s.group);
      at.tile = 0;
    }
    __syncthreads();  // the outputs are read, pages take their place again
  }
}

// Sums of exponentials with their maxima: (best, total, sum) and another's.
__device__ __forceinline__ void add(float& best, float& total, f32x4& sum, float top, float more, f32x4 v) {
  const float up = fmaxf(best, top), base = up == -INFINITY ? 0.0f : up;
  const float a = __builtin_amdgcn_exp2f(best - base), b = __builtin_amdgcn_exp2f(top - base);
  best = up;
  total = total * a + more * b;
  sum = sum * a + v * b;
}

// The pieces of a tile together. kAtOnce groups of threads take a row or a part of one's pieces each, four values a thread: as many groups a
// row as leave each four pieces at most.
template <class T, int NB>
__global__ __launch_bounds__(64 * kWaves) void join_kernel(tsa_cache c, tsa_attend_cached_args a, CachedShape s, const float* parts, const float2* stats, const Pieces* pieces) {
  constexpr uint32_t D = 32 * NB, kLanes = D / 4, kAtOnce = 64 * kWaves / kLanes;
  __shared__ f32x4 sum_s[kAtOnce][kLanes];
  __shared__ float2 stat_s[kAtOnce];
  __shared__ uint32_t found_s;
  // whose tile this is: the request by stretches of requests first, then inside one
  auto place = [&](uint32_t i) { return tile_place(i, uint32_t(max(0, min(a.first[i], int32_t(a.tokens)))), s.group); };
  uint32_t i0 = 0;
  for (uint32_t have = a.requests; have > 1;) {
    const uint32_t step = (have + 64 * kWaves - 1) / (64 * kWaves);
    if (threadIdx.x == 0) found_s = ~0u;
    __syncthreads();
    const uint64_t off = uint64_t(threadIdx.x) * step;
    if (off < have) {
      const uint32_t i = i0 + uint32_t(off), next = off + step < have ? i + step : i0 + have;
      if (place(i) <= blockIdx.x && (next >= a.requests || blockIdx.x < place(next))) found_s = i;
    }
    __syncthreads();
    i0 = found_s;
    if (i0 == ~0u) return;
    have = min(step, a.requests - i0);
    __syncthreads();
  }
  i0 = __builtin_amdgcn_readfirstlane(i0);
  const Request r(a, i0, s.group);
  const uint32_t tile = blockIdx.x - place(i0), kept = blockIdx.y;
  if (tile >= r.tiles) return;
  const Pieces p = pieces[uint64_t(blockIdx.x) * c.kv_heads + kept];
  if (p.end == 0) return;
  const uint32_t begin = p.at / p.share, end = min((p.end - 1) / p.share, s.shares - 1);  // the shares that hold it
  uint32_t turns = 1;
  while (turns * 4 <= end - begin && turns * 2 <= kAtOnce) turns *= 2;
  const uint32_t group = threadIdx.x / kLanes, lane = threadIdx.x % kLanes, turn = group % turns, rows = kAtOnce / turns;
  const uint32_t there = min(r.fresh * s.group - tile * kRows, kRows);
  for (uint32_t row0 = blockIdx.z * rows; row0 < there; row0 += gridDim.z * rows) {
    const uint32_t row = row0 + group / turns, y = tile * kRows + row;
    const bool on = group < rows * turns && row < there;
    f32x4 sum = {0, 0, 0, 0};
    float total = 0.0f, best = -INFINITY;
    if (on) {
      for (uint32_t k = begin + turn; k <= end; k += 4 * turns) {  // (four on their way at a time: they come from memory)
        float2 st[4];
        f32x4 v[4];
#pragma unroll
        for (uint32_t u = 0; u < 4; ++u) {
          const uint32_t piece = min(k + u * turns, end);
          const uint64_t part = (2 * piece + (p.at > piece * p.share)) * c.kv_heads + kept;
          st[u] = stats[part * kRows + row];
          v[u] = *reinterpret_cast<const f32x4*>(parts + (part * kRows + row) * D + 4 * lane);
        }
#pragma unroll
        for (uint32_t u = 0; u < 4; ++u)
          if (k + u * turns <= end) add(best, total, sum, st[u].x, st[u].y, v[u]);
      }
    }
    if (turns > 1) {
      __syncthreads();  // the last rows' sums are read
      if (on) {
        sum_s[group][lane] = sum;
        if (lane == 0) stat_s[group] = {best, total};
      }
      __syncthreads();
    }
    if (on && turn == 0) {
      for (uint32_t k = 1; k < turns; ++k) add(best, total, sum, stat_s[group + k].x, stat_s[group + k].y, sum_s[group + k][lane]);
      u16* out = const_cast<u16*>(row_of<u16>(a.out, r.first + y / s.group, kept * s.group + y % s.group));
#pragma unroll
      for (uint32_t k = 0; k < 4; ++k) out[4 * lane + k] = T::down(total == 0.0f ? 0.0f : sum[k] / total);
    }
  }
}

// Tiles of 16 rows of all requests together, at most, and the places of a list of them.
uint64_t tiles_at_most(const tsa_attend_cached_args& a, uint32_t group) {
  return (a.requests < a.tokens ? a.requests : a.tokens) + uint64_t(a.tokens) * group / kRows;
}
uint64_t tile_places(const tsa_attend_cached_args& a, uint32_t group) { return a.requests + uint64_t(a.tokens) * group / kRows; }
// Shares that the rounds make: groups() together, fewer where there are not as many rounds.
CachedShape shape_of(const tsa_cache& c, const tsa_attend_cached_args& a) {
  CachedShape s;
  s.group = a.q.heads / c.kv_heads;
  const uint64_t shares = (groups(c.head_dim) + c.kv_heads - 1) / c.kv_heads, most = tiles_at_most(a, s.group) * ((a.width + kWaves - 1) / kWaves);
  s.shares = uint32_t(shares < most ? shares : most);
  s.c = std::max(std::fabs(a.scale) * 1.44269504f, std::numeric_limits<float>::min());
  s.flip = std::signbit(a.scale) ? 0x80008000u : 0;
  s.aligned = vector_heads(a.q) && vector_heads(a.out);
  return s;
}

template <class T, int NB>
void attend_cached(const tsa_cache& c, const tsa_attend_cached_args& a, const CachedShape& s, void* workspace, hipStream_t stream) {
  const uint32_t groups = s.shares * c.kv_heads;
  float* parts = static_cast<float*>(workspace);
  float2* stats = reinterpret_cast<float2*>(parts + uint64_t(2) * groups * kRows * 32 * NB);
  Pieces* pieces = reinterpret_cast<Pieces*>(stats + uint64_t(2) * groups * kRows);
  hipLaunchKernelGGL((cached_kernel<T, NB>), dim3(groups), dim3(64 * kWaves), 0, stream, c, a, s, parts, stats, pieces);
  if (s.shares == 1) return;  // (it holds every tile whole)
  // (a workgroup a row where there are few tiles: 24 pieces of 12 rows take one workgroup 20 us, and one a row 6)
  const uint32_t tiles = uint32_t(tile_places(a, s.group)), all = tiles * c.kv_heads, rows = all * kRows <= 1024 ? kRows : all < 1024 ? 1024 / all : 1;
  hipLaunchKernelGGL((join_kernel<T, NB>), dim3(tiles, c.kv_heads, rows), dim3(64 * kWaves), 0, stream, c, a, s, parts, stats, pieces);
}

}  // namespace
}  // namespace op

uint64_t attend_cached_workspace(const tsa_cache& c, const tsa_attend_cached_args& a) {
  const op::CachedShape s = op::shape_of(c, a);
  return c.kv_heads * (uint64_t(s.shares) * 2 * op::kRows * (4 * c.head_dim + 8) + op::tile_places(a, s.group) * sizeof(op::Pieces));
}

int launch_attend_cached(const tsa_cache& c, const tsa_attend_cached_args& a, void* workspace, hipStream_t stream) {
  const op::CachedShape s = op::shape_of(c, a);
#define CALL(NB)                                                                                     \
  do {                                                                                               \
    if (a.type == TSA_BF16) op::attend_cached<op::Bf16, NB>(c, a, s, workspace, stream);             \
    else op::attend_cached<op::F16, NB>(c, a, s, workspace, stream);                                 \
  } while (0)
  switch (c.head_dim / 32) {
    case 1: CALL(1); break;
    case 2: CALL(2); break;
    case 3: CALL(3); break;
    default: CALL(4); break;
  }
#undef CALL
  return int(hipGetLastError());
}

}  // namespace tsa
