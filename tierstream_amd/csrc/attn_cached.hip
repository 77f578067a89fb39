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
// exponent (128 + n, in half precision 16 + n), exactly; the offset is taken off by the product's own accumulator (keys) and by a product
// with a constant (values). A key block's scale multiplies its 32-value product in 32 bits; a value's scale multiplies
// its probability, which is then rounded once (bf16), or split into two bf16 numbers (half precision, whose range would not hold it).
// Values are read transposed, 16 tokens of one column a lane, by ds_read_b64_tr_b4.
#include "attn_device.hpp"

namespace tsa {
namespace op {
namespace {

constexpr uint32_t kWaves = 4, kRows = 16, kMinShare = kWaves;  // waves, query rows and the fewest pages of a workgroup
// Probabilities times scales go to the matrix instruction as two bf16 numbers each, rounded to 16 bits, in half precision; in bf16 too up to so
// many pages (of all heads): few outputs may be off by more than their own rounding otherwise, and such calls are all latency (one token
// behind 4096: 10.4 us either way). Beyond, as one number: its error is like the output's own, and the second takes a fifth of the time.
constexpr uint64_t kSplitPages = 2048;
// Workgroups of a CU that the registers leave room for, and of the chip.
constexpr uint32_t per_cu(uint32_t head_dim) { return head_dim <= 64 ? 4 : 3; }
constexpr uint32_t groups(uint32_t head_dim) { return 256 * per_cu(head_dim); }

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
  float c;            // scale / ln 2
  bool aligned;       // q and out in pieces of 8
};

// ---- who does what --------------------------------------------------------------------------------------------------------
// All requests' tiles of 16 query rows, one behind the other, each with its pages (one at least), are one row of pages. It is
// cut into equal shares, a workgroup each, wherever the cuts fall. A tile inside one share is written at once; a share's piece of any
// other is left in the workspace: at place 0 of the share where it begins with the share, at place 1 where it begins inside.

// Request i's new tokens, the tokens it ends with, its tiles and their pages.
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
  __device__ __forceinline__ uint32_t places() const { return pages ? pages : 1; }
};

struct Place {
  uint32_t share, all;  // pages of a share and of all
  uint32_t at;          // first page of the tile
  uint32_t request, tile;
};
struct PlaceMemory {
  uint32_t pages[kWaves], tiles[kWaves];
  Place found;
};

template <class V>
__device__ __forceinline__ V lanes_up_to(V v) {
#pragma unroll
  for (uint32_t s = 1; s < 64; s <<= 1) {
    const V o = __shfl_up(v, s, 64);
    if ((threadIdx.x & 63u) >= s) v += o;
  }
  return v;
}

// The tile that holds the first page of share `want` (kByTile: tile number `want`). By the whole workgroup; false: there is none.
template <bool kByTile>
__device__ __forceinline__ bool find_place(const tsa_attend_cached_args& a, const CachedShape& s, uint32_t want, PlaceMemory& m, Place& out) {
  const uint32_t t = threadIdx.x, lane = t & 63u, wave = t >> 6, per = (a.requests + 64 * kWaves - 1) / (64 * kWaves);
  const uint32_t i0 = min(t * per, a.requests), i1 = min(i0 + per, a.requests);
  uint32_t pages = 0, tiles = 0;
  for (uint32_t i = i0; i < i1; ++i) {
    const Request r(a, i, s.group);
    pages += r.tiles * r.places();
    tiles += r.tiles;
  }
  const uint32_t pages_upto = lanes_up_to(pages);
  const uint32_t tiles_upto = kByTile ? lanes_up_to(tiles) : 0;
  if (lane == 63) {
    m.pages[wave] = pages_upto;
    m.tiles[wave] = tiles_upto;
  }
  __syncthreads();
  Place p = {};
  uint32_t page0 = pages_upto - pages, tile0 = tiles_upto - tiles, every = 0;
#pragma unroll
  for (uint32_t w = 0; w < kWaves; ++w) {
    p.all += m.pages[w];
    every += m.tiles[w];
    if (w < wave) page0 += m.pages[w], tile0 += m.tiles[w];
  }
  const uint32_t even = p.all / s.shares + (p.all % s.shares != 0);
  p.share = even < kMinShare ? kMinShare : even;
  const uint64_t page = uint64_t(want) * p.share;  // (past all of them, perhaps by far)
  if (kByTile ? want >= every : page >= p.all) return false;
  if (kByTile ? want >= tile0 && want < tile0 + tiles : page >= page0 && page < page0 + pages) {
    for (uint32_t i = i0; i < i1; ++i) {
      const Request r(a, i, s.group);
      const uint32_t have = r.tiles * r.places();
      if (kByTile ? want < tile0 + r.tiles : page < page0 + have) {
        p.request = i;
        p.tile = kByTile ? want - tile0 : uint32_t((page - page0) / r.places());
        p.at = page0 + p.tile * r.places();
        m.found = p;
        break;
      }
      page0 += have, tile0 += r.tiles;
    }
  }
  __syncthreads();
  out = m.found;
  return true;
}

// ---- numbers of 4 bits ----------------------------------------------------------------------------------------------------
// The half bytes 0, 4, 1, 5, 2, 6, 3, 7 of a word as 16-bit numbers n + 128 (bf16) or n + 16 (half precision).
// `one` and `mask` are kept in registers: as literals each would take an instruction of its own.
template <bool kHalf>
struct Numbers {
  uint32_t mask = kHalf ? 0x03C003C0u : 0x000F000Fu, one = kHalf ? 0x4C004C00u : 0x43004300u;
  __device__ __forceinline__ Numbers() { asm("" : "+s"(mask), "+v"(one)); }
  __device__ __forceinline__ bits8 of(uint32_t x) const {
    u32x4 v;
    if constexpr (kHalf) v = u32x4{((x << 6) & mask) | one, ((x << 2) & mask) | one, ((x >> 2) & mask) | one, ((x >> 6) & mask) | one};
    else v = u32x4{(x & mask) | one, ((x >> 4) & mask) | one, ((x >> 8) & mask) | one, ((x >> 12) & mask) | one};
    return __builtin_bit_cast(bits8, v);
  }
};
__device__ __forceinline__ uint32_t pack(float a, float b) {
  typedef __bf16 two __attribute__((ext_vector_type(2)));
  typedef float two_f __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((two_f{a, b}), two));
}

// The larger of a value in the four lanes of a column.
__device__ __forceinline__ float column_max(float v) {
  v = fmaxf(v, __shfl_xor(v, 16, 64));
  return fmaxf(v, __shfl_xor(v, 32, 64));
}
__device__ __forceinline__ float column_sum(float v) {
  v += __shfl_xor(v, 16, 64);
  return v + __shfl_xor(v, 32, 64);
}

// ---- the pages --------------------------------------------------------------------------------------------------------------
// A page of a head in memory, and in LDS, where the scales have room for whole loads.
template <int NB>
struct Page {
  static constexpr uint32_t kBytes = 2304 * NB, kKeyScalesAt = 1024 * NB, kValueScalesAt = 1152 * NB, kValuesAt = 1280 * NB;
  static constexpr uint32_t kScaleLoads = (NB + 1) / 2, kLoads = NB + kScaleLoads;  // of the keys' half, and of the values'
  static constexpr uint32_t kKeyScales = 1024 * NB, kValueScales = kKeyScales + 256 * kScaleLoads, kValues = kValueScales + 256 * kScaleLoads,
                            kRoom = kValues + 1024 * NB;
};

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

template <class T, int NB, bool kSplit>
__global__ __launch_bounds__(64 * kWaves, per_cu(32 * NB)) void cached_kernel(tsa_cache c, tsa_attend_cached_args a, CachedShape s, float* parts, float2* stats) {
  typedef Page<NB> P;
  constexpr bool kHalf = std::is_same_v<T, F16>;
  constexpr uint32_t D = 32 * NB;
  __shared__ __attribute__((aligned(16))) unsigned char page_s[kWaves][P::kRoom];
  __shared__ __attribute__((aligned(16))) u16 query_s[kRows][D + 4];  // (rows apart by banks)
  __shared__ float2 stat_s[kWaves][kRows];
  __shared__ PlaceMemory place_s;
  static_assert(P::kRoom >= kRows * D * 4, "a wave's outputs take its page's place");
  Place at;
  const uint32_t kept = blockIdx.x % c.kv_heads, share = blockIdx.x / c.kv_heads;
  if (!find_place<false>(a, s, share, place_s, at)) return;
  const uint32_t from = share * at.share, upto = min(from + at.share, at.all);  // this share's pages
  const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4;
  const uint32_t lds = __builtin_amdgcn_readfirstlane(lds_offset(page_s[wave]));
  const Numbers<kHalf> keys;
  const Numbers<false> values;
  const bits8 eight = {0xC308, 0xC308, 0xC308, 0xC308, 0xC308, 0xC308, 0xC308, 0xC308};  // -136
  Request r(a, at.request, s.group);
  while (true) {  // the share's tiles
    const uint32_t x = at.tile * kRows + (lane & 15u);
    const bool on = x < r.fresh * s.group;
    const uint32_t token = on ? x / s.group : 0;
    const int32_t limit = on ? r.end - int32_t(r.fresh) + int32_t(token) + 1 : 0;  // keys that this row attends to
    const int32_t whole = r.end - int32_t(r.fresh) + 1;                            // keys that every row attends to

    // The queries, once for all waves (each by itself, value by value, took 9 us). Pieces of 8 where they start 16-byte aligned.
    for (uint32_t i = threadIdx.x; i < kRows * D / 8; i += 64 * kWaves) {
      const uint32_t y = at.tile * kRows + i / (D / 8), d = i % (D / 8) * 8;
      bits8 v = {0, 0, 0, 0, 0, 0, 0, 0};
      if (y < r.fresh * s.group) {
        const u16* p = row_of<u16>(a.q, r.first + y / s.group, kept * s.group + y % s.group) + d;
        if (s.aligned) {
          v = *reinterpret_cast<const bits8*>(p);
        } else {
#pragma unroll
          for (int k = 0; k < 8; ++k) v[k] = p[k];
        }
      }
      *reinterpret_cast<uint2*>(&query_s[i / (D / 8)][d]) = uint2{__builtin_bit_cast(u32x4, v)[0], __builtin_bit_cast(u32x4, v)[1]};
      *reinterpret_cast<uint2*>(&query_s[i / (D / 8)][d + 4]) = uint2{__builtin_bit_cast(u32x4, v)[2], __builtin_bit_cast(u32x4, v)[3]};
    }
    __syncthreads();
    // this row's, in the order of the keys' half bytes, and what takes their offset off
    bits8 q[NB];
    f32x4 off[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      const bits4 lo = *reinterpret_cast<const bits4*>(&query_s[lane & 15u][32 * b + 4 * g]), hi = *reinterpret_cast<const bits4*>(&query_s[lane & 15u][32 * b + 16 + 4 * g]);
      q[b] = bits8{lo[0], lo[2], hi[0], hi[2], lo[1], lo[3], hi[1], hi[3]};
      float sum = 0.0f;
#pragma unroll
      for (uint32_t i = 0; i < 8; ++i) sum += T::up(q[b][i]);
      sum = column_sum(sum) * (kHalf ? -24.0f : -136.0f);
      off[b] = f32x4{sum, sum, sum, sum};
    }

    f32x4 o[2 * NB];
#pragma unroll
    for (int i = 0; i < 2 * NB; ++i) o[i] = f32x4{0, 0, 0, 0};
    float top = -INFINITY, total = 0.0f;

    const uint32_t begin = max(from, at.at) - at.at, end = min(r.pages, upto - at.at);
    const int32_t* table = a.table + uint64_t(at.request) * a.table_stride;
    // Half a page to LDS, keys or values. While the keys of one are multiplied its values are on their way, and while these are the next
    // page's keys: one buffer is enough for that, and three or four workgroups fit a CU.
    auto fetch = [&](uint32_t page, bool value) {
      const unsigned char* at = static_cast<const unsigned char*>(c.pages) + (uint64_t(page) * c.kv_heads + kept) * P::kBytes;
      const unsigned char* scales = at + (value ? P::kValueScalesAt : P::kKeyScalesAt);
#pragma unroll
      for (uint32_t i = 0; i < uint32_t(NB); ++i) load_to_lds(at + (value ? P::kValuesAt : 0) + i * 1024 + lane * 16, lds + (value ? P::kValues : 0) + i * 1024);
#pragma unroll
      for (uint32_t i = 0; i < P::kScaleLoads; ++i)  // (what a last half load is too much stays in its room)
        load_words_to_lds(scales + min(i * 256 + lane * 4, 128u * NB - 4), lds + (value ? P::kValueScales : P::kKeyScales) + i * 256);
    };
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
    if (p < end) {
      fetch(page, false);
      fetch(page, true);
    }
    while (p < end) {
      const int32_t key0 = int32_t(p * kPage);
      const bool edge = key0 + int32_t(kPage) > whole;
      p += kWaves, ++turn;
      page = page_here();  // the next one
      const bool more = p < end;
      loads_left<P::kLoads>();
      // Tokens that not every row attends to must not reach the others through 0 x NaN: behind the last key the values' scales become 0;
      // before it one that is no number becomes 0 and its key's scale NaN, which reaches only the rows that attend to it.
      if (edge) loads_left<0>();
      if (edge && key0 + int32_t(lane) >= whole) {
#pragma unroll
        for (uint32_t b = 0; b < NB; ++b) {
          lds_half_t* const scale = reinterpret_cast<lds_half_t*>(lds + P::kValueScales + (lane * NB + b) * 2);
          const bool none = (*scale & 0x7C00u) == 0x7C00u;
          if (none) *reinterpret_cast<lds_half_t*>(lds + P::kKeyScales + (lane * NB + b) * 2) = 0x7E00;
          if (none || key0 + int32_t(lane) >= r.end) *scale = 0;
        }
      }

      // scores: tile j holds tokens 16 j + 4 g + 0..3 of this lane's row
      f32x4 score[4];
#pragma unroll
      for (uint32_t j = 0; j < 4; ++j) {
        typedef uint32_t row_words __attribute__((ext_vector_type(NB)));
        const uint32_t key = lds + (16 * j + (lane & 15u)) * 16 * NB + g * 4 * NB;
        row_words words;
        if constexpr (NB == 3) {  // (4-byte aligned)
#pragma unroll
          for (int b = 0; b < NB; ++b) words[b] = reinterpret_cast<lds_word_t*>(key)[b];
        } else {
          words = *reinterpret_cast<__attribute__((address_space(3))) const row_words*>(key);
        }
        const Scales<NB> scale(lds + P::kKeyScales + (16 * j + 4 * g) * 2 * NB);
        f32x4 sum = {0, 0, 0, 0};
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          const f32x4 v = T::mfma(keys.of(words[b]), q[b], off[b]);
#pragma unroll
          for (uint32_t k = 0; k < 4; ++k) sum[k] = __builtin_fmaf(scale.at(k, b), v[k], sum[k]);
        }
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k) score[j][k] = sum[k] * s.c;
      }
      if (edge) {
        asm volatile("" ::: "memory");  // (kept out of the other pages' way)
        const int32_t left = limit - key0 - int32_t(4 * g);
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j)
#pragma unroll
          for (uint32_t k = 0; k < 4; ++k)
            if (int32_t(16 * j + k) >= left) score[j][k] = -INFINITY;
      }

      reads_done();
      if (more) fetch(page, false);

      // the running maximum: followed only where it is passed by 2^8 (probabilities are then up to 2^8, which 32 bits and bf16 hold)
      float most = -INFINITY;
#pragma unroll
      for (uint32_t j = 0; j < 4; ++j)
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k) most = fmaxf(most, score[j][k]);
      most = column_max(most);
      if (__any(most > top + 8.0f)) {
        const float up = fmaxf(most, top), keep = top == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(top - up);
        top = up;
        total *= keep;
#pragma unroll
        for (int i = 0; i < 2 * NB; ++i) o[i] *= keep;
      }
      const float base = top == -INFINITY ? 0.0f : top;
#pragma unroll
      for (uint32_t j = 0; j < 4; ++j)
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k) {
          score[j][k] = __builtin_amdgcn_exp2f(score[j][k] - base);
          total += score[j][k];
        }

      // outputs, 32 tokens a step; a lane's eight are tiles 2 t and 2 t + 1
      if (more) loads_left<P::kLoads>();
      else loads_left<0>();
      // row i of the transposed read is lane i's token, of both halves of a block: a word of the result holds, in the order of Numbers, the
      // lane's eight tokens of one column
      const uint32_t i16 = lane & 15u, e = ((i16 & 3u) << 1) | ((i16 >> 2) & 1u);
      const uint32_t row = (e < 4 ? 4 * g + e : 16 + 4 * g + e - 4) * 16 + 8 * (i16 >> 3);
#pragma unroll
      for (uint32_t t = 0; t < 2; ++t) {
        Scales<NB> scales[2];
#pragma unroll
        for (uint32_t j = 0; j < 2; ++j) scales[j] = Scales<NB>(lds + P::kValueScales + (32 * t + 16 * j + 4 * g) * 2 * NB);
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          const i32x2 words = __builtin_amdgcn_ds_read_tr4_b64_v2i32(
              reinterpret_cast<lds_i32x2_t*>(lds + P::kValues + b * 1024 + t * 512 + row));
          float w[8];
#pragma unroll
          for (uint32_t i = 0; i < 8; ++i)
            w[i] = __builtin_fmaf(score[2 * t + i / 4][i % 4], scales[i / 4].at(i % 4, b), 0.0f);  // (takes the scale as it is)
          const u32x4 hi = {pack(w[0], w[1]), pack(w[2], w[3]), pack(w[4], w[5]), pack(w[6], w[7])};
          const bits8 p16 = __builtin_bit_cast(bits8, hi);
#pragma unroll
          for (uint32_t h = 0; h < 2; ++h) {
            o[2 * b + h] = Bf16::mfma(eight, p16, o[2 * b + h]);
            o[2 * b + h] = Bf16::mfma(values.of(uint32_t(words[h])), p16, o[2 * b + h]);
          }
          if constexpr (kSplit) {
            u32x4 lo;
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i)
              lo[i] = pack(w[2 * i] - Bf16::up(u16(hi[i])), w[2 * i + 1] - Bf16::up(u16(hi[i] >> 16)));
            const bits8 rest = __builtin_bit_cast(bits8, lo);
#pragma unroll
            for (uint32_t h = 0; h < 2; ++h) {
              o[2 * b + h] = Bf16::mfma(eight, rest, o[2 * b + h]);
              o[2 * b + h] = Bf16::mfma(values.of(uint32_t(words[h])), rest, o[2 * b + h]);
            }
          }
        }
      }
      reads_done();
      if (more) fetch(page, true);
    }

    // the waves' parts together
    total = column_sum(total);
    if (lane < kRows) stat_s[wave][lane] = {top, total};
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __syncthreads();  // every wave is done with its pages
    float best = -INFINITY, sum = 0.0f;
#pragma unroll
    for (uint32_t w = 0; w < kWaves; ++w) best = fmaxf(best, stat_s[w][lane & 15u].x);
    const float base = best == -INFINITY ? 0.0f : best;
#pragma unroll
    for (uint32_t w = 0; w < kWaves; ++w) {
      const float2 st = stat_s[w][lane & 15u];
      sum += st.y * __builtin_amdgcn_exp2f(st.x - base);
    }
    const bool whole_tile = at.at >= from && at.at + r.places() <= upto;
    const float by = __builtin_amdgcn_exp2f(top - base) * (!whole_tile ? 1.0f : sum == 0.0f ? 0.0f : 1.0f / sum);
    float* mine = reinterpret_cast<float*>(page_s[wave]) + (lane & 15u) * D;
#pragma unroll
    for (int i = 0; i < 2 * NB; ++i)
#pragma unroll
      for (uint32_t k = 0; k < 4; ++k)  // column 4 g + k of the tile: byte (4 g + k) / 2 of the half block, low half bytes first
        mine[32 * (i / 2) + 8 * (i % 2) + (4 * g + k) / 2 + 16 * (k & 1u)] = o[i][k] * by;
    __syncthreads();
    const uint32_t part = (2 * share + (at.at > from)) * c.kv_heads + kept;
    if (!whole_tile && threadIdx.x < kRows) stats[part * kRows + threadIdx.x] = {best, sum};
    for (uint32_t i = threadIdx.x; i < kRows * D / 4; i += 64 * kWaves) {
      const uint32_t y = at.tile * kRows + i / (D / 4), d = i % (D / 4) * 4;
      if (y >= r.fresh * s.group) break;
      f32x4 v = {0, 0, 0, 0};
#pragma unroll
      for (uint32_t w = 0; w < kWaves; ++w) v += reinterpret_cast<const f32x4*>(page_s[w])[i];
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
    at.at += r.places();
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

// The pieces of a tile together: threads of a row take four values and every eighth piece or so.
template <class T, int NB>
__global__ __launch_bounds__(64 * kWaves) void join_kernel(tsa_cache c, tsa_attend_cached_args a, CachedShape s, const float* parts, const float2* stats) {
  constexpr uint32_t D = 32 * NB, kLanes = D / 4, kTurns = 64 * kWaves / kLanes;
  __shared__ PlaceMemory place_s;
  __shared__ f32x4 sum_s[kTurns][kLanes];
  __shared__ float2 stat_s[kTurns];
  Place at;
  const uint32_t kept = blockIdx.x % c.kv_heads;
  if (!find_place<true>(a, s, blockIdx.x / c.kv_heads, place_s, at)) return;
  const Request r(a, at.request, s.group);
  const uint32_t begin = at.at / at.share, end = (at.at + r.places() - 1) / at.share;  // the shares that hold it
  if (begin == end) return;
  const uint32_t turn = threadIdx.x / kLanes, lane = threadIdx.x % kLanes;
  for (uint32_t col = blockIdx.y; col < kRows; col += gridDim.y) {
    const uint32_t y = at.tile * kRows + col;
    if (y >= r.fresh * s.group) break;
    f32x4 sum = {0, 0, 0, 0};
    float total = 0.0f, best = -INFINITY;
    if (turn < kTurns) {
#pragma unroll 4
      for (uint32_t k = begin + turn; k <= end; k += kTurns) {
        const uint64_t part = (2 * k + (at.at > k * at.share)) * c.kv_heads + kept;
        const float2 st = stats[part * kRows + col];
        const f32x4 v = *reinterpret_cast<const f32x4*>(parts + (part * kRows + col) * D + 4 * lane);
        add(best, total, sum, st.x, st.y, v);
      }
    }
    __syncthreads();  // the last row's sums are read
    if (turn < kTurns) {
      sum_s[turn][lane] = sum;
      if (lane == 0) stat_s[turn] = {best, total};
    }
    __syncthreads();
    if (threadIdx.x < kLanes) {
      for (uint32_t k = 1; k < kTurns; ++k) add(best, total, sum, stat_s[k].x, stat_s[k].y, sum_s[k][lane]);
      u16* out = const_cast<u16*>(row_of<u16>(a.out, r.first + y / s.group, kept * s.group + y % s.group));
#pragma unroll
      for (uint32_t k = 0; k < 4; ++k) out[4 * lane + k] = T::down(total == 0.0f ? 0.0f : sum[k] / total);
    }
  }
}

// Tiles of 16 rows of all requests together, at most.
uint64_t tiles_at_most(const tsa_attend_cached_args& a, uint32_t group) {
  return (a.requests < a.tokens ? a.requests : a.tokens) + uint64_t(a.tokens) * group / kRows;
}
// Shares that the pages make: groups() together, fewer where there are not kMinShare pages for each.
CachedShape shape_of(const tsa_cache& c, const tsa_attend_cached_args& a) {
  CachedShape s;
  s.group = a.q.heads / c.kv_heads;
  const uint64_t shares = (groups(c.head_dim) + c.kv_heads - 1) / c.kv_heads, most = (tiles_at_most(a, s.group) * a.width + kMinShare - 1) / kMinShare;
  s.shares = uint32_t(shares < most ? shares : most);
  s.c = a.scale * 1.44269504f;
  s.aligned = vector_heads(a.q) && vector_heads(a.out);
  return s;
}

template <class T, int NB>
void attend_cached(const tsa_cache& c, const tsa_attend_cached_args& a, const CachedShape& s, void* workspace, hipStream_t stream) {
  const uint32_t tiles = uint32_t(tiles_at_most(a, s.group)) * c.kv_heads;
  float* parts = static_cast<float*>(workspace);
  float2* stats = reinterpret_cast<float2*>(parts + uint64_t(2) * s.shares * c.kv_heads * kRows * 32 * NB);
  const dim3 grid(s.shares * c.kv_heads), block(64 * kWaves);
  constexpr bool kHalf = std::is_same_v<T, F16>;
  if (kHalf || uint64_t(tiles) * a.width <= kSplitPages) hipLaunchKernelGGL((cached_kernel<T, NB, true>), grid, block, 0, stream, c, a, s, parts, stats);
  else hipLaunchKernelGGL((cached_kernel<T, NB, kHalf>), grid, block, 0, stream, c, a, s, parts, stats);
  // (a workgroup a row where there are few; one share holds every tile whole)
  const uint32_t rows = tiles * kRows <= 1024 ? kRows : tiles < 1024 ? 1024 / tiles : 1;
  if (s.shares > 1) hipLaunchKernelGGL((join_kernel<T, NB>), dim3(tiles, rows), dim3(64 * kWaves), 0, stream, c, a, s, parts, stats);
}

}  // namespace
}  // namespace op

uint64_t attend_cached_workspace(const tsa_cache& c, const tsa_attend_cached_args& a) {
  return uint64_t(2) * op::shape_of(c, a).shares * c.kv_heads * op::kRows * (4 * c.head_dim + 8);
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
