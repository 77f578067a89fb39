// Tiles of packed sequences for the attention kernels: 64 rows of a head in LDS, read two ways as the first operand of
// v_mfma_f32_32x32x16. A wave's own 32 rows (queries, or keys) are the columns of every product and stay in registers; what it
// runs over comes through LDS:
//   rows     the tile's rows against the wave's (scores, and gradients of probabilities): 16 bytes of a row a lane;
//   columns  the tile transposed against a 32 x 64 result of the first kind, whose registers are the second operand as they are (outputs and
//            gradients): ds_read_b64_tr_b16 gives each lane of 16 one column of 4 rows.
// A lane of the result holds column l % 32 at rows 8 (i / 4) + 4 (l / 32) + i % 4, i = 0..15; its registers 8 u..8 u + 7 are those rows of
// 16 u.., and the transposed reads bring the same rows in the same order.
//
// A row is kD values (64 or 128; behind head_dim zeros) in pieces of 16 bytes; piece c of row r stands at c ^ turn(r), so that neither
// 16 rows' same piece nor 4 rows' same 64 bytes meet in a bank. The loads' addresses make the permutation: LDS is filled in lane order.
#pragma once

#include "attn_device.hpp"

namespace tsa {
namespace op {

constexpr uint32_t kTile = 64, kOwn = 32, kTileWaves = 4, kTileOwn = kOwn * kTileWaves;

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4_t lds_four_t;
typedef __attribute__((address_space(3))) const bits8 lds_eight_t;
typedef __attribute__((address_space(3))) bits8 lds_eight_put_t;

template <class T>
__device__ __forceinline__ f32x16 mfma32(bits8 a, bits8 b, f32x16 c) {
  typedef typename T::v8 v8;
  if constexpr (std::is_same_v<T, Bf16>) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
}

// Two values rounded to 16 bits.
template <class T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  typedef std::conditional_t<std::is_same_v<T, Bf16>, __bf16, _Float16> half;
  typedef half two __attribute__((ext_vector_type(2)));
  typedef float two_f __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((two_f{a, b}), two));
}
template <class T>
__device__ __forceinline__ bits8 pack8(const f32x16& v, int u) {
  return __builtin_bit_cast(bits8, u32x4{pack2<T>(v[8 * u], v[8 * u + 1]), pack2<T>(v[8 * u + 2], v[8 * u + 3]), pack2<T>(v[8 * u + 4], v[8 * u + 5]),
                                         pack2<T>(v[8 * u + 6], v[8 * u + 7])});
}

// Rows 16 u.. of a result as the second operand of the next product: rounded to 16 bits, and (kSplit) what that leaves of them.
template <class T, bool kSplit>
struct Second {
  bits8 part[kSplit ? 2 : 1];
  __device__ __forceinline__ Second(const f32x16& v, int u) {
    part[0] = pack8<T>(v, u);
    if constexpr (kSplit) {
      f32x16 rest;
#pragma unroll
      for (int i = 0; i < 8; ++i) rest[i] = v[8 * u + i] - T::up(part[0][i]);
      part[1] = pack8<T>(rest, 0);
    }
  }
  __device__ __forceinline__ void add(bits8 a, f32x16& sum) const {
    sum = mfma32<T>(a, part[0], sum);
    if constexpr (kSplit) sum = mfma32<T>(a, part[1], sum);
  }
};
// Sequences of so many pairs of a query and a key take both parts, in the forward pass and in the gradients: a sequence's results do not depend
// on what else is in the call (keys' gradients but for the order of sums in 32 bits) or how it lies in memory. The error against 64 bits is then that of rounding the results (bf16 0.0016, with
// one part 0.0020 to 0.0024). It costs nothing where a call is latency (301 rows of 4 heads: 10.4 us, gradients 27.3, either way), and where short
// sequences fill the chip some of the products' time: 32 of 256 rows, 32 heads of 128, 70 us for 64 and 319 for 305; 16 of 512, which is
// beyond, 93 for 80 and 388 for 358.
constexpr uint32_t kSplitPairs = 1u << 17;
__device__ __forceinline__ bool both_parts(uint32_t queries, uint32_t keys) { return uint64_t(queries) * keys <= kSplitPairs; }

template <int kD>
struct TileShapes {
  static constexpr uint32_t kRowBytes = 2 * kD, kPieces = kD / 8, kBytes = kTile * kRowBytes, kRowsALoad = 64 / kPieces,
                            kLoads = kTile / kRowsALoad / kTileWaves;
  static __device__ __forceinline__ uint32_t turn(uint32_t row) {
    return kD == 128 ? ((row & 3u) << 2) | ((row >> 2) & 3u) : (((row >> 1) & 1u) << 2) | ((row >> 2) & 3u);
  }
};

// 64 lanes x 16 bytes from base + offset to LDS at `at` (base and at the same in every lane) in lane order.
__device__ __forceinline__ void load_from_to_lds(const void* base, uint32_t offset, uint32_t at) {
  asm volatile(
      "s_mov_b32 m0, %2\n\t"
      "s_nop 0\n\t"
      "global_load_lds_dwordx4 %0, %1"
      :
      : "v"(offset), "s"(base), "s"(at)
      : "memory", "m0");
}

// Loads of one head's tiles. kAligned: pieces start 16-byte aligned, and a tile's rows lie within 2^31 bytes; otherwise value by value.
template <int kD, bool kAligned>
struct TileLoads {
  typedef TileShapes<kD> S;
  const u16* p;       // the head's first row
  uint64_t stride;
  uint32_t row, at, dim;
  uint32_t offset[kAligned ? S::kLoads : 1];  // this lane's pieces from a tile's first row, in bytes
  __device__ __forceinline__ TileLoads(const tsa_heads& h, uint64_t first, uint32_t head, uint32_t head_dim) {
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    row = wave * S::kLoads * S::kRowsALoad + lane / S::kPieces;
    p = row_of<u16>(h, first, head);
    stride = h.token_stride;
    at = __builtin_amdgcn_readfirstlane(wave) * S::kLoads * 1024;
    dim = head_dim;
    if constexpr (kAligned) {
#pragma unroll
      for (uint32_t j = 0; j < S::kLoads; ++j) offset[j] = uint32_t((row + j * S::kRowsALoad) * stride * 2) + 2 * value_of(j);
    }
  }
  __device__ __forceinline__ uint32_t value_of(uint32_t j) const {
    return 8 * (((threadIdx.x & 63u) % S::kPieces) ^ S::turn(row + j * S::kRowsALoad));
  }
  // Rows row0.. of `rows` to a buffer in LDS; rows behind the last are zeros.
  __device__ __forceinline__ void fetch(uint32_t row0, uint32_t rows, uint32_t buffer) const {
    const uint32_t lds = __builtin_amdgcn_readfirstlane(buffer + at);
    if constexpr (kAligned) {
      const u16* const base = p + row0 * stride;
      if (row0 + kTile <= rows && dim == kD) {
#pragma unroll
        for (uint32_t j = 0; j < S::kLoads; ++j) load_from_to_lds(base, offset[j], lds + j * 1024);
      } else {
#pragma unroll
        for (uint32_t j = 0; j < S::kLoads; ++j) {
          const bool in = row0 + row + j * S::kRowsALoad < rows && value_of(j) < dim;
          load_to_lds(in ? static_cast<const void*>(base + offset[j] / 2) : &kZeroPiece, lds + j * 1024);
        }
      }
    } else {
#pragma unroll
      for (uint32_t j = 0; j < S::kLoads; ++j) {
        const uint32_t r = row0 + row + j * S::kRowsALoad;
        bits8 v = {0, 0, 0, 0, 0, 0, 0, 0};
        if (r < rows && value_of(j) < dim) {
          const u16* g = p + r * stride + value_of(j);
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] = g[i];
        }
        *reinterpret_cast<lds_eight_put_t*>(lds + j * 1024 + (threadIdx.x & 63u) * 16) = v;
      }
    }
  }
};
// Whether heads are read in whole pieces, offsets inside a tile in 32 bits.
inline bool tile_heads(const tsa_heads& h) { return vector_heads(h) && h.token_stride < (uint64_t(1) << 24); }

// This wave's own rows as the second operand: column l % 32, values 16 k + 8 (l / 32)..; zeros where there is none.
template <int kD, bool kAligned>
struct OwnRows {
  bits8 v[kD / 16];
  __device__ __forceinline__ OwnRows(const tsa_heads& h, uint64_t row, uint32_t head, uint32_t dim, bool on) {
    const u16* g = row_of<u16>(h, on ? row : 0, head) + 8 * ((threadIdx.x & 63u) >> 5);
#pragma unroll
    for (uint32_t k = 0; k < kD / 16; ++k) {
      v[k] = bits8{0, 0, 0, 0, 0, 0, 0, 0};
      if (on && 16 * k + 8 * ((threadIdx.x & 63u) >> 5) < dim) {
        if constexpr (kAligned) {
          v[k] = *reinterpret_cast<const bits8*>(g + 16 * k);
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) v[k][i] = g[16 * k + i];
        }
      }
    }
  }
};

// The two ways to read a tile.
template <int kD>
struct TileReads {
  typedef TileShapes<kD> S;
  uint32_t rows_at[kD / 16];       // of piece 2 k + l / 32 of row l % 32
  uint32_t columns_at[kD / 32][2];  // of columns 32 t.. of rows 4 (l / 32).., and 8 further
  __device__ __forceinline__ TileReads() {
    const uint32_t lane = threadIdx.x & 63u, row = lane & 31u, h = lane >> 5;
#pragma unroll
    for (uint32_t k = 0; k < kD / 16; ++k) rows_at[k] = row * S::kRowBytes + ((2 * k + h) ^ S::turn(row)) * 16;
    const uint32_t l = lane & 15u;
#pragma unroll
    for (uint32_t t = 0; t < kD / 32; ++t)
#pragma unroll
      for (uint32_t s = 0; s < 2; ++s) {
        const uint32_t r = 8 * s + 4 * h + l / 4, piece = 4 * t + ((lane >> 4) & 1u) * 2 + ((l & 3u) >> 1);
        columns_at[t][s] = r * S::kRowBytes + (piece ^ S::turn(r)) * 16 + (l & 1u) * 8;
      }
  }
  // The places in the buffer at lds, added up once a tile (the compiler would add the buffer's to each read's).
  struct Rows {
    uint32_t at[kD / 16];
    __device__ __forceinline__ bits8 operator()(uint32_t r, uint32_t k) const {  // rows 32 r.. at values 16 k..
      return *reinterpret_cast<lds_eight_t*>(at[k] + r * 32 * S::kRowBytes);
    }
  };
  struct Columns {
    uint32_t at[kD / 32][2];
    __device__ __forceinline__ bits8 operator()(uint32_t t, uint32_t u) const {  // columns 32 t.. of rows 16 u..
      const s16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lds_four_t*>(at[t][0] + u * 16 * S::kRowBytes));
      const s16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lds_four_t*>(at[t][1] + u * 16 * S::kRowBytes));
      return __builtin_bit_cast(bits8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    }
  };
  __device__ __forceinline__ Rows rows(uint32_t lds) const {
    Rows r;
#pragma unroll
    for (uint32_t k = 0; k < kD / 16; ++k) {
      r.at[k] = lds + rows_at[k];
      asm("" : "+v"(r.at[k]));
    }
    return r;
  }
  __device__ __forceinline__ Columns columns(uint32_t lds) const {
    Columns c;
#pragma unroll
    for (uint32_t t = 0; t < kD / 32; ++t)
#pragma unroll
      for (uint32_t s = 0; s < 2; ++s) {
        c.at[t][s] = lds + columns_at[t][s];
        asm("" : "+v"(c.at[t][s]));
      }
    return c;
  }
};

template <int N>
__device__ __forceinline__ void clear(f32x16 (&v)[N]) {
#pragma unroll
  for (int t = 0; t < N; ++t)
#pragma unroll
    for (int i = 0; i < 16; ++i) v[t][i] = 0.0f;
}

// The order of kProducts matrix instructions and the 16-byte reads from LDS that feed one each: kAhead reads stand before the
// first, so that each has the time of kAhead products (left to itself the compiler reads one ahead, and every product waits).
template <int kProducts, int kAhead>
__device__ __forceinline__ void products_behind_reads() {
  __builtin_amdgcn_sched_group_barrier(0x100, kAhead, 0);
#pragma unroll
  for (int i = 0; i < kProducts - kAhead; ++i) {
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
  }
  __builtin_amdgcn_sched_group_barrier(0x008, kAhead, 0);
}

// Own loads landed, own reads done, and all waves here.
__device__ __forceinline__ void tile_ready() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// What a mask leaves out must not reach a sum through 0 x infinity or 0 x NaN. Where a mask cuts a tile, its values that are no numbers
// become 0 and their rows' marks NaN (others' 0), which are added to the scores before the mask is: rows that attend to them are NaN as a
// whole then. By the whole workgroup, four threads a row; clean_done() before the marks or the tile are read.
template <class T, int kD>
__device__ __forceinline__ bool clean_tile(uint32_t lds) {
  constexpr uint32_t kExponents = std::is_same_v<T, Bf16> ? 0x7F807F80u : 0x7C007C00u, kCarry = std::is_same_v<T, Bf16> ? 0x00800080u : 0x04000400u;
  typedef __attribute__((address_space(3))) u32x4 piece_t;
  bool bad = false;
#pragma unroll
  for (uint32_t i = 0; i < kD / 32; ++i) {
    piece_t* const at = reinterpret_cast<piece_t*>(lds + threadIdx.x * (kD / 2) + i * 16);
    u32x4 v = *at;
    uint32_t none = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) none |= ((v[k] & kExponents) + kCarry) & 0x80008000u;  // an exponent of ones carries into the sign's place
    if (none) {
      bad = true;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t n = ((v[k] & kExponents) + kCarry) & 0x80008000u;
        v[k] &= ~((n >> 15) * 0xFFFFu);
      }
      *at = v;
    }
  }
  return bad;
}
__device__ __forceinline__ void mark_rows(bool bad, float* marks) {
  const uint64_t all = __ballot(bad);
  if ((threadIdx.x & 3u) == 0) marks[threadIdx.x / 4] = (all >> (threadIdx.x & 60u)) & 15u ? __builtin_nanf("") : 0.0f;
}
__device__ __forceinline__ void clean_done() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }
// Marks of the rows that a result's registers 4 q.. stand for.
__device__ __forceinline__ f32x4 marks_of(const float* marks, uint32_t r, uint32_t q) {
  return *reinterpret_cast<const f32x4*>(marks + 32 * r + 8 * q + 4 * ((threadIdx.x & 63u) >> 5));
}

// ---- which rows -----------------------------------------------------------------------------------------------------------
// A workgroup takes 128 rows of a sequence: queries from the last ones on, keys from the first (those have the most to do under a causal
// mask).
struct OwnTile {
  uint32_t sequence, row0;  // its first row inside the sequence
};
struct OwnTileMemory {
  uint32_t sums[kTileWaves];
  OwnTile found;
};
// Number `want`, from the end or from the first. By the whole workgroup; false: there are fewer. Of sequences that follow each other all
// tiles are below 2^25; spans that overlap (first not ascending) may have more than 32 bits count, which the sums keep to: then there is none.
template <bool kFromEnd>
__device__ __forceinline__ bool find_own_tile(const int32_t* first, uint32_t n, uint32_t rows, uint32_t want, OwnTileMemory& m, OwnTile& out) {
  const uint32_t t = threadIdx.x, lane = t & 63u, wave = t >> 6, per = (n + 64 * kTileWaves - 1) / (64 * kTileWaves);
  const uint32_t i0 = min(t * per, n), i1 = min(i0 + per, n);
  uint32_t sum = 0;
  for (uint32_t i = i0; i < i1; ++i) sum = add_sat(sum, (span_of(first, i, rows).count + kTileOwn - 1) / kTileOwn);
  uint32_t upto = sum;
#pragma unroll
  for (uint32_t s = 1; s < 64; s <<= 1) {
    const uint32_t o = __shfl_up(upto, s, 64);
    if (lane >= s) upto = add_sat(upto, o);
  }
  if (lane == 63) m.sums[wave] = upto;
  __syncthreads();
  uint32_t all = 0, before = upto - sum;
#pragma unroll
  for (uint32_t w = 0; w < kTileWaves; ++w) {
    all = add_sat(all, m.sums[w]);
    if (w < wave) before += m.sums[w];
  }
  if (want >= all || all >> 31) return false;
  if (kFromEnd) want = all - 1 - want;
  if (want >= before && want < before + sum) {
    uint32_t at = want - before;
    for (uint32_t i = i0; i < i1; ++i) {
      const uint32_t have = (span_of(first, i, rows).count + kTileOwn - 1) / kTileOwn;
      if (at < have) {
        m.found = {i, at * kTileOwn};
        break;
      }
      at -= have;
    }
  }
  __syncthreads();
  out = {uint32_t(__builtin_amdgcn_readfirstlane(m.found.sequence)), uint32_t(__builtin_amdgcn_readfirstlane(m.found.row0))};  // (the same in every lane)
  return true;
}
// Tiles of `rows` rows in n sequences, at most.
inline uint64_t own_tiles_at_most(uint32_t n, uint32_t rows) { return (n < rows ? n : rows) + uint64_t(rows) / kTileOwn; }

// The head of a workgroup: workgroups of one XCD (every eighth) take neighbouring heads, which share keys and values in its L2.
__device__ __forceinline__ uint32_t head_of_group(uint32_t i, uint32_t heads) { return heads % 8 == 0 ? (i % 8) * (heads / 8) + i / 8 : i; }

// 4 consecutive values to an output row.
template <class T, bool kAligned>
__device__ __forceinline__ void put4(u16* p, float a, float b, float c, float d) {
  typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
  const u32x2 v = {pack2<T>(a, b), pack2<T>(c, d)};
  if constexpr (kAligned) {
    *reinterpret_cast<u32x2*>(p) = v;
  } else {
    p[0] = u16(v[0]), p[1] = u16(v[0] >> 16), p[2] = u16(v[1]), p[3] = u16(v[1] >> 16);
  }
}
// A result of the second kind, columns 32 t.. of head_dim x this wave's rows, times `by`.
template <class T, int kD, bool kAligned>
__device__ __forceinline__ void put_columns(const tsa_heads& h, uint64_t row, uint32_t head, uint32_t dim, const f32x16 (&v)[kD / 32], float by) {
  u16* p = const_cast<u16*>(row_of<u16>(h, row, head));
#pragma unroll
  for (uint32_t t = 0; t < kD / 32; ++t)
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {
      const uint32_t d = 32 * t + 8 * i + 4 * ((threadIdx.x & 63u) >> 5);
      if (d < dim) put4<T, kAligned>(p + d, v[t][4 * i] * by, v[t][4 * i + 1] * by, v[t][4 * i + 2] * by, v[t][4 * i + 3] * by);
    }
}

}  // namespace op
}  // namespace tsa
