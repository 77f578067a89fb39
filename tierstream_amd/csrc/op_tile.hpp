// Products with many rows: tiles of 32 NI rows of `a` times 32 MJ rows of `b`, by four waves (2 x 2, each 16 NI x 16 MJ) whose
// accumulators stay in registers, two workgroups to a CU. Both operands go through LDS: waves of 128 x 64 read 96 KiB there for
// the 64 matrix instructions of a SIMD, and 48 are written, 9/8 of what LDS moves in their time.
//
// A step is 32 values of the sum. Its operands are loaded straight to LDS (global_load_lds_dwordx4, NB buffers in turn) and
// from there to a second set of registers while the step before is multiplied. Two steps, a cache line of every row, are
// loaded together: by themselves each took the lines' halves from L2 again (a quarter of the time of a long product).
// With 3 buffers, so that two workgroups of the big tile fit a CU, step t (even) loads t + 2 and t + 3, behind a barrier and
// over t - 1 and t, whose reads every wave has done, and step t + 1 waits for them. With more, step t (odd) waits for steps
// t + 1 and t + 2 and behind its barrier loads t + NB - 1 and t + NB over t - 1 and t.
//
// Operands come in two forms. Rows: the values of the sum lie next to each other; a row's 64 bytes a step are 4 pieces,
// piece c at place c ^ (row / 2 mod 4), so that the lanes reading one piece of 16 rows hit all banks
// (with row / 4 in its place the reads took twice the cycles: 4.4e7 of conflicts in one long product, now none). Columns (the operand
// is transposed in memory): 32 rows of the tile's columns, read with ds_read_b64_tr_b16, which gives each lane of 16 one
// column of 4 rows; pairs of pieces are permuted by the row so that the 8 rows of a half wave hit all banks. In both, the
// permutation is made by the loads' addresses: LDS itself is filled in lane order.
//
// 2047 rows through 4096 x 28672 with bias, tanh gelu and residual: 520 us, 920 TFLOP/s (970 in a product of 2048 rows without
// them; 1065 with operands of zeros, which take less power). What bounds it are the loads: without them the loop runs at 1625,
// with one operand always in L2 at 1075; the matrix cores are busy 44 % of the time, L2 gives 12.7 TB/s. Tried without gain: 256 x 256 by eight waves (a third less from L2, but one workgroup a
// CU, whose epilogue stands alone: 517 us for 496), lines sent for to L2 six steps ahead, buffers of whole lines (552 for 523),
// priorities.
#pragma once

#include "op_device.hpp"

namespace tsa {
namespace op {

constexpr uint32_t kTileThreads = 256;

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4_t;
typedef __attribute__((address_space(3))) const bits8 lds_bits8_t;

__device__ __forceinline__ void meet() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }
template <int N>
__device__ __forceinline__ void wait_loads_and_meet() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

// An operand of 32 NF rows, in rows: at(r) gives row r's first value (any valid row for r behind the last).
template <int NF>
struct TileRowsSource {
  static constexpr int kLoads = NF / 2;
  const u16* p[kLoads];
  uint32_t k, n, mine;
  uint32_t frag;  // this lane's place of its wave's first fragment

  template <class At>
  __device__ __forceinline__ TileRowsSource(uint32_t n_, uint32_t half, At&& at) : n(n_) {
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    mine = __builtin_amdgcn_readfirstlane(wave) * kLoads * 1024;
    k = ((lane & 3u) ^ ((lane >> 3) & 3u)) * 8;
#pragma unroll
    for (int j = 0; j < kLoads; ++j) p[j] = at((wave * kLoads + j) * 16 + lane / 4) + k;
    frag = (half * NF * 16 + (lane & 15u)) * 64 + (((lane >> 4) ^ ((lane >> 1) & 3u)) * 16);
  }
  // Load j of the next two steps (kCheck: the sum may end inside them); then, after all of them, on to the two behind.
  template <bool kCheck>
  __device__ __forceinline__ void issue(int j, uint32_t lds0, uint32_t lds1) {
    if (kCheck) {
      load_to_lds(k < n ? static_cast<const void*>(p[j]) : &kZeroPiece, lds0 + mine + j * 1024);
      load_to_lds(k + 32 < n ? static_cast<const void*>(p[j] + 32) : &kZeroPiece, lds1 + mine + j * 1024);
    } else {
      load_to_lds(p[j], lds0 + mine + j * 1024);
      load_to_lds(p[j] + 32, lds1 + mine + j * 1024);
    }
    p[j] += 64;
  }
  __device__ __forceinline__ void advance() { k += 64; }
  __device__ __forceinline__ void stage(uint32_t, uint32_t) {}
  __device__ __forceinline__ bits8 read(uint32_t lds, int i) const {
    return *reinterpret_cast<lds_bits8_t*>(lds + frag + i * 1024);
  }
};

// Rows of 4-bit blocks: 128 weight rows as 256 rows of the tile, 64 of each wave's half the values' leading 16 bits and 64
// what is left of them. A value (q - 8) s has 15 bits, so both together are exact: bf16 takes the value itself, half
// precision an eighth of it (no scale overflows) and 2^12 times the rest (none underflows). whole() joins the two sums.
// A thread takes one block of a row every two steps: from memory to registers two steps ahead, then to LDS in the places
// where loads put rows.
template <class T>
struct TileQ4Source {
  static constexpr int kLoads = 0;
  static constexpr bool kHalf = std::is_same_v<T, F16>;
  const unsigned char* p;
  uint32_t k, n, put, turn, frag;
  u32x4 v;
  u16 scale;

  typedef u32x4 words_any __attribute__((aligned(2)));
  typedef __attribute__((address_space(1))) const words_any gwords_t;
  typedef __attribute__((address_space(1))) const u16 ghalf_t;
  typedef __attribute__((address_space(3))) bits8 lds_put_t;

  template <class At>
  __device__ __forceinline__ TileQ4Source(uint32_t n_, uint32_t half, At&& at) : n(n_) {
    const uint32_t lane = threadIdx.x & 63u, r = threadIdx.x / 2, second = threadIdx.x & 1u;
    p = at(r) + second * kQ4Bytes;
    k = second * kQ4Block;
    const uint32_t row = (r / 64) * 128 + r % 64;
    put = row * 64;
    turn = (row >> 1) & 3u;
    frag = (half * 128 + (lane & 15u)) * 64 + (((lane >> 4) ^ ((lane >> 1) & 3u)) * 16);
    fetch();
  }
  __device__ __forceinline__ void fetch() {
    v = u32x4{0, 0, 0, 0};
    scale = 0;
    if (k < n) {
      const uintptr_t at = reinterpret_cast<uintptr_t>(p);
      scale = *reinterpret_cast<ghalf_t*>(at);
      v = *reinterpret_cast<gwords_t*>(at + 2);
    }
    p += 2 * kQ4Bytes;
    k += 2 * kQ4Block;
  }
  template <bool kCheck>
  __device__ __forceinline__ void issue(int, uint32_t, uint32_t) {}
  __device__ __forceinline__ void advance() {}
  // The fetched blocks to the buffers of their two steps, and the next ones from memory.
  __device__ __forceinline__ void stage(uint32_t lds0, uint32_t lds1) {
    const uint32_t to = (threadIdx.x & 1u ? lds1 : lds0) + put;
    const float s = F16::up(scale) * (kHalf ? 0.125f : 1.0f), s8 = -8.0f * s;
#pragma unroll
    for (uint32_t c = 0; c < 4; ++c) {  // values 8 c..: bytes 8 (c mod 2).. of the block, low halves first
      bits8 hi, lo;
#pragma unroll
      for (uint32_t i = 0; i < 8; ++i) {
        const uint32_t byte = 8 * (c & 1u) + i, q = (v[byte / 4] >> (8 * (byte & 3u) + 4 * (c >> 1))) & 15u;
        const float w = __builtin_fmaf(float(q), s, s8);  // exact
        hi[i] = T::down(w);
        lo[i] = T::down((w - T::up(hi[i])) * (kHalf ? 4096.0f : 1.0f));
      }
      *reinterpret_cast<lds_put_t*>(to + ((c ^ turn) * 16)) = hi;
      *reinterpret_cast<lds_put_t*>(to + 64 * 64 + ((c ^ turn) * 16)) = lo;
    }
    fetch();
  }
  __device__ __forceinline__ bits8 read(uint32_t lds, int i) const {
    return *reinterpret_cast<lds_bits8_t*>(lds + frag + i * 1024);
  }
  static __device__ __forceinline__ f32x4 whole(f32x4 hi, f32x4 lo) {
    return kHalf ? (hi + lo * (1.0f / 4096)) * 8.0f : hi + lo;
  }
};

__device__ __forceinline__ uint64_t uniform(uint64_t v) {
  return uint64_t(uint32_t(__builtin_amdgcn_readfirstlane(uint32_t(v >> 32)))) << 32 |
         uint32_t(__builtin_amdgcn_readfirstlane(uint32_t(v)));
}
// 64 lanes x 16 bytes from one base (the same in every lane) and a 32-bit offset each.
__device__ __forceinline__ void load_offset_to_lds(uint64_t base, uint32_t offset, uint32_t at) {
  asm volatile(
      "s_mov_b32 m0, %2\n\t"
      "s_nop 0\n\t"
      "global_load_lds_dwordx4 %0, %1"
      :
      : "v"(offset), "s"(base), "s"(at)
      : "memory", "m0");
}

// A map in LDS is a ring of kMapRing entries, refilled half by half while the sum goes on.
constexpr uint32_t kMapRing = 2048;

// In columns: 32 NF columns from `first` on (n_cols in all, a multiple of 8), row k of the sum at at + k stride, or with a
// map (in LDS) at at + map[k] stride. stride is below 2^24. Buffers are 512-byte aligned: a fragment's place is its wave's
// first one's with the fragment's number in three bits that the permutation turns.
template <int NF, bool kMap>
struct TileColumnsSource {
  static constexpr int kLoads = NF / 2;
  static constexpr uint32_t kPieces = 4 * NF;  // 16-byte pieces of a row
  static constexpr bool kEven = (kPieces & (kPieces - 1)) == 0;  // rows of 256 bytes or a power of two of it; else of 128 more
  uint64_t base;
  uint32_t offset[kLoads];  // bytes: of the lane's column, and without a map of its row
  uint32_t stride, k, n, mine, frag[kEven ? 1 : NF];
  const uint32_t* map;

  static __device__ __forceinline__ uint32_t turn(uint32_t kk) {
    return kEven ? (((kk & 3u) | ((kk >> 3) & 1u) << 2) << 1) & (kPieces - 1) : ((kk >> 1 & 1u) | ((kk >> 3) & 1u) << 1) << 1;
  }
  __device__ __forceinline__ TileColumnsSource(uint32_t n_, uint32_t half, const u16* at, uint64_t stride_, uint32_t first,
                                               uint32_t n_cols, const uint32_t* map_ = nullptr)
      : base(uniform(reinterpret_cast<uint64_t>(at))), stride(uint32_t(stride_) * 2), k(0), n(n_), map(map_) {
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    mine = __builtin_amdgcn_readfirstlane(wave) * kLoads * 1024;
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
      const uint32_t i = (wave * kLoads + j) * 64 + lane;
      const uint32_t c = first + ((i % kPieces) ^ turn(i / kPieces)) * 8;
      offset[j] = (c < n_cols ? c : n_cols - 8) * 2 + (kMap ? 0 : i / kPieces * stride);
    }
    const uint32_t kk = (lane >> 4) * 8 + ((lane & 15u) >> 2);
#pragma unroll
    for (int i = 0; i < (kEven ? 1 : NF); ++i)
      frag[i] = kk * (kPieces * 16) + ((half * NF * 2 + 2 * i + ((lane & 3u) >> 1)) ^ turn(kk)) * 16 + (lane & 1u) * 8;
  }
  __device__ __forceinline__ uint32_t row_of(int j) const {  // of the lane's piece, in its step
    return (mine + j * 1024 + (threadIdx.x & 63u) * 16) / (kPieces * 16);
  }
  // Load j of the next two steps, as TileRowsSource's.
  template <bool kCheck>
  __device__ __forceinline__ void issue(int j, uint32_t lds0, uint32_t lds1) {
#pragma unroll
    for (uint32_t s = 0; s < 2; ++s) {
      const uint32_t to = (s ? lds1 : lds0) + mine + j * 1024;
      if constexpr (kMap || kCheck) {
        const uint32_t row = k + 32 * s + row_of(j);
        const bool in = !kCheck || row < n;
        uint64_t g = base + offset[j];
        if constexpr (kMap) g += uint64_t(map[in ? row % kMapRing : 0]) * stride;
        else g += uint64_t(32 * s) * stride;
        load_to_lds(in ? reinterpret_cast<const void*>(g) : &kZeroPiece, to);
      } else {
        load_offset_to_lds(base + uint64_t(32 * s) * stride, offset[j], to);
      }
    }
  }
  __device__ __forceinline__ void advance() {
    k += 64;
    if (!kMap) base += uint64_t(64) * stride;
  }
  __device__ __forceinline__ void stage(uint32_t, uint32_t) {}
  __device__ __forceinline__ bits8 read(uint32_t lds, int i) const {
    const uint32_t at = kEven ? (lds + frag[0]) ^ (32u * i) : lds + frag[kEven ? 0 : i];
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lds_s16x4_t*>(at));
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lds_s16x4_t*>(at + 4 * kPieces * 16));
    return __builtin_bit_cast(bits8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
  }
};

constexpr uint32_t tile_lds(int NI, int MJ, int NB) { return uint32_t(NI + MJ) * 2048u * uint32_t(NB); }

// A tile: 32 NI rows of a, 32 MJ rows of b, NB buffers.
template <int NI_, int MJ_, int NB_>
struct TileShape {
  static constexpr int NI = NI_, MJ = MJ_, NB = NB_;
  static constexpr uint32_t kA = 32 * NI, kB = 32 * MJ, kLds = tile_lds(NI, MJ, NB);
};
typedef TileShape<6, 4, 4> BigTile;
typedef TileShape<8, 4, 3> WideTile;
typedef TileShape<2, 2, 8> SmallTile;

// Every accumulator through an empty statement: what is written before it is not read, and what is read after it not
// written, on the other side. The compiler counts no wait states behind assembly, so they stand beside it.
template <int NI, int MJ>
__device__ __forceinline__ void settle(f32x4 (&acc)[NI][MJ]) {
#pragma unroll
  for (int i = 0; i < NI; ++i)
#pragma unroll
    for (int j = 0; j < MJ; ++j) asm volatile("" : "+a"(acc[i][j]));
}

// acc[i][j] += a's rows 16 i.. of this wave's half times b's rows 16 j.. of its half, over the sources' n values. Lane l
// holds a-rows 4 (l / 16) + 0..3 and b-row l % 16 of each.
// every_two(k): behind the barrier of each second step (3 buffers), when every wave has issued the loads of the values below
// k + 64.
struct Nothing {
  __device__ __forceinline__ void operator()(uint32_t) const {}
};
template <class T, int NI, int MJ, int NB, class A, class B, class F = Nothing>
__device__ __forceinline__ void tile_product(A& a, B& b, uint32_t n, uint32_t lds, f32x4 (&acc)[NI][MJ], F&& every_two = F{}) {
  static_assert(NB == 3 || (NB >= 4 && NB % 2 == 0), "buffers");
  constexpr int kLoads = A::kLoads + B::kLoads;  // of a step, each thread
  constexpr uint32_t kA = NI * 2048, kBuffer = (NI + MJ) * 2048;
  const auto issue = [&](auto check, int j, uint32_t at0, uint32_t at1) {  // load j of two steps, of both operands
    if (j < A::kLoads) a.template issue<decltype(check)::value>(j, at0, at1);
    else b.template issue<decltype(check)::value>(j - A::kLoads, at0 + kA, at1 + kA);
  };
  const auto issue_all = [&](uint32_t at0, uint32_t at1) {
#pragma unroll
    for (int j = 0; j < kLoads; ++j) issue(std::true_type{}, j, at0, at1);
    a.advance();
    b.advance();
  };
  __syncthreads();  // the last product's reads are done
  a.stage(lds, lds + kBuffer);
  issue_all(lds, lds + kBuffer);
#pragma unroll
  for (int i = 2; i + 1 < NB; i += 2) issue_all(lds + i * kBuffer, lds + (i + 1) * kBuffer);
  wait_loads_and_meet<NB == 3 ? 0 : (NB - 2) * kLoads>();
  bits8 fa[2][NI], fb[2][MJ];
#pragma unroll
  for (int i = 0; i < NI; ++i) fa[0][i] = a.read(lds, i);
#pragma unroll
  for (int j = 0; j < MJ; ++j) fb[0][j] = b.read(lds + kA, j);
  settle(acc);
  asm volatile("s_nop 7");
  uint32_t at = 0;  // this step's buffer
  const auto behind = [&](uint32_t steps) { return lds + (at + steps >= NB ? at + steps - NB : at + steps) * kBuffer; };
  // A step, product by product: a read of the next step's operands every kPer, the loads in between. Left to itself the
  // compiler puts the reads behind the last product, where nothing hides them.
  const auto step = [&](auto now_, auto loads, auto check) {
    constexpr int now = decltype(now_)::value, kFrags = NI + MJ, kPer = NI * MJ / kFrags;
    const uint32_t from = behind(1);
    const uint32_t to0 = NB == 3 ? behind(2) : behind(NB - 1), to1 = lds + at * kBuffer;
#pragma unroll
    for (int x = 0; x < NI * MJ; ++x) {
      if (x % kPer == 0 && x / kPer < kFrags) {
        const int r = x / kPer;
        if (r < MJ) fb[now ^ 1][r] = b.read(from + kA, r);
        else fa[now ^ 1][r - MJ] = a.read(from, r - MJ);
        if (decltype(loads)::value && r % 2 == 0 && r / 2 < kLoads) issue(check, r / 2, to0, to1);
      }
      T::mfma_in_place(acc[x / MJ][x % MJ], fa[now][x / MJ], fb[now][x % MJ]);
      if (x % kPer == kPer - 1) __builtin_amdgcn_sched_barrier(0);
    }
    if (decltype(loads)::value) {
      a.advance();
      b.advance();
    }
    at = at + 1 == NB ? 0 : at + 1;
  };
  const auto two_steps = [&](auto check, uint32_t t) {
    using Zero = std::integral_constant<int, 0>;
    using One = std::integral_constant<int, 1>;
    if (NB != 3) {
      step(Zero{}, std::false_type{}, check);
      wait_loads_and_meet<NB == 3 ? 0 : (NB - 4) * kLoads>();
      every_two(t * 32);
      step(One{}, std::true_type{}, check);
    } else {
      meet();
      every_two(t * 32);
      a.stage(behind(2), lds + at * kBuffer);
      step(Zero{}, std::true_type{}, check);
      wait_loads_and_meet<0>();
      step(One{}, std::false_type{}, check);
    }
  };
  constexpr uint32_t kAhead = NB == 3 ? 4 : NB + 2;  // the last step that two steps from t on load, + 1
  uint32_t t = 0;
  for (; (t + kAhead) * 32 <= n; t += 2) two_steps(std::false_type{}, t);
  for (; t * 32 < n; t += 2) two_steps(std::true_type{}, t);  // (steps past the end multiply zeros)
  // The loads past the end have landed, and the last results are written before anything reads them (18 wait states).
  asm volatile("s_waitcnt vmcnt(0)\n\ts_nop 15\n\ts_nop 3" ::: "memory");
  settle(acc);
}

// Hands a wave's part of a tile to `out`, 4 values of a-rows next to each other at a time, rows counted in the tile: by way
// of LDS (the wave's own JP fragments of b at a time), so that lanes next to each other have values next to each other.
// out.columns(a-row): this lane's 4 a-rows, once; out.fetch(b-row) gives what finish() of that row needs from memory, for up
// to 8 rows before the first finish(b-row, values, fetched): one after the other, each would be a memory latency.
template <int NI, int MJ, class Out>
__device__ __forceinline__ void hand_out(void* memory, const f32x4 (&acc)[NI][MJ], Out& out) {
  constexpr int JP = NI >= 6 ? MJ / 2 : MJ;  // (what the buffers hold)
  constexpr uint32_t kLanes = NI * 4, kRows = kLanes > 16 ? (kLanes > 32 ? 1 : 2) : kLanes > 8 ? 4 : 64 / kLanes;  // lanes a row, rows at once
  constexpr uint32_t kBatch = 16 * JP / kRows < 8 ? 16 * JP / kRows : 8;
  // Piece p of row r: turned by the row, so that both ways hit all banks.
  const auto place = [](uint32_t p, uint32_t r) {
    return r * kLanes + ((kLanes & (kLanes - 1)) == 0 ? p ^ (r & 15u) % kLanes : (p + (r & 15u)) % kLanes);
  };
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
  f32x4* mine = static_cast<f32x4*>(memory) + wave * (JP * 16 * kLanes);
  out.columns((wave & 1u) * 16 * NI + (lane % kLanes) * 4);
  __syncthreads();  // the product's reads are done
#pragma unroll
  for (int j0 = 0; j0 < MJ; j0 += JP) {
#pragma unroll
    for (int j = 0; j < JP; ++j)
#pragma unroll
      for (int i = 0; i < NI; ++i) mine[place(4 * i + (lane >> 4), 16 * j + (lane & 15u))] = acc[i][j0 + j];
    __builtin_amdgcn_wave_barrier();
    if (lane < kLanes * kRows)
#pragma unroll 1
      for (uint32_t r0 = lane / kLanes; r0 < 16 * JP; r0 += kBatch * kRows) {
        const uint32_t base = (wave >> 1) * 16 * MJ + 16 * j0 + r0;
        typename Out::Fetched got[kBatch];
#pragma unroll
        for (uint32_t x = 0; x < kBatch; ++x) got[x] = out.fetch(base + x * kRows);
#pragma unroll
        for (uint32_t x = 0; x < kBatch; ++x)
          out.finish(base + x * kRows, mine[place(lane % kLanes, r0 + x * kRows)], got[x]);
      }
    __builtin_amdgcn_wave_barrier();
  }
}

// A wave's part of a tile as 16-bit values to rows of `out`: through LDS as hand_out, 8 values a lane. out: the tile's first row
// and column, 16-byte aligned; rows and columns there are (columns a multiple of 8). With 4 bytes a value in LDS and 8-byte
// stores the weights' gradients of a training step of 128 experts took 535 us; straight from the registers (16 rows of 32 bytes
// a store) 644. kOnce: nothing that follows soon reads them, so they pass the caches by (1.2 GB of gradients: 492 and 461 us, and the
// next call finds its inputs there: its first product 157 and 122).
template <class T, int NI, int MJ, bool kOnce = false>
__device__ __forceinline__ void hand_out_bits(void* memory, const f32x4 (&acc)[NI][MJ], u16* out, uint64_t stride, uint32_t rows,
                                              uint32_t cols) {
  constexpr uint32_t kPieces = 2 * NI, kRows = kPieces > 8 ? 4 : kPieces > 4 ? 8 : 64 / kPieces;  // pieces a row, rows at once
  const auto place = [](uint32_t p, uint32_t r) {
    return r * kPieces + ((kPieces & (kPieces - 1)) == 0 ? p ^ r % kPieces : (p + r) % kPieces);
  };
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
  bits8* mine = static_cast<bits8*>(memory) + wave * (16 * MJ * kPieces);
  __syncthreads();  // the product's reads are done
#pragma unroll
  for (int j = 0; j < MJ; ++j)
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      bits4 v;
#pragma unroll
      for (int q = 0; q < 4; ++q) v[q] = T::down(acc[i][j][q]);
      reinterpret_cast<bits4*>(mine + place(2 * i + (lane >> 5), 16 * j + (lane & 15u)))[lane >> 4 & 1u] = v;
    }
  __builtin_amdgcn_wave_barrier();
  const uint32_t c = (wave & 1u) * 16 * NI + lane % kPieces * 8;
  if (lane < kPieces * kRows && c < cols)
#pragma unroll 4
    for (uint32_t r0 = 0; r0 < 16 * MJ; r0 += kRows) {
      const uint32_t r = r0 + lane / kPieces, row = (wave >> 1) * 16 * MJ + r;
      bits8* to = reinterpret_cast<bits8*>(out + row * stride + c);
      if (row >= rows) continue;
      if constexpr (kOnce) __builtin_nontemporal_store(mine[place(lane % kPieces, r)], to);
      else *to = mine[place(lane % kPieces, r)];
    }
}

// Which tile a workgroup takes: neighbouring workgroups go to the 8 XCDs in turn, each with a cache of its own, so each
// XCD gets a stretch of tiles, and a stretch walks 8 b-tiles by 8, a-tile after a-tile: what runs at once shares operands.
struct TileAt {
  uint32_t a, b;
};
__device__ __forceinline__ TileAt tile_at(uint32_t block, uint32_t na, uint32_t nb) {
  const uint32_t total = na * nb, per = total / 8, rest = total % 8, xcd = block % 8;
  const uint32_t id = xcd * per + (xcd < rest ? xcd : rest) + block / 8;
  const uint32_t group = id / (8 * na), first = group * 8, in = id - group * 8 * na;
  const uint32_t wide = nb - first < 8 ? nb - first : 8;
  return {in / wide, first + in % wide};
}

}  // namespace op
}  // namespace tsa
