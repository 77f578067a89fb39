// What the gated feed-forward blocks' forward and backward passes share: the pairs (row, j) of a call grouped by expert, where
// experts' weights are, tiles over an expert's pairs, and the sum over a row's pairs.
#pragma once

#include "op_tile.hpp"

namespace tsa {

// Groups the pairs of `ids` by expert into p (its arrays in the workspace), tiles of rows_per_tile pairs of one expert.
int launch_plan(const ExpertMap& e, const int32_t* ids, const Plan& p, uint32_t rows_per_tile, hipStream_t s);

namespace op {
namespace {

// What ss_dg_slot gives for id e (below m.n), with its loads at once instead of one behind the other's test: they stand in
// front of every product of a decode step.
__device__ __forceinline__ int32_t slot_of(const ExpertMap& m, uint32_t e) {
  const ss_dg_device_view& v = m.view;
  const uint32_t abort = __hip_atomic_load(v.abort, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  const uint32_t base = v.unit_base[m.gated], end = v.unit_base[m.gated + 1];
  const bool in = e < end - base;
  const int32_t s = in ? __hip_atomic_load(v.slot_of + base + e, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 0;
  if (abort || !in) return int32_t(v.guard_slot);
  if (s >= 0) return s;
  if (v.absent_err) atomicOr(v.absent_err, 1u);  // (null where the view's version has none)
  return int32_t(v.guard_slot);
}

__device__ __forceinline__ void part_pointers(const ExpertMap& m, uint32_t e, const char* (&p)[3]) {
  if (m.form == 2) {
    const uint64_t s = uint32_t(slot_of(m, e));
    for (int i = 0; i < 3; ++i) p[i] = static_cast<const char*>(m.view.parts[i].base) + s * m.view.parts[i].stride;
  } else if (m.form == 1) {
    for (int i = 0; i < 3; ++i) p[i] = reinterpret_cast<const char*>(m.table[e]) + m.stride[i];
  } else {
    for (int i = 0; i < 3; ++i) p[i] = m.part[i] + e * m.stride[i];
  }
}

// The expert of a pair, or ~0: an id out of range, or a table entry of 0.
__device__ __forceinline__ uint32_t expert_of(const ExpertMap& m, const int32_t* ids, uint32_t pair) {
  const uint32_t e = ids ? uint32_t(ids[pair]) : 0;
  if (e >= m.n || (m.form == 1 && m.table[e] == 0)) return ~0u;
  return e;
}

// One tile's expert and rows (rows_per_tile of the plan); false behind the last tile.
struct TileRows {
  uint32_t tile, e, first, rows;
  const uint32_t* map;
};
__device__ __forceinline__ bool tile_rows(const Plan& p, uint32_t tile, uint32_t rows_per_tile, TileRows& t) {
  if (tile >= *p.n_tiles) return false;
  t.tile = tile;
  t.e = p.tile[2 * tile];
  t.first = p.tile[2 * tile + 1];
  const uint32_t end = p.first[t.e + 1];
  t.rows = end - t.first < rows_per_tile ? end - t.first : rows_per_tile;
  t.map = p.row + t.first;
  return true;
}

// ---- any stride and alignment: 64 x 64 tiles ------------------------------------------------------------------------
template <class T, bool kQ4, class B>
__device__ __forceinline__ void weight_tile(const char* w, uint64_t rows, uint32_t n, uint32_t r0, const B& x, TileMemory& m,
                                            f32x4 (&acc)[2][2]) {
  if constexpr (kQ4) {
    const Q4Operand<T> a{reinterpret_cast<const unsigned char*>(w), uint64_t(n / kQ4Block) * kQ4Bytes, uint32_t(rows), n};
    tile64<T, true>(a, r0, x, 0, n, m, acc);
  } else {
    const Operand a{reinterpret_cast<const u16*>(w), n, 1, uint32_t(rows), n, nullptr};
    tile64<T, false>(a, r0, x, 0, n, m, acc);
  }
}

// ---- tiles of pairs of an expert ---------------------------------------------------------------------------------------

// The plan's tile and the a-tile of a workgroup, over the tiles there are (known on the device only).
template <class S>
__device__ __forceinline__ bool tile_of(const Plan& p, uint32_t na, TileRows& t, uint32_t& a) {
  if (blockIdx.x >= na * *p.n_tiles) return false;
  const TileAt at = tile_at(blockIdx.x, na, *p.n_tiles);
  a = at.a;
  return tile_rows(p, at.b, S::kB, t);
}

// 4 values next to each other a lane, to rows of 32 bits.
struct FloatRows {
  struct Fetched {};
  float* out;
  uint64_t stride;
  uint32_t rows, c0, n_cols, c = 0;
  __device__ __forceinline__ void columns(uint32_t a) { c = c0 + a; }
  __device__ __forceinline__ Fetched fetch(uint32_t) const { return {}; }
  __device__ __forceinline__ void finish(uint32_t r, f32x4 v, const Fetched&) const {
    if (r < rows && c < n_cols) *reinterpret_cast<f32x4*>(out + r * stride + c) = v;  // (columns are a multiple of 8)
  }
};

// A wave's part of a tile to rows of what is held (stride and columns multiples of 8): out is the first row, c0 the tile's first column.
template <class T, int NI, int MJ>
__device__ __forceinline__ void hand_out_held(void* memory, const f32x4 (&acc)[NI][MJ], held<T>* out, uint64_t stride, uint32_t rows,
                                              uint32_t c0, uint32_t n_cols) {
  if constexpr (std::is_same_v<T, F16>) {
    FloatRows o{out, stride, rows, c0, n_cols};
    hand_out<NI, MJ>(memory, acc, o);
  } else {
    hand_out_bits<T, NI, MJ>(memory, acc, out + c0, stride, rows, n_cols - c0);
  }
}

// Gate and up rows of the same 16 NI columns as one operand of 32 NI: each wave gets 8 NI of both.
template <int NI>
__device__ __forceinline__ TileRowsSource<NI> gate_up_source(const Plan& p, const TileRows& t, uint32_t d, uint32_t f,
                                                             uint32_t f0) {
  const u16 *gate = reinterpret_cast<const u16*>(p.part[3 * t.e]), *up = reinterpret_cast<const u16*>(p.part[3 * t.e + 1]);
  return TileRowsSource<NI>(d, threadIdx.x >> 6 & 1u, [&](uint32_t r) {
    const uint32_t c = f0 + r / (16 * NI) * (8 * NI) + r % (8 * NI);
    return (r % (16 * NI) >= 8 * NI ? up : gate) + uint64_t(c < f ? c : f - 1) * d;
  });
}
template <int MJ>
__device__ __forceinline__ TileRowsSource<MJ> mapped_rows(const TileRows& t, const u16* x, uint64_t stride, uint32_t n) {
  return TileRowsSource<MJ>(n, threadIdx.x >> 7, [&](uint32_t r) { return x + t.map[r < t.rows ? r : t.rows - 1] * stride; });
}
template <int MJ>
__device__ __forceinline__ TileRowsSource<MJ> sorted_rows(const TileRows& t, const u16* x, uint64_t stride, uint32_t n) {
  return TileRowsSource<MJ>(n, threadIdx.x >> 7,
                            [&](uint32_t r) { return x + uint64_t(t.first + (r < t.rows ? r : t.rows - 1)) * stride; });
}

// out_t = residual_t + sum_j w_tj scale_{at(t, j)} v_{at(t, j)}, in the order of j; kWide columns a thread (a multiple of 4: one access each).
// By blocks first.. of `n_blocks` of 256 threads.
struct Combine {
  Plan p;
  uint32_t rows = 0, d = 0, n_blocks = 0;
  const float *v = nullptr, *weights = nullptr;
  const float* scale = nullptr;  // of the sorted positions' v (null: 1)
  const u16* residual = nullptr;
  uint64_t residual_stride = 0;
  u16* out = nullptr;
  uint64_t out_stride = 0;
};
template <class T, int kWide>
__device__ __forceinline__ void combine(const Combine& a, uint32_t block) {
  const Plan& p = a.p;
  const float *v = a.v, *weights = a.weights;
  const u16* residual = a.residual;
  u16* out = a.out;
  const uint64_t residual_stride = a.residual_stride, out_stride = a.out_stride;
  const uint32_t d = a.d, per = d / kWide;
  const uint64_t total = uint64_t(a.rows) * per;
  for (uint64_t i = uint64_t(block) * 256 + threadIdx.x; i < total; i += uint64_t(a.n_blocks) * 256) {
    const uint32_t row = uint32_t(i / per), c = uint32_t(i % per) * kWide;
    float s[kWide];
    if constexpr (kWide == 4) {
      const bits4 r = residual ? *reinterpret_cast<const bits4*>(residual + row * residual_stride + c) : bits4{0, 0, 0, 0};
#pragma unroll
      for (int q = 0; q < 4; ++q) s[q] = T::up(r[q]);
    } else {
      s[0] = residual ? T::up(residual[row * residual_stride + c]) : 0.0f;
    }
    for (uint32_t j0 = 0; j0 < p.top_k; j0 += 4) {  // four at once: one after the other each is a memory latency
      int32_t at[4];
      float w[4], x[4][kWide];
#pragma unroll
      for (uint32_t j = 0; j < 4; ++j) {
        const uint64_t pair = uint64_t(row) * p.top_k + j0 + j;
        at[j] = j0 + j < p.top_k ? p.at[pair] : -1;
        w[j] = j0 + j < p.top_k && weights ? weights[pair] : 1.0f;
      }
#pragma unroll
      for (uint32_t j = 0; j < 4; ++j) {
        const uint32_t pos = uint32_t(at[j] < 0 ? 0 : at[j]);
        const float* from = v + uint64_t(pos) * d + c;
        if (a.scale) w[j] *= at[j] < 0 ? 1.0f : a.scale[pos];
        if constexpr (kWide == 4) {
          const f32x4 y = at[j] >= 0 ? *reinterpret_cast<const f32x4*>(from) : f32x4{0, 0, 0, 0};
#pragma unroll
          for (int q = 0; q < 4; ++q) x[j][q] = y[q];
        } else {
          x[j][0] = at[j] >= 0 ? *from : 0.0f;
        }
      }
#pragma unroll
      for (uint32_t j = 0; j < 4; ++j)
        if (at[j] >= 0)
#pragma unroll
          for (int q = 0; q < kWide; ++q) s[q] += w[j] * x[j][q];
    }
    if constexpr (kWide == 4) {
      bits4 o;
#pragma unroll
      for (int q = 0; q < 4; ++q) o[q] = T::down(s[q]);
      *reinterpret_cast<bits4*>(out + row * out_stride + c) = o;
    } else {
      out[row * out_stride + c] = T::down(s[0]);
    }
  }
}

// ---- the workspace --------------------------------------------------------------------------------------------------
struct Room {
  uint64_t bytes = 0;
  char* base;
  explicit Room(void* p) : base(static_cast<char*>(p)) {}
  template <class V>
  V* take(uint64_t n) {
    V* p = reinterpret_cast<V*>(base + bytes);
    bytes += up_to(n * sizeof(V), 256);
    return p;
  }
};

uint32_t most_tiles(uint32_t pairs, uint32_t n, uint32_t rows_per_tile) {
  return pairs / rows_per_tile + (n < pairs ? n : pairs);
}

// Pairs that one workgroup groups (a multiple of 1024); more than kPlanMost times as many are shared by at most so many workgroups.
constexpr uint32_t kPlanOne = 2048, kPlanMost = 64;

Plan take_plan(Room& r, uint32_t n, uint32_t pairs, uint32_t top_k, uint32_t rows_per_tile) {
  Plan p;
  p.part = r.take<const char*>(uint64_t(3) * n);
  p.first = r.take<uint32_t>(n + 1);
  p.pair = r.take<uint32_t>(pairs);
  p.row = r.take<uint32_t>(pairs);
  p.at = r.take<int32_t>(pairs);
  p.tile = r.take<uint32_t>(uint64_t(2) * most_tiles(pairs, n, rows_per_tile));
  p.n_tiles = r.take<uint32_t>(1);
  p.pairs = pairs;
  p.stretch = pairs > kPlanOne ? kPlanOne : pairs;
  const bool many = pairs > kPlanMost * kPlanOne;
  if (many) p.stretch = uint32_t(up_to((pairs + kPlanMost - 1) / kPlanMost, 1024));
  p.groups = pairs > kPlanOne ? (pairs + p.stretch - 1) / p.stretch : 1;
  // (kPlanMost of them however few there are: a workspace that holds a call holds every one of fewer rows)
  p.counts = r.take<uint32_t>(p.groups > 1 ? uint64_t(many ? kPlanMost : p.groups) * n : 0);
  p.top_k = top_k;
  p.n = n;
  return p;
}

uint32_t blocks(uint64_t n) { return uint32_t(n < (1u << 20) ? n : (1u << 20)); }

// Which tile the pairs' products take. A big tile's workgroup alone on a CU waits for its loads: below about 150 of them (128
// pairs by 192 columns, half a tile more for every expert) small ones are as fast or faster, above they read too much; and
// with fewer than about 24 pairs an expert most of a big tile is empty. Big and small, forward: 600 rows, 2 of 8 experts of
// 2048 x 1024 (147): 78 and 62 us; 1200 rows, 2048 x 2048 (253): 141 and 179; 400 rows of one expert of 4096 x 8192 (88): 241 and
// 196; 8 of 128 experts of 2048 x 768, 32 rows: 160 and 146, 256: 284 and 269, 512: 298 and 308. Gradients: 300 rows of one
// expert of 2048 x 2048 (33): 165 and 107 us; 2000 rows, 2048 x 4096 (176): 392 and 470.
inline bool small_tiles(uint32_t rows, uint32_t top_k, uint32_t n, uint32_t d, uint32_t f) {
  const uint64_t pairs = uint64_t(rows) * top_k, tiles = pairs / 128 + (n < pairs ? n + 1 : pairs + 1) / 2;
  return pairs < uint64_t(24) * n || tiles * (((d < f ? d : f) + BigTile::kA - 1) / BigTile::kA) < 150;
}

// The sum's arguments; wide: whether four columns a thread can be.
inline Combine combine_of(const Plan& p, uint32_t rows, uint32_t d, const float* v, const float* weights, const void* residual,
                          uint64_t residual_stride, void* out, uint64_t out_stride, bool& wide) {
  const uint64_t odd = reinterpret_cast<uintptr_t>(residual) | 2 * residual_stride | reinterpret_cast<uintptr_t>(out) | 2 * out_stride;
  wide = d % 4 == 0 && odd % 8 == 0;
  Combine c;
  c.p = p;
  c.rows = rows;
  c.d = d;
  c.n_blocks = blocks((uint64_t(rows) * (wide ? d / 4 : d) + 255) / 256);
  c.v = v;
  c.weights = weights;
  c.residual = static_cast<const u16*>(residual);
  c.residual_stride = residual_stride;
  c.out = static_cast<u16*>(out);
  c.out_stride = out_stride;
  return c;
}

bool aligned16(const void* p, uint64_t stride_bytes) { return (reinterpret_cast<uintptr_t>(p) | stride_bytes) % 16 == 0; }

// Whether every weight row, x row and row of h starts 16-byte aligned and holds whole groups of 8 values. The addresses of
// a table's units are the device's: that they are 16-byte aligned is the caller's part (the library lays units out at the
// descriptor's unit_align, 256 by default).
bool wide_weights(const ExpertMap& e) {
  for (int p = 0; p < 3; ++p) {
    if (e.form == 0 && !aligned16(e.part[p], e.stride[p])) return false;
    if (e.form == 1 && e.stride[p] % 16) return false;
    if (e.form == 2 && !aligned16(e.view.parts[p].base, e.view.parts[p].stride)) return false;
  }
  return true;
}
bool wide_rows(const ExpertMap& e, uint32_t d, uint32_t f, bool q4, const void* x, uint64_t x_stride) {
  if (d % 8 || f % 8 || !aligned16(x, 2 * x_stride) || x_stride >= 1u << 24) return false;
  return q4 || wide_weights(e);
}

}  // namespace
}  // namespace op
}  // namespace tsa
