// Gated feed-forward blocks of the chosen experts, and their gradients.
//
// The pairs (row, j) are grouped by expert first (plan_kernel, one workgroup). Then
//   forward:   h = act(gate x) * (up x) of every pair; y' = down h; y_t = residual_t + sum_j w_tj y'_tj.
//   backward:  b = down^T dy; d w = <h, b>; the two halves dg = w b up act'(gate), du = w b act(gate), and w h of every
//              pair; dx' = gate^T dg + up^T du, added over a row's pairs; d gate = dg^T x, d up = du^T x and
//              d down = dy^T (w h) over an expert's pairs.
// h, dg, du and w h are rounded once to the operands' 16 bits, as the matrix instructions take them; y' and dx' stay in
// 32 bits until the row's sum, and w is applied there or before the rounding. No sum depends on an order that changes.
#include "op_stream.hpp"
#include "op_tile.hpp"

namespace tsa {
namespace op {
namespace {

constexpr uint32_t kPlanThreads = 1024, kPlanWaves = kPlanThreads / 64;

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

// Sum of v over the threads before this one, and over all of them (kPlanThreads threads).
__device__ __forceinline__ uint32_t scan(uint32_t v, uint32_t* buf, uint32_t* total) {
  const uint32_t t = threadIdx.x;
  buf[t] = v;
  __syncthreads();
  for (uint32_t s = 1; s < kPlanThreads; s <<= 1) {
    const uint32_t o = t >= s ? buf[t - s] : 0;
    __syncthreads();
    buf[t] += o;
    __syncthreads();
  }
  const uint32_t r = buf[t] - v;
  *total = buf[kPlanThreads - 1];
  __syncthreads();
  return r;
}

// Groups the pairs by expert, stably: each wave counts its stretch of pairs per expert, the counts are summed over
// experts and waves, then each wave places its stretch 64 pairs at a time, a pair behind those of its expert in lower
// lanes. `rows_per_tile` sorted positions of one expert make a tile.
__global__ __launch_bounds__(kPlanThreads) void plan_kernel(ExpertMap m, const int32_t* ids, Plan p, uint32_t rows_per_tile) {
  extern __shared__ uint32_t lds[];
  uint32_t* buf = lds;                    // [kPlanThreads]
  uint32_t* count = lds + kPlanThreads;   // [kPlanWaves][n]
  const uint32_t t = threadIdx.x, lane = t & 63u, wave = t >> 6, n = m.n;
  for (uint32_t i = t; i < kPlanWaves * n; i += kPlanThreads) count[i] = 0;
  __syncthreads();
  const uint32_t stretch = ((p.pairs + kPlanThreads - 1) / kPlanThreads) * 64;
  const uint64_t from = uint64_t(wave) * stretch;
  for (uint32_t i = 0; i < stretch; i += 64) {
    const uint64_t pair = from + i + lane;
    if (pair >= p.pairs) break;
    const uint32_t e = expert_of(m, ids, uint32_t(pair));
    if (e != ~0u) atomicAdd(&count[wave * n + e], 1u);
  }
  __syncthreads();
  uint32_t mine = 0;
  if (t < n)
    for (uint32_t w = 0; w < kPlanWaves; ++w) mine += count[w * n + t];
  uint32_t all, tiles;
  const uint32_t first = scan(mine, buf, &all);
  const uint32_t n_tiles = (mine + rows_per_tile - 1) / rows_per_tile;
  const uint32_t tile0 = scan(n_tiles, buf, &tiles);
  if (t < n) {
    p.first[t] = first;
    uint32_t at = first;
    for (uint32_t w = 0; w < kPlanWaves; ++w) {
      const uint32_t c = count[w * n + t];
      count[w * n + t] = at;
      at += c;
    }
    if (mine) {
      const char* q[3];
      part_pointers(m, t, q);
      for (int i = 0; i < 3; ++i) p.part[3 * t + i] = q[i];
    }
    for (uint32_t i = 0; i < n_tiles; ++i) {
      p.tile[2 * (tile0 + i)] = t;
      p.tile[2 * (tile0 + i) + 1] = first + i * rows_per_tile;
    }
  }
  if (t == 0) {
    p.first[n] = all;
    *p.n_tiles = tiles;
  }
  __syncthreads();
  for (uint32_t i = 0; i < stretch; i += 64) {
    const uint64_t pair = from + i + lane;
    if (from + i >= p.pairs) break;
    const bool on = pair < p.pairs;
    const uint32_t e = on ? expert_of(m, ids, uint32_t(pair)) : ~0u;
    uint64_t same = __ballot(e != ~0u);
    for (uint32_t b = 0; b < 9; ++b) {  // (n <= 512)
      const uint64_t set = __ballot((e >> b) & 1u);
      same &= (e >> b) & 1u ? set : ~set;
    }
    uint32_t at = 0;
    if (e != ~0u) {
      at = __hip_atomic_load(&count[wave * n + e], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP) +
           uint32_t(__popcll(same & ((1ull << lane) - 1)));
      p.pair[at] = uint32_t(pair);
      p.row[at] = uint32_t(pair) / p.top_k;
    }
    __builtin_amdgcn_wave_barrier();
    if (e != ~0u && (same >> lane) == 1)  // the last lane of its expert
      __hip_atomic_store(&count[wave * n + e], at + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
    __builtin_amdgcn_wave_barrier();
    if (on) p.at[pair] = e != ~0u ? int32_t(at) : -1;
  }
}

// One tile's expert and rows (rows_per_tile of the plan); false behind the last tile.
struct TileRows {
  uint32_t e, first, rows;
  const uint32_t* map;
};
__device__ __forceinline__ bool tile_rows(const Plan& p, uint32_t tile, uint32_t rows_per_tile, TileRows& t) {
  if (tile >= *p.n_tiles) return false;
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

template <class T, bool kQ4>
__global__ __launch_bounds__(256) void gate_up_any_kernel(Plan p, const u16* x, uint64_t x_stride, uint32_t d, uint32_t f,
                                                          uint32_t act, u16* h) {
  __shared__ TileMemory m;
  const uint32_t tf = (f + 63) / 64;
  const uint32_t f0 = blockIdx.x % tf * 64;
  TileRows t;
  if (!tile_rows(p, blockIdx.x / tf, 64, t)) return;
  const Operand xs{x, x_stride, 1, t.rows, d, t.map};
  f32x4 g[2][2] = {}, u[2][2] = {};
  weight_tile<T, kQ4>(p.part[3 * t.e], f, d, f0, xs, m, g);
  weight_tile<T, kQ4>(p.part[3 * t.e + 1], f, d, f0, xs, m, u);
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) g[i][j][r] = activate(act, g[i][j][r]) * u[i][j][r];
  each64(g, [&](uint32_t i, uint32_t j, float v) {
    if (f0 + i < f && j < t.rows) h[uint64_t(t.first + j) * f + f0 + i] = T::down(v);
  });
}

template <class T, bool kQ4>
__global__ __launch_bounds__(256) void down_any_kernel(Plan p, const u16* h, uint32_t d, uint32_t f, float* out) {
  __shared__ TileMemory m;
  const uint32_t td = (d + 63) / 64;
  const uint32_t d0 = blockIdx.x % td * 64;
  TileRows t;
  if (!tile_rows(p, blockIdx.x / td, 64, t)) return;
  const Operand hs{h + uint64_t(t.first) * f, f, 1, t.rows, f, nullptr};
  f32x4 acc[2][2] = {};
  weight_tile<T, kQ4>(p.part[3 * t.e + 2], d, f, d0, hs, m, acc);
  each64(acc, [&](uint32_t i, uint32_t j, float v) {
    if (d0 + i < d && j < t.rows) out[uint64_t(t.first + j) * d + d0 + i] = v;
  });
}

// ---- few rows: the weights' bytes -------------------------------------------------------------------------------------
// The part pointers of an expert in LDS, by thread 0 of the workgroup; false (to every thread) if there is none.
__device__ __forceinline__ bool resolve(const ExpertMap& m, uint32_t e, const char* (&p)[3]) {
  if (e == ~0u) return false;
  part_pointers(m, e, p);
  return true;
}

// One row of x: pair j is blockIdx.y, h_j = w_j act(gate x) (up x) for 16 columns a workgroup.
template <class T, class W, bool kTail>
__global__ __launch_bounds__(64 * most_waves(1)) void gate_up_one_kernel(ExpertMap m, const int32_t* ids, const float* weights,
                                                                         const u16* x, uint32_t d, uint32_t f, uint32_t act,
                                                                         u16* h) {
  extern __shared__ f32x4 part[];
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  const char* p[3];
  if (!resolve(m, expert_of(m, ids, blockIdx.y), p)) return;
  const uint32_t c0 = blockIdx.x * 16 + (lane & 15u), col = c0 < f ? c0 : f - 1;
  f32x4 acc[2][1] = {};
  stream_chunks<W, 2, 1, kTail>((d + kChunk - 1) / kChunk, wave, waves, [&](uint32_t c, W (&w)[2], const u16* (&row)[1]) {
    w[0] = W(p[0], d, col, d);
    w[1] = W(p[1], d, col, d);
    row[0] = x;
    return c * kChunk;
  }, acc);
  const f32x4 v[2] = {acc[0][0], acc[1][0]};
  join_waves<2>(part, v, wave, waves, [&](auto&& sum) {
    if (wave != 0) return;
    const float g = sum(0)[0], u = sum(1)[0];
    if (lane < 16 && c0 < f) h[uint64_t(blockIdx.y) * f + c0] = T::down((weights ? weights[blockIdx.y] : 1.0f) * activate(act, g) * u);
  });
}

// The experts of one row that add something: part `which` of each and its j, in the order of j.
struct LiveExperts {
  const char* part[TSA_ROUTE_MAX_TOP_K];
  uint32_t from[TSA_ROUTE_MAX_TOP_K], n;
};
__device__ __forceinline__ void find_live(const ExpertMap& m, const int32_t* ids, uint32_t top_k, int which, LiveExperts& live) {
  const uint32_t lane = threadIdx.x;
  if (lane < 64) {
    const char* p[3];
    const bool on = lane < top_k && resolve(m, expert_of(m, ids, lane), p);
    const uint64_t has = __ballot(on);
    if (on) {
      const uint32_t i = uint32_t(__popcll(has & ((1ull << lane) - 1)));
      live.part[i] = p[which];
      live.from[i] = lane;
    }
    if (lane == 0) live.n = uint32_t(__popcll(has));
  }
  __syncthreads();
}

// y = residual + sum_j down_j h_j: one row over the chunks of all its experts.
template <class T, class W, bool kTail>
__global__ __launch_bounds__(64 * most_waves(1)) void down_one_kernel(ExpertMap m, const int32_t* ids, uint32_t top_k,
                                                                      const u16* h, uint32_t d, uint32_t f,
                                                                      const u16* residual, u16* y) {
  extern __shared__ f32x4 part[];
  __shared__ LiveExperts live;
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  find_live(m, ids, top_k, 2, live);
  const uint32_t c0 = blockIdx.x * 16 + (lane & 15u), col = c0 < d ? c0 : d - 1, per = (f + kChunk - 1) / kChunk;
  f32x4 acc[1][1] = {};
  stream_chunks<W, 1, 1, kTail>(live.n * per, wave, waves, [&](uint32_t c, W (&w)[1], const u16* (&row)[1]) {
    const uint32_t j = c / per;
    w[0] = W(live.part[j], f, col, f);
    row[0] = h + uint64_t(live.from[j]) * f;
    return (c - j * per) * kChunk;
  }, acc);
  const f32x4 v[1] = {acc[0][0]};
  join_waves<1>(part, v, wave, waves, [&](auto&& sum) {
    if (wave != 0) return;
    const float s = sum(0)[0] + (residual && c0 < d ? T::up(residual[c0]) : 0.0f);
    if (lane < 16 && c0 < d) y[c0] = T::down(s);
  });
}

// The same two with 4-bit weights by way of LDS (d and f multiples of 256, 16-byte aligned weights).
template <class T>
__global__ __launch_bounds__(64 * kQ4Waves) void gate_up_q4_kernel(ExpertMap m, const int32_t* ids, const float* weights,
                                                                   const u16* x, uint32_t d, uint32_t f, uint32_t act, u16* h) {
  extern __shared__ f32x4 memory[];
  __shared__ float part[kQ4Waves * 2 * 16];
  const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
  const char* p[3];
  if (!resolve(m, expert_of(m, ids, blockIdx.y), p)) return;
  const uint32_t c0 = blockIdx.x * 16;
  const uint64_t row = uint64_t(d / kQ4Block) * kQ4Bytes;
  float acc[2] = {};
  stream_q4<T, 2>((d + 511) / 512, wave, waves, f - c0 < 16 ? f - c0 : 16, d, lds_offset(memory) + wave * 2 * Q4Stage<2>::kBytes,
                  [&](uint32_t s, const char* (&base)[2], const u16*& xs) {
                    base[0] = p[0] + c0 * row;
                    base[1] = p[1] + c0 * row;
                    xs = x;
                    return s * 512;
                  }, acc);
  join_q4<2>(part, acc, wave, waves, [&](const float (&s)[2]) {
    if (c0 + lane < f)
      h[uint64_t(blockIdx.y) * f + c0 + lane] = T::down((weights ? weights[blockIdx.y] : 1.0f) * activate(act, s[0]) * s[1]);
  });
}

template <class T>
__global__ __launch_bounds__(64 * kQ4Waves) void down_q4_kernel(ExpertMap m, const int32_t* ids, uint32_t top_k, const u16* h,
                                                                uint32_t d, uint32_t f, const u16* residual, u16* y) {
  extern __shared__ f32x4 memory[];
  __shared__ float part[kQ4Waves * 16];
  __shared__ LiveExperts live;
  const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
  find_live(m, ids, top_k, 2, live);
  const uint32_t c0 = blockIdx.x * 16, per = (f + 1023) / 1024;
  const uint64_t row = uint64_t(f / kQ4Block) * kQ4Bytes;
  float acc[1] = {};
  stream_q4<T, 1>(live.n * per, wave, waves, d - c0 < 16 ? d - c0 : 16, f, lds_offset(memory) + wave * 2 * Q4Stage<1>::kBytes,
                  [&](uint32_t s, const char* (&base)[1], const u16*& xs) {
                    const uint32_t j = s / per;
                    base[0] = live.part[j] + c0 * row;
                    xs = h + uint64_t(live.from[j]) * f;
                    return (s - j * per) * 1024;
                  }, acc);
  join_q4<1>(part, acc, wave, waves, [&](const float (&s)[1]) {
    if (c0 + lane < d) y[c0 + lane] = T::down(s[0] + (residual ? T::up(residual[c0 + lane]) : 0.0f));
  });
}

// A tile of at most 16 CT pairs of one expert, 16 columns of gate and up a workgroup.
template <class T, class W, int CT, bool kTail>
__global__ __launch_bounds__(64 * most_waves(CT)) void gate_up_few_kernel(Plan p, const u16* x, uint64_t x_stride, uint32_t d,
                                                                          uint32_t f, uint32_t act, u16* h) {
  extern __shared__ f32x4 part[];
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  TileRows t;
  if (!tile_rows(p, blockIdx.y, 16 * CT, t)) return;
  const char *gate = p.part[3 * t.e], *up = p.part[3 * t.e + 1];
  const uint32_t c0 = blockIdx.x * 16 + (lane & 15u), col = c0 < f ? c0 : f - 1;
  const u16* rows[CT];
#pragma unroll
  for (int i = 0; i < CT; ++i) {
    const uint32_t r = 16 * i + (lane & 15u);
    rows[i] = r < t.rows ? x + t.map[r] * x_stride : nullptr;
  }
  f32x4 acc[2][CT] = {};
  stream_chunks<W, 2, CT, kTail>((d + kChunk - 1) / kChunk, wave, waves, [&](uint32_t c, W (&w)[2], const u16* (&row)[CT]) {
    w[0] = W(gate, d, col, d);
    w[1] = W(up, d, col, d);
#pragma unroll
    for (int i = 0; i < CT; ++i) row[i] = rows[i];
    return c * kChunk;
  }, acc);
  f32x4 v[2 * CT];
#pragma unroll
  for (int i = 0; i < 2 * CT; ++i) v[i] = acc[i / CT][i % CT];
  join_waves<2 * CT>(part, v, wave, waves, [&](auto&& sum) {
    for (uint32_t i = wave; i < CT; i += waves) {
      const f32x4 g = sum(i), u = sum(CT + i);
#pragma unroll
      for (uint32_t q = 0; q < 4; ++q) {
        const uint32_t r = 16 * i + (lane >> 4) * 4 + q;
        if (r < t.rows && c0 < f) h[uint64_t(t.first + r) * f + c0] = T::down(activate(act, g[q]) * u[q]);
      }
    }
  });
}

template <class T, class W, int CT, bool kTail>
__global__ __launch_bounds__(64 * most_waves(CT)) void down_few_kernel(Plan p, const u16* h, uint32_t d, uint32_t f, float* out) {
  extern __shared__ f32x4 part[];
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  TileRows t;
  if (!tile_rows(p, blockIdx.y, 16 * CT, t)) return;
  const char* down = p.part[3 * t.e + 2];
  const uint32_t c0 = blockIdx.x * 32 + (lane & 15u);
  f32x4 acc[2][CT] = {};
  stream_chunks<W, 2, CT, kTail>((f + kChunk - 1) / kChunk, wave, waves, [&](uint32_t c, W (&w)[2], const u16* (&row)[CT]) {
    w[0] = W(down, f, c0 < d ? c0 : d - 1, f);
    w[1] = W(down, f, c0 + 16 < d ? c0 + 16 : d - 1, f);
#pragma unroll
    for (uint32_t i = 0; i < CT; ++i) {
      const uint32_t r = 16 * i + (lane & 15u);
      row[i] = r < t.rows ? h + uint64_t(t.first + r) * f : nullptr;
    }
    return c * kChunk;
  }, acc);
  f32x4 v[2 * CT];
#pragma unroll
  for (int i = 0; i < 2 * CT; ++i) v[i] = acc[i / CT][i % CT];
  join_waves<2 * CT>(part, v, wave, waves, [&](auto&& sum) {
    for (uint32_t i = wave; i < 2 * CT; i += waves) {
      const f32x4 s = sum(i);
      const uint32_t c = c0 + 16 * (i / CT);
#pragma unroll
      for (uint32_t q = 0; q < 4; ++q) {
        const uint32_t r = 16 * (i % CT) + (lane >> 4) * 4 + q;
        if (r < t.rows && c < d) out[uint64_t(t.first + r) * d + c] = s[q];
      }
    }
  });
}

// ---- many rows: tiles of 128 pairs of an expert ----------------------------------------------------------------------
constexpr uint32_t kTileRows = 128;

// The plan's tile and the a-tile of a workgroup, over the tiles there are (known on the device only).
__device__ __forceinline__ bool tile_of(const Plan& p, uint32_t na, TileRows& t, uint32_t& a) {
  if (blockIdx.x >= na * *p.n_tiles) return false;
  const TileAt at = tile_at(blockIdx.x, na, *p.n_tiles);
  a = at.a;
  return tile_rows(p, at.b, kTileRows, t);
}

// 4 values next to each other a lane, to rows of 16 bits or 32.
template <class V>
struct RowsOut {
  struct Fetched {};
  V* out;
  uint64_t stride;
  uint32_t rows, c0, n_cols, c = 0;
  __device__ __forceinline__ void columns(uint32_t a) { c = c0 + a; }
  __device__ __forceinline__ Fetched fetch(uint32_t) const { return {}; }
  template <class T>
  __device__ __forceinline__ void put(uint32_t r, f32x4 v) const {
    if (r >= rows || c >= n_cols) return;  // (columns are a multiple of 8: all four or none)
    if constexpr (sizeof(V) == 4) {
      *reinterpret_cast<f32x4*>(out + r * stride + c) = v;
    } else {
      bits4 o;
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] = T::down(v[i]);
      *reinterpret_cast<bits4*>(out + r * stride + c) = o;
    }
  }
};
template <class T, class V>
struct TypedOut : RowsOut<V> {
  __device__ __forceinline__ void finish(uint32_t r, f32x4 v, const typename RowsOut<V>::Fetched&) const {
    this->template put<T>(r, v);
  }
};

// Gate and up rows of the same 128 columns as one operand of 256: each wave gets 64 of both.
template <class T>
__device__ __forceinline__ TileRowsSource<8> gate_up_source(const Plan& p, const TileRows& t, uint32_t d, uint32_t f,
                                                            uint32_t f0) {
  const u16 *gate = reinterpret_cast<const u16*>(p.part[3 * t.e]), *up = reinterpret_cast<const u16*>(p.part[3 * t.e + 1]);
  return TileRowsSource<8>(d, threadIdx.x >> 6 & 1u, [&](uint32_t r) {
    const uint32_t c = f0 + (r >> 7) * 64 + (r & 63u);
    return (r & 64u ? up : gate) + uint64_t(c < f ? c : f - 1) * d;
  });
}
__device__ __forceinline__ TileRowsSource<4> mapped_rows(const TileRows& t, const u16* x, uint64_t stride, uint32_t n) {
  return TileRowsSource<4>(n, threadIdx.x >> 7, [&](uint32_t r) { return x + t.map[r < t.rows ? r : t.rows - 1] * stride; });
}
__device__ __forceinline__ TileRowsSource<4> sorted_rows(const TileRows& t, const u16* x, uint64_t stride, uint32_t n) {
  return TileRowsSource<4>(n, threadIdx.x >> 7,
                           [&](uint32_t r) { return x + uint64_t(t.first + (r < t.rows ? r : t.rows - 1)) * stride; });
}

template <class T>
__global__ __launch_bounds__(kTileThreads, 2) void gate_up_tile_kernel(Plan p, const u16* x, uint64_t x_stride, uint32_t d,
                                                                       uint32_t f, uint32_t act, u16* h) {
  extern __shared__ __attribute__((aligned(1024))) f32x4 memory[];
  TileRows t;
  uint32_t at;
  if (!tile_of(p, (f + 127) / 128, t, at)) return;
  auto w = gate_up_source<T>(p, t, d, f, at * 128);
  auto xs = mapped_rows(t, x, x_stride, d);
  f32x4 acc[8][4] = {};
  tile_product<T, 8, 4, 3>(w, xs, d, lds_offset(memory), acc);
  f32x4 v[4][4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) v[i][j][q] = activate(act, acc[i][j][q]) * acc[i + 4][j][q];
  TypedOut<T, u16> out{{h + uint64_t(t.first) * f, f, t.rows, at * 128, f}};
  hand_out<4, 4, 4>(memory, v, out);
}

template <class T>
__global__ __launch_bounds__(kTileThreads, 2) void down_tile_kernel(Plan p, const u16* h, uint32_t d, uint32_t f, float* out) {
  extern __shared__ __attribute__((aligned(1024))) f32x4 memory[];
  TileRows t;
  uint32_t at;
  if (!tile_of(p, (d + 255) / 256, t, at)) return;
  const u16* down = reinterpret_cast<const u16*>(p.part[3 * t.e + 2]);
  TileRowsSource<8> w(f, threadIdx.x >> 6 & 1u, [&](uint32_t r) {
    const uint32_t c = at * 256 + r;
    return down + uint64_t(c < d ? c : d - 1) * f;
  });
  auto hs = sorted_rows(t, h, f, f);
  f32x4 acc[8][4] = {};
  tile_product<T, 8, 4, 3>(w, hs, f, lds_offset(memory), acc);
  TypedOut<T, float> o{{out + uint64_t(t.first) * d, d, t.rows, at * 256, d}};
  hand_out<8, 4, 2>(memory, acc, o);
}

// The two with 4-bit weights: 64 columns of gate and up, 128 of down a tile.
template <class T>
__global__ __launch_bounds__(kTileThreads, 2) void gate_up_q4_tile_kernel(Plan p, const u16* x, uint64_t x_stride, uint32_t d,
                                                                          uint32_t f, uint32_t act, u16* h) {
  extern __shared__ __attribute__((aligned(1024))) f32x4 memory[];
  TileRows t;
  uint32_t at;
  if (!tile_of(p, (f + 63) / 64, t, at)) return;
  const char *gate = p.part[3 * t.e], *up = p.part[3 * t.e + 1];
  TileQ4Source<T> w(d, threadIdx.x >> 6 & 1u, [&](uint32_t r) {  // of each wave's 64 rows: 32 gate, 32 up
    const uint32_t c = at * 64 + (r >> 6) * 32 + (r & 31u);
    return reinterpret_cast<const unsigned char*>(r & 32u ? up : gate) + uint64_t(c < f ? c : f - 1) * (d / kQ4Block * kQ4Bytes);
  });
  auto xs = mapped_rows(t, x, x_stride, d);
  f32x4 acc[8][4] = {};
  tile_product<T, 8, 4, 3>(w, xs, d, lds_offset(memory), acc);
  f32x4 v[2][4];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const f32x4 g = TileQ4Source<T>::whole(acc[i][j], acc[i + 4][j]), u = TileQ4Source<T>::whole(acc[i + 2][j], acc[i + 6][j]);
#pragma unroll
      for (int q = 0; q < 4; ++q) v[i][j][q] = activate(act, g[q]) * u[q];
    }
  TypedOut<T, u16> out{{h + uint64_t(t.first) * f, f, t.rows, at * 64, f}};
  hand_out<2, 4, 4>(memory, v, out);
}

template <class T>
__global__ __launch_bounds__(kTileThreads, 2) void down_q4_tile_kernel(Plan p, const u16* h, uint32_t d, uint32_t f, float* out) {
  extern __shared__ __attribute__((aligned(1024))) f32x4 memory[];
  TileRows t;
  uint32_t at;
  if (!tile_of(p, (d + 127) / 128, t, at)) return;
  const unsigned char* down = reinterpret_cast<const unsigned char*>(p.part[3 * t.e + 2]);
  TileQ4Source<T> w(f, threadIdx.x >> 6 & 1u, [&](uint32_t r) {
    const uint32_t c = at * 128 + r;
    return down + uint64_t(c < d ? c : d - 1) * (f / kQ4Block * kQ4Bytes);
  });
  auto hs = sorted_rows(t, h, f, f);
  f32x4 acc[8][4] = {};
  tile_product<T, 8, 4, 3>(w, hs, f, lds_offset(memory), acc);
  f32x4 v[4][4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) v[i][j] = TileQ4Source<T>::whole(acc[i][j], acc[i + 4][j]);
  TypedOut<T, float> o{{out + uint64_t(t.first) * d, d, t.rows, at * 128, d}};
  hand_out<4, 4, 4>(memory, v, o);
}

// back = down^T dy of every pair, 256 columns of d_ff: in 32 bits, for the kernel behind it. (One kernel for all three
// products needs 192 accumulators a lane, so one workgroup a CU: 496 us in a training step of 128 experts.)
template <class T>
__global__ __launch_bounds__(kTileThreads, 2) void back_tile_kernel(Plan p, const u16* dy, uint64_t dy_stride, uint32_t d,
                                                                    uint32_t f, float* back) {
  extern __shared__ __attribute__((aligned(1024))) f32x4 memory[];
  TileRows t;
  uint32_t at;
  if (!tile_of(p, (f + 255) / 256, t, at)) return;
  TileColumnsSource<8, false> w(d, threadIdx.x >> 6 & 1u, reinterpret_cast<const u16*>(p.part[3 * t.e + 2]), f, at * 256, f);
  auto dys = mapped_rows(t, dy, dy_stride, d);
  f32x4 acc[8][4] = {};
  tile_product<T, 8, 4, 3>(w, dys, d, lds_offset(memory), acc);
  TypedOut<T, float> o{{back + uint64_t(t.first) * f, f, t.rows, at * 256, f}};
  hand_out<8, 4, 2>(memory, acc, o);
}

// As hidden_grad_any_kernel from gate's and up's products and `back`, 128 columns of d_ff.
template <class T>
__global__ __launch_bounds__(kTileThreads, 2) void hidden_grad_tile_kernel(Plan p, const u16* x, uint64_t x_stride,
                                                                           const float* back, const float* weights, uint32_t d,
                                                                           uint32_t f, uint32_t act, u16* dgu, u16* wh,
                                                                           float* d_share) {
  extern __shared__ __attribute__((aligned(1024))) f32x4 memory[];
  __shared__ float share[kTileRows][2];
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
  TileRows t;
  uint32_t at;
  if (!tile_of(p, (f + 127) / 128, t, at)) return;
  const uint32_t f0 = at * 128;
  f32x4 gu[8][4] = {};
  auto ws = gate_up_source<T>(p, t, d, f, f0);
  auto xs = mapped_rows(t, x, x_stride, d);
  tile_product<T, 8, 4, 3>(ws, xs, d, lds_offset(memory), gu);
  f32x4 h[4][4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t r = (wave >> 1) * 64 + 16 * j + (lane & 15u), pos = t.first + (r < t.rows ? r : t.rows - 1);
    const float w = weights ? weights[p.pair[pos]] : 1.0f;
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t c = f0 + (wave & 1u) * 64 + 16 * i + (lane >> 4) * 4;
      const f32x4 b = c < f ? *reinterpret_cast<const f32x4*>(back + uint64_t(pos) * f + c) : f32x4{0, 0, 0, 0};
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float g = gu[i][j][q], u = gu[i + 4][j][q], a = activate(act, g);
        sum += a * u * b[q];
        h[i][j][q] = w * a * u;
        gu[i][j][q] = w * b[q] * u * slope(act, g);  // dg, du in the products' places
        gu[i + 4][j][q] = w * b[q] * a;
      }
    }
    sum += __shfl_xor(sum, 16, 64);
    sum += __shfl_xor(sum, 32, 64);
    if (lane < 16) share[(wave >> 1) * 64 + 16 * j + lane][wave & 1u] = sum;
  }
  TypedOut<T, u16> out{{wh + uint64_t(t.first) * f, f, t.rows, f0, f}};
  hand_out<4, 4, 4>(memory, h, out);  // (behind its barrier `share` is whole)
  if (threadIdx.x < t.rows) d_share[uint64_t(at) * p.pairs + t.first + threadIdx.x] = share[threadIdx.x][0] + share[threadIdx.x][1];
#pragma unroll
  for (int half = 0; half < 2; ++half) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) h[i][j] = gu[i + 4 * half][j];
    out.out = dgu + uint64_t(t.first) * 2 * f + half * f;
    out.stride = uint64_t(2) * f;
    hand_out<4, 4, 4>(memory, h, out);
  }
}

template <class T>
__global__ __launch_bounds__(kTileThreads, 2) void input_grad_tile_kernel(Plan p, const u16* dgu, uint32_t d, uint32_t f,
                                                                          float* out) {
  extern __shared__ __attribute__((aligned(1024))) f32x4 memory[];
  TileRows t;
  uint32_t at;
  if (!tile_of(p, (d + 255) / 256, t, at)) return;
  f32x4 acc[8][4] = {};
  const auto add = [&](uint32_t half) {
    TileColumnsSource<8, false> w(f, threadIdx.x >> 6 & 1u, reinterpret_cast<const u16*>(p.part[3 * t.e + half]), d, at * 256, d);
    auto v = sorted_rows(t, dgu + half * f, uint64_t(2) * f, f);
    tile_product<T, 8, 4, 3>(w, v, f, lds_offset(memory), acc);
  };
  add(0);
  add(1);
  TypedOut<T, float> o{{out + uint64_t(t.first) * d, d, t.rows, at * 256, d}};
  hand_out<8, 4, 2>(memory, acc, o);
}

// As weight_grad_any_kernel, out[e][b][a]: 256 columns a of `left` and 128 columns b of `right` a workgroup, the sum over the
// expert's pairs. One of the two is read through the rows' map (kMapLeft: left). Columns from n_right on belong to out2 (the
// gradients of gate and up are one product).
template <class T, bool kMapLeft>
__global__ __launch_bounds__(kTileThreads, 2) void weight_grad_tile_kernel(Plan p, const u16* left, uint64_t left_stride,
                                                                           uint32_t n_left, const u16* right,
                                                                           uint64_t right_stride, uint32_t n_right,
                                                                           uint32_t n_outs, u16* out, u16* out2) {
  extern __shared__ __attribute__((aligned(1024))) f32x4 memory[];
  uint32_t* map = reinterpret_cast<uint32_t*>(memory) + tile_lds(8, 4, 3) / 4;
  const uint32_t wave = threadIdx.x >> 6;
  const uint32_t ta = (n_left + 255) / 256, tb = (n_right + 127) / 128, per = ta * tb * n_outs;
  const uint32_t e = blockIdx.x / per, in = blockIdx.x % per;
  const uint32_t a0 = in % ta * 256, which = in / ta / tb, b0 = in / ta % tb * 128;
  const uint32_t first = p.first[e], pairs = p.first[e + 1] - first;
  right += which * n_right;
  f32x4 acc[8][4] = {};
  const auto fill = [&](uint32_t from) {  // half of the ring
    for (uint32_t i = from + threadIdx.x; i < from + kMapRing / 2 && i < pairs; i += kTileThreads)
      map[i % kMapRing] = p.row[first + i];
  };
  const auto refill = [&](uint32_t k) {
    if (k && k % (kMapRing / 2) == 0 && k + kMapRing / 2 < pairs) fill(k + kMapRing / 2);
  };
  if (pairs) {  // (an expert without pairs gets zeros)
    fill(0);
    fill(kMapRing / 2);
    __syncthreads();
    if constexpr (kMapLeft) {
      TileColumnsSource<8, true> l(pairs, wave & 1u, left, left_stride, a0, n_left, map);
      TileColumnsSource<4, false> r(pairs, wave >> 1, right + uint64_t(first) * right_stride, right_stride, b0, n_right);
      tile_product<T, 8, 4, 3>(l, r, pairs, lds_offset(memory), acc, refill);
    } else {
      TileColumnsSource<8, false> l(pairs, wave & 1u, left + uint64_t(first) * left_stride, left_stride, a0, n_left);
      TileColumnsSource<4, true> r(pairs, wave >> 1, right, right_stride, b0, n_right, map);
      tile_product<T, 8, 4, 3>(l, r, pairs, lds_offset(memory), acc, refill);
    }
  }
  TypedOut<T, u16> o{{(which ? out2 : out) + (uint64_t(e) * n_right + b0) * n_left, n_left, n_right - b0, a0, n_left}};
  hand_out<8, 4, 2>(memory, acc, o);
}

// out_t = residual_t + sum_j w_tj v_{at(t, j)}, in the order of j; kWide columns a thread (a multiple of 4: one access each).
template <class T, int kWide>
__global__ __launch_bounds__(256) void combine_kernel(Plan p, uint32_t rows, uint32_t d, const float* v, const float* weights,
                                                      const u16* residual, uint64_t residual_stride, u16* out,
                                                      uint64_t out_stride) {
  const uint32_t per = d / kWide;
  const uint64_t total = uint64_t(rows) * per;
  for (uint64_t i = uint64_t(blockIdx.x) * 256 + threadIdx.x; i < total; i += uint64_t(gridDim.x) * 256) {
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
        const float* from = v + uint64_t(uint32_t(at[j] < 0 ? 0 : at[j])) * d + c;
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

// Of every pair: dg | du as one row of 2 f values, w h, and this tile's share of d w (d_share[f tile][sorted position]).
template <class T>
__global__ __launch_bounds__(256) void hidden_grad_any_kernel(Plan p, const u16* x, uint64_t x_stride, const u16* dy,
                                                              uint64_t dy_stride, const float* weights, uint32_t d, uint32_t f,
                                                              uint32_t act, u16* dgu, u16* wh, float* d_share) {
  __shared__ TileMemory m;
  __shared__ float share[64][2];
  const uint32_t tf = (f + 63) / 64;
  const uint32_t ft = blockIdx.x % tf, f0 = ft * 64;
  TileRows t;
  if (!tile_rows(p, blockIdx.x / tf, 64, t)) return;
  const Operand xs{x, x_stride, 1, t.rows, d, t.map}, dys{dy, dy_stride, 1, t.rows, d, t.map};
  f32x4 g[2][2] = {}, u[2][2] = {}, b[2][2] = {};
  weight_tile<T, false>(p.part[3 * t.e], f, d, f0, xs, m, g);
  weight_tile<T, false>(p.part[3 * t.e + 1], f, d, f0, xs, m, u);
  const Operand down{reinterpret_cast<const u16*>(p.part[3 * t.e + 2]), 1, f, f, d, nullptr};  // (f, d): its columns as rows
  tile64<T, false>(down, f0, dys, 0, d, m, b);
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const uint32_t r = (wave >> 1) * 32 + 16 * j + (lane & 15u);
    const uint32_t pos = t.first + r;
    const float w = r < t.rows && weights ? weights[p.pair[pos]] : 1.0f;
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const uint32_t c = f0 + (wave & 1u) * 32 + 16 * i + (lane >> 4) * 4 + q;
        const float a = activate(act, g[i][j][q]), back = b[i][j][q];
        if (c >= f || r >= t.rows) continue;
        sum += a * u[i][j][q] * back;
        dgu[uint64_t(pos) * 2 * f + c] = T::down(w * back * u[i][j][q] * slope(act, g[i][j][q]));
        dgu[uint64_t(pos) * 2 * f + f + c] = T::down(w * back * a);
        wh[uint64_t(pos) * f + c] = T::down(w * a * u[i][j][q]);
      }
    sum += __shfl_xor(sum, 16, 64);
    sum += __shfl_xor(sum, 32, 64);
    if (lane < 16) share[r][wave & 1u] = sum;
  }
  __syncthreads();
  if (threadIdx.x < t.rows) d_share[uint64_t(ft) * p.pairs + t.first + threadIdx.x] = share[threadIdx.x][0] + share[threadIdx.x][1];
}

template <class T>
__global__ __launch_bounds__(256) void input_grad_any_kernel(Plan p, const u16* dgu, uint32_t d, uint32_t f, float* out) {
  __shared__ TileMemory m;
  const uint32_t td = (d + 63) / 64;
  const uint32_t d0 = blockIdx.x % td * 64;
  TileRows t;
  if (!tile_rows(p, blockIdx.x / td, 64, t)) return;
  f32x4 acc[2][2] = {};
  for (int half = 0; half < 2; ++half) {
    const Operand w{reinterpret_cast<const u16*>(p.part[3 * t.e + half]), 1, d, d, f, nullptr};
    const Operand v{dgu + uint64_t(t.first) * 2 * f + half * f, uint64_t(2) * f, 1, t.rows, f, nullptr};
    tile64<T, false>(w, d0, v, 0, f, m, acc);
  }
  each64(acc, [&](uint32_t i, uint32_t j, float v) {
    if (d0 + i < d && j < t.rows) out[uint64_t(t.first + j) * d + d0 + i] = v;
  });
}

// out[e][b][a] = sum over expert e's pairs of left[pair][a] right[pair][b] (0 for an expert without pairs): left through
// the rows' map where left_map, right where right_map.
template <class T>
__global__ __launch_bounds__(256) void weight_grad_any_kernel(Plan p, const u16* left, uint64_t left_stride, bool left_map,
                                                              uint32_t n_left, const u16* right, uint64_t right_stride,
                                                              bool right_map, uint32_t n_right, u16* out) {
  __shared__ TileMemory m;
  const uint32_t ta = (n_left + 63) / 64, tb = (n_right + 63) / 64;
  const uint32_t per = ta * tb;
  for (uint64_t tile = blockIdx.x; tile < uint64_t(p.n) * per; tile += gridDim.x) {
    const uint32_t e = uint32_t(tile / per), a0 = uint32_t(tile % per) % ta * 64, b0 = uint32_t(tile % per) / ta * 64;
    const uint32_t first = p.first[e], n = p.first[e + 1] - first;
    // (k runs over the pairs: element (r, k) at k stride + r)
    struct Rows {
      const u16* base;
      uint64_t stride;
      const uint32_t* map;
      uint32_t rows, n;
      __device__ __forceinline__ bits8 load8(uint32_t r, uint32_t k) const {
        bits8 v = {0, 0, 0, 0, 0, 0, 0, 0};
        if (r >= rows) return v;
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i)
          if (k + i < n) v[i] = base[uint64_t(map ? map[k + i] : k + i) * stride + r];
        return v;
      }
    };
    const Rows l{left_map ? left : left + first * left_stride, left_stride, left_map ? p.row + first : nullptr, n_left, n};
    const Rows r{right_map ? right : right + first * right_stride, right_stride, right_map ? p.row + first : nullptr, n_right, n};
    f32x4 acc[2][2] = {};
    tile64<T, false>(l, a0, r, b0, n, m, acc);
    each64(acc, [&](uint32_t i, uint32_t j, float v) {
      if (a0 + i < n_left && b0 + j < n_right) out[(uint64_t(e) * n_right + b0 + j) * n_left + a0 + i] = T::down(v);
    });
    __syncthreads();
  }
}

__global__ __launch_bounds__(256) void weights_grad_kernel(Plan p, uint32_t shares, const float* d_share, float* dweights) {
  for (uint64_t i = uint64_t(blockIdx.x) * 256 + threadIdx.x; i < p.pairs; i += uint64_t(gridDim.x) * 256) {
    const int32_t at = p.at[i];
    float s = 0.0f;
    if (at >= 0)
      for (uint32_t k = 0; k < shares; ++k) s += d_share[uint64_t(k) * p.pairs + uint32_t(at)];
    dweights[i] = s;
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
  p.top_k = top_k;
  p.n = n;
  return p;
}

struct Forward {
  Plan plan;
  u16* h;
  float* out;
};
Forward take_forward(Room& r, uint32_t n, uint32_t d, uint32_t f, uint32_t rows, uint32_t top_k) {
  Forward w;
  w.plan = take_plan(r, n, rows * top_k, top_k, 16);  // (the smallest tiles any path takes)
  w.h = r.take<u16>(uint64_t(rows) * top_k * f);
  w.out = r.take<float>(uint64_t(rows) * top_k * d);
  return w;
}
struct Backward {
  Plan plan;
  u16 *dgu, *wh;
  float *share, *out, *back;  // (back and out share their place: out is written behind back's last reader)
};
Backward take_backward(Room& r, uint32_t n, uint32_t d, uint32_t f, uint32_t rows, uint32_t top_k) {
  const uint64_t pairs = uint64_t(rows) * top_k;
  Backward w;
  w.plan = take_plan(r, n, uint32_t(pairs), top_k, 64);
  w.dgu = r.take<u16>(pairs * 2 * f);
  w.wh = r.take<u16>(pairs * f);
  w.share = r.take<float>(pairs * ((f + 63) / 64));
  w.out = w.back = r.take<float>(pairs * (d > f ? d : f));
  return w;
}

uint32_t blocks(uint64_t n) { return uint32_t(n < (1u << 20) ? n : (1u << 20)); }

int launch_plan(const ExpertMap& e, const int32_t* ids, const Plan& p, uint32_t rows_per_tile, hipStream_t s) {
  hipLaunchKernelGGL(plan_kernel, dim3(1), dim3(kPlanThreads), 4 * (kPlanThreads + kPlanWaves * e.n), s, e, ids, p,
                     rows_per_tile);
  return int(hipGetLastError());
}

template <class T>
int launch_combine(const Plan& p, uint32_t rows, uint32_t d, const float* v, const float* weights, const void* residual,
                   uint64_t residual_stride, void* out, uint64_t out_stride, hipStream_t s) {
  const u16* r = static_cast<const u16*>(residual);
  u16* o = static_cast<u16*>(out);
  const uint64_t odd = reinterpret_cast<uintptr_t>(residual) | 2 * residual_stride | reinterpret_cast<uintptr_t>(out) | 2 * out_stride;
  if (d % 4 == 0 && odd % 8 == 0)
    hipLaunchKernelGGL((combine_kernel<T, 4>), dim3(blocks((uint64_t(rows) * d / 4 + 255) / 256)), dim3(256), 0, s, p, rows, d, v,
                       weights, r, residual_stride, o, out_stride);
  else
    hipLaunchKernelGGL((combine_kernel<T, 1>), dim3(blocks((uint64_t(rows) * d + 255) / 256)), dim3(256), 0, s, p, rows, d, v,
                       weights, r, residual_stride, o, out_stride);
  return int(hipGetLastError());
}

bool aligned16(const void* p, uint64_t stride_bytes) { return (reinterpret_cast<uintptr_t>(p) | stride_bytes) % 16 == 0; }

// Whether every weight row, x row and row of h starts 16-byte aligned and holds whole groups of 8 values. The addresses of
// a table's units are the device's: its units are 256-byte aligned, as the library lays them out.
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

template <class T, class W, bool kTail>
int forward_one(const ExpertMap& e, uint32_t d, uint32_t f, const tsa_ffn_args& a, void* ws, hipStream_t s) {
  u16* h = static_cast<u16*>(ws);
  const uint32_t tf = (f + 15) / 16, td = (d + 15) / 16;
  const uint32_t w1 = stream_waves(uint64_t(tf) * a.top_k, chunks_of(d), 16);
  hipLaunchKernelGGL((gate_up_one_kernel<T, W, kTail>), dim3(tf, a.top_k), dim3(64 * w1), w1 * 2048, s, e, a.ids, a.weights,
                     static_cast<const u16*>(a.x), d, f, a.act, h);
  const uint32_t w2 = stream_waves(td, uint64_t(chunks_of(f)) * a.top_k, 16);
  hipLaunchKernelGGL((down_one_kernel<T, W, kTail>), dim3(td), dim3(64 * w2), w2 * 1024, s, e, a.ids, a.top_k, h, d, f,
                     static_cast<const u16*>(a.residual), static_cast<u16*>(a.y));
  return int(hipGetLastError());
}

template <class T>
int forward_one_q4(const ExpertMap& e, uint32_t d, uint32_t f, const tsa_ffn_args& a, void* ws, hipStream_t s) {
  u16* h = static_cast<u16*>(ws);
  const uint32_t tf = (f + 15) / 16, td = (d + 15) / 16;
  const uint32_t w1 = q4_waves(uint64_t(tf) * a.top_k, (d + 511) / 512);
  hipLaunchKernelGGL((gate_up_q4_kernel<T>), dim3(tf, a.top_k), dim3(64 * w1), w1 * 2 * Q4Stage<2>::kBytes, s, e, a.ids, a.weights,
                     static_cast<const u16*>(a.x), d, f, a.act, h);
  const uint32_t w2 = q4_waves(td, uint64_t((f + 1023) / 1024) * a.top_k);
  hipLaunchKernelGGL((down_q4_kernel<T>), dim3(td), dim3(64 * w2), w2 * 2 * Q4Stage<1>::kBytes, s, e, a.ids, a.top_k, h, d, f,
                     static_cast<const u16*>(a.residual), static_cast<u16*>(a.y));
  return int(hipGetLastError());
}

template <class T, class W, int CT, bool kTail>
int forward_few(const ExpertMap& e, uint32_t d, uint32_t f, const tsa_ffn_args& a, const Forward& w, hipStream_t s) {
  if (int err = launch_plan(e, a.ids, w.plan, 16 * CT, s)) return err;
  const uint32_t tiles = most_tiles(w.plan.pairs, e.n, 16 * CT), tf = (f + 15) / 16, td = (d + 31) / 32;
  const uint32_t w1 = stream_waves(uint64_t(tf) * tiles, chunks_of(d), most_waves(CT));
  hipLaunchKernelGGL((gate_up_few_kernel<T, W, CT, kTail>), dim3(tf, tiles), dim3(64 * w1), w1 * CT * 2048, s, w.plan,
                     static_cast<const u16*>(a.x), a.x_stride, d, f, a.act, w.h);
  const uint32_t w2 = stream_waves(uint64_t(td) * tiles, chunks_of(f), most_waves(CT));
  hipLaunchKernelGGL((down_few_kernel<T, W, CT, kTail>), dim3(td, tiles), dim3(64 * w2), w2 * CT * 2048, s, w.plan, w.h, d, f,
                     w.out);
  return launch_combine<T>(w.plan, a.rows, d, w.out, a.weights, a.residual, a.residual_stride, a.y, a.y_stride, s);
}

template <class T, class W, bool kTail>
int forward_stream(const ExpertMap& e, uint32_t d, uint32_t f, const tsa_ffn_args& a, void* ws, hipStream_t s) {
  if (a.rows == 1) return forward_one<T, W, kTail>(e, d, f, a, ws, s);
  Room room(ws);
  const Forward w = take_forward(room, e.n, d, f, a.rows, a.top_k);
  const uint32_t each = w.plan.pairs / e.n;  // pairs of an expert if all are asked for alike
  if (each <= 8) return forward_few<T, W, 1, kTail>(e, d, f, a, w, s);
  if (each <= 24) return forward_few<T, W, 2, kTail>(e, d, f, a, w, s);
  return forward_few<T, W, 4, kTail>(e, d, f, a, w, s);
}

template <class T, bool kQ4>
int forward_tiles(const ExpertMap& e, uint32_t d, uint32_t f, const tsa_ffn_args& a, void* ws, hipStream_t s) {
  Room room(ws);
  const Forward w = take_forward(room, e.n, d, f, a.rows, a.top_k);
  if (int err = launch_plan(e, a.ids, w.plan, kTileRows, s)) return err;
  const uint32_t tiles = most_tiles(w.plan.pairs, e.n, kTileRows);
  constexpr uint32_t kF = kQ4 ? 64 : 128, kD = kQ4 ? 128 : 256;  // columns a tile
  const dim3 up(tiles * ((f + kF - 1) / kF)), down(tiles * ((d + kD - 1) / kD));
  const u16* x = static_cast<const u16*>(a.x);
  if constexpr (kQ4) {
    hipLaunchKernelGGL((gate_up_q4_tile_kernel<T>), up, dim3(kTileThreads), tile_lds(8, 4, 3), s, w.plan, x, a.x_stride, d, f, a.act, w.h);
    hipLaunchKernelGGL((down_q4_tile_kernel<T>), down, dim3(kTileThreads), tile_lds(8, 4, 3), s, w.plan, w.h, d, f, w.out);
  } else {
    hipLaunchKernelGGL((gate_up_tile_kernel<T>), up, dim3(kTileThreads), tile_lds(8, 4, 3), s, w.plan, x, a.x_stride, d, f, a.act, w.h);
    hipLaunchKernelGGL((down_tile_kernel<T>), down, dim3(kTileThreads), tile_lds(8, 4, 3), s, w.plan, w.h, d, f, w.out);
  }
  return launch_combine<T>(w.plan, a.rows, d, w.out, a.weights, a.residual, a.residual_stride, a.y, a.y_stride, s);
}

template <class T, bool kQ4>
int forward(const ExpertMap& e, uint32_t d, uint32_t f, const tsa_ffn_args& a, void* ws, hipStream_t s) {
  typedef std::conditional_t<kQ4, RowsQ4<T>, Rows16<T>> W;
  if constexpr (kQ4)
    if (a.rows == 1 && d % 256 == 0 && f % 256 == 0 && aligned16(a.x, 0) && wide_weights(e)) return forward_one_q4<T>(e, d, f, a, ws, s);
  if (uint64_t(a.rows) * a.top_k <= uint64_t(64) * e.n)
    return d % kChunk || f % kChunk ? forward_stream<T, W, true>(e, d, f, a, ws, s) : forward_stream<T, W, false>(e, d, f, a, ws, s);
  if (wide_rows(e, d, f, kQ4, a.x, a.x_stride)) return forward_tiles<T, kQ4>(e, d, f, a, ws, s);
  Room room(ws);
  const Forward w = take_forward(room, e.n, d, f, a.rows, a.top_k);
  if (int err = launch_plan(e, a.ids, w.plan, 64, s)) return err;
  const uint32_t tiles = most_tiles(w.plan.pairs, e.n, 64);
  hipLaunchKernelGGL((gate_up_any_kernel<T, kQ4>), dim3(tiles * ((f + 63) / 64)), dim3(256), 0, s, w.plan,
                     static_cast<const u16*>(a.x), a.x_stride, d, f, a.act, w.h);
  hipLaunchKernelGGL((down_any_kernel<T, kQ4>), dim3(tiles * ((d + 63) / 64)), dim3(256), 0, s, w.plan, w.h, d, f, w.out);
  return launch_combine<T>(w.plan, a.rows, d, w.out, a.weights, a.residual, a.residual_stride, a.y, a.y_stride, s);
}

template <class T>
int backward_tiles(const ExpertMap& e, uint32_t d, uint32_t f, const tsa_ffn_grad_args& a, void* ws, hipStream_t s) {
  Room room(ws);
  const Backward w = take_backward(room, e.n, d, f, a.rows, a.top_k);
  if (int err = launch_plan(e, a.ids, w.plan, kTileRows, s)) return err;
  const uint32_t tiles = most_tiles(w.plan.pairs, e.n, kTileRows), tf = (f + 127) / 128, td = (d + 255) / 256;
  const u16 *x = static_cast<const u16*>(a.x), *dy = static_cast<const u16*>(a.dy);
  if (tiles) {
    hipLaunchKernelGGL((back_tile_kernel<T>), dim3(tiles * ((f + 255) / 256)), dim3(kTileThreads), tile_lds(8, 4, 3), s, w.plan, dy,
                       a.dy_stride, d, f, w.back);
    hipLaunchKernelGGL((hidden_grad_tile_kernel<T>), dim3(tiles * tf), dim3(kTileThreads), tile_lds(8, 4, 3), s, w.plan, x,
                       a.x_stride, w.back, a.weights, d, f, a.act, w.dgu, w.wh, w.share);
  }
  if (a.dx && tiles) {
    hipLaunchKernelGGL((input_grad_tile_kernel<T>), dim3(tiles * td), dim3(kTileThreads), tile_lds(8, 4, 3), s, w.plan, w.dgu, d, f,
                       w.out);
    if (int err = launch_combine<T>(w.plan, a.rows, d, w.out, nullptr, nullptr, 0, a.dx, a.dx_stride, s)) return err;
  }
  if (a.dweights && tiles)
    hipLaunchKernelGGL(weights_grad_kernel, dim3(blocks((w.plan.pairs + 255) / 256)), dim3(256), 0, s, w.plan, tf, w.share,
                       a.dweights);
  if (a.dgate) {
    constexpr uint32_t kLds = tile_lds(8, 4, 3) + 4 * kMapRing;
    hipLaunchKernelGGL((weight_grad_tile_kernel<T, true>), dim3(e.n * td * tf * 2), dim3(kTileThreads), kLds, s, w.plan, x,
                       a.x_stride, d, w.dgu, uint64_t(2) * f, f, 2u, static_cast<u16*>(a.dgate), static_cast<u16*>(a.dup));
    hipLaunchKernelGGL((weight_grad_tile_kernel<T, false>), dim3(e.n * ((f + 255) / 256) * ((d + 127) / 128)), dim3(kTileThreads),
                       kLds, s, w.plan, w.wh, uint64_t(f), f, dy, a.dy_stride, d, 1u, static_cast<u16*>(a.ddown),
                       static_cast<u16*>(nullptr));
  }
  return int(hipGetLastError());
}

template <class T>
int backward(const ExpertMap& e, uint32_t d, uint32_t f, const tsa_ffn_grad_args& a, void* ws, hipStream_t s) {
  if (wide_rows(e, d, f, false, a.x, a.x_stride) && aligned16(a.dy, 2 * a.dy_stride) && a.dy_stride < 1u << 24 && aligned16(a.dgate, 0) && aligned16(a.dup, 0) &&
      aligned16(a.ddown, 0))
    return backward_tiles<T>(e, d, f, a, ws, s);
  Room room(ws);
  const Backward w = take_backward(room, e.n, d, f, a.rows, a.top_k);
  if (int err = launch_plan(e, a.ids, w.plan, 64, s)) return err;
  const uint32_t tiles = most_tiles(w.plan.pairs, e.n, 64), tf = (f + 63) / 64, td = (d + 63) / 64;
  const u16 *x = static_cast<const u16*>(a.x), *dy = static_cast<const u16*>(a.dy);
  if (tiles)
    hipLaunchKernelGGL((hidden_grad_any_kernel<T>), dim3(tiles * tf), dim3(256), 0, s, w.plan, x, a.x_stride, dy, a.dy_stride,
                       a.weights, d, f, a.act, w.dgu, w.wh, w.share);
  if (a.dx && tiles) {
    hipLaunchKernelGGL((input_grad_any_kernel<T>), dim3(tiles * td), dim3(256), 0, s, w.plan, w.dgu, d, f, w.out);
    if (int err = launch_combine<T>(w.plan, a.rows, d, w.out, nullptr, nullptr, 0, a.dx, a.dx_stride, s)) return err;
  }
  if (a.dweights && tiles)
    hipLaunchKernelGGL(weights_grad_kernel, dim3(blocks((w.plan.pairs + 255) / 256)), dim3(256), 0, s, w.plan, tf, w.share,
                       a.dweights);
  if (a.dgate) {
    const uint32_t g = blocks(uint64_t(e.n) * tf * td);
    for (int half = 0; half < 2; ++half)
      hipLaunchKernelGGL((weight_grad_any_kernel<T>), dim3(g), dim3(256), 0, s, w.plan, x, a.x_stride, true, d,
                         w.dgu + half * uint64_t(f), uint64_t(2) * f, false, f, static_cast<u16*>(half ? a.dup : a.dgate));
    hipLaunchKernelGGL((weight_grad_any_kernel<T>), dim3(g), dim3(256), 0, s, w.plan, w.wh, uint64_t(f), false, f, dy,
                       a.dy_stride, true, d, static_cast<u16*>(a.ddown));
  }
  return int(hipGetLastError());
}

}  // namespace
}  // namespace op

uint64_t ffn_workspace(uint32_t n, uint32_t d, uint32_t f, uint32_t, uint32_t rows, uint32_t top_k) {
  op::Room room(nullptr);
  op::take_forward(room, n, d, f, rows, top_k);
  return room.bytes;
}
int launch_ffn(const ExpertMap& e, uint32_t d, uint32_t f, uint32_t w_type, const tsa_ffn_args& a, void* ws,
               hipStream_t stream) {
  if (a.rows == 0) return 0;
  const bool q4 = w_type == TSA_Q4;
  if (a.type == TSA_BF16)
    return q4 ? op::forward<op::Bf16, true>(e, d, f, a, ws, stream) : op::forward<op::Bf16, false>(e, d, f, a, ws, stream);
  return q4 ? op::forward<op::F16, true>(e, d, f, a, ws, stream) : op::forward<op::F16, false>(e, d, f, a, ws, stream);
}

uint64_t ffn_backward_workspace(uint32_t n, uint32_t d, uint32_t f, uint32_t rows, uint32_t top_k) {
  op::Room room(nullptr);
  op::take_backward(room, n, d, f, rows, top_k);
  return room.bytes;
}
int launch_ffn_backward(const ExpertMap& e, uint32_t d, uint32_t f, const tsa_ffn_grad_args& a, void* ws, hipStream_t stream) {
  return a.type == TSA_BF16 ? op::backward<op::Bf16>(e, d, f, a, ws, stream) : op::backward<op::F16>(e, d, f, a, ws, stream);
}

}  // namespace tsa
