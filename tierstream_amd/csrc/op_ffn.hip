// Gated feed-forward blocks of the chosen experts.
//
// The pairs (row, j) are grouped by expert first; then h = act(gate x) * (up x) of every pair, y' = down h, and
// y_t = residual_t + sum_j w_tj y'_tj. h is rounded once to the operands' 16 bits, as the matrix instructions take them (half
// precision: as what a power of two leaves of it, so that no finite h overflows or loses bits); y' stays in 32 bits until the
// row's sum. One row (a decode step of one token) needs no grouping: its h carries w, and one product over all its experts gives
// y. No sum depends on an order that changes.
#include "op_pairs.hpp"
#include "op_stream.hpp"

namespace tsa {
namespace op {
namespace {

// Rows of n values to half precision: each row times the power of two that its largest value asks for, whose inverse goes to scale.
// `parts` workgroups a row: each finds the largest value of the whole row and rounds its share. Bound by the bytes: 8002 rows of
// 14336 (688 MB) 161 us, 4.3 TB/s; the 28672 values of one row 5 us, a launch.
template <int kWide>
__global__ __launch_bounds__(1024) void fit_kernel(const float* from, u16* to, float* scale, uint32_t n, const uint32_t* n_rows,
                                                   uint32_t parts) {
  __shared__ float tops[16];
  const uint32_t row = blockIdx.x / parts, part = blockIdx.x % parts, lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
  if (n_rows && row >= *n_rows) return;
  typedef float wide_t __attribute__((ext_vector_type(kWide)));
  typedef u16 bits_t __attribute__((ext_vector_type(kWide)));
  const wide_t* v = reinterpret_cast<const wide_t*>(from + uint64_t(row) * n);
  bits_t* out = reinterpret_cast<bits_t*>(to + uint64_t(row) * n);
  const uint32_t all = n / kWide, share = (all + parts - 1) / parts, begin = part * share, end = begin + share < all ? begin + share : all;
  float top = 0.0f;
#pragma unroll 4
  for (uint32_t i = threadIdx.x; i < all; i += blockDim.x) {
    const wide_t x = v[i];
#pragma unroll
    for (int q = 0; q < kWide; ++q) top = peak(top, x[q]);
  }
  for (int s = 1; s < 64; s <<= 1) top = fmaxf(top, __shfl_xor(top, s, 64));
  if (lane == 0) tops[wave] = top;
  __syncthreads();
  for (uint32_t w = 0; w < blockDim.x / 64; ++w) top = fmaxf(top, tops[w]);
  const Fit fit(top);
  if (part == 0 && threadIdx.x == 0) scale[row] = fit.up;
#pragma unroll 4
  for (uint32_t i = begin + threadIdx.x; i < end; i += blockDim.x) {
    const wide_t x = v[i];
    bits_t o;
#pragma unroll
    for (int q = 0; q < kWide; ++q) o[q] = F16::down(x[q] * fit.down);
    out[i] = o;
  }
}

template <class T, bool kQ4>
__global__ __launch_bounds__(256) void gate_up_any_kernel(Plan p, const u16* x, uint64_t x_stride, uint32_t d, uint32_t f,
                                                          uint32_t act, held<T>* h) {
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
    if (f0 + i < f && j < t.rows) h[uint64_t(t.first + j) * f + f0 + i] = Held<T>::of(v);
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
// The part pointers of an expert, in every thread that asks; false if there is none.
__device__ __forceinline__ bool resolve(const ExpertMap& m, uint32_t e, const char* (&p)[3]) {
  if (e == ~0u) return false;
  part_pointers(m, e, p);
  return true;
}

// What an expert that adds nothing leaves of a row's h: nothing reads it, except (half precision) the search for the largest.
template <class T>
__device__ __forceinline__ void no_pair(held<T>* h, uint32_t c0, uint32_t f) {
  if (std::is_same_v<T, F16> && threadIdx.x < 16 && c0 + threadIdx.x < f) h[c0 + threadIdx.x] = 0;
}

// One row of x: pair j is blockIdx.y, h_j = w_j act(gate x) (up x) for 16 columns a workgroup.
template <class T, class W, bool kTail, bool kStaged>
__global__ __launch_bounds__(64 * most_waves(1)) void gate_up_one_kernel(ExpertMap m, const int32_t* ids, const float* weights,
                                                                         const u16* x, uint32_t d, uint32_t f, uint32_t act,
                                                                         held<T>* h) {
  extern __shared__ f32x4 part[];
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  const char* p[3];
  if (!resolve(m, expert_of(m, ids, blockIdx.y), p)) {
    no_pair<T>(h + uint64_t(blockIdx.y) * f, blockIdx.x * 16, f);
    return;
  }
  const uint32_t c0 = blockIdx.x * 16 + (lane & 15u), col = c0 < f ? c0 : f - 1;
  f32x4 acc[2][1] = {};
  const auto at = [&](uint32_t c, W (&w)[2]) {
    w[0] = W(p[0], d, col, d);
    w[1] = W(p[1], d, col, d);
    return c * kChunk;
  };
  if constexpr (kStaged) {
    u16* xs = reinterpret_cast<u16*>(part + waves * 128);
    stream_one<T, 2, kTail>((d + kChunk - 1) / kChunk, wave, waves, lds_offset(xs), at, [&] {
      stage_row(xs, x, d);
      __syncthreads();
    }, acc);
  } else {
    stream_chunks<W, 2, 1, kTail>((d + kChunk - 1) / kChunk, wave, waves, [&](uint32_t c, W (&w)[2], const u16* (&row)[1]) {
      row[0] = x;
      return at(c, w);
    }, acc);
  }
  const f32x4 v[2] = {acc[0][0], acc[1][0]};
  join_waves<2>(part, v, wave, waves, [&](auto&& sum) {
    if (wave != 0) return;
    const float g = sum(0)[0], u = sum(1)[0];
    if (lane < 16 && c0 < f) h[uint64_t(blockIdx.y) * f + c0] = Held<T>::of((weights ? weights[blockIdx.y] : 1.0f) * activate(act, g) * u);
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
template <class T, class W, bool kTail, bool kStaged>
__global__ __launch_bounds__(64 * most_waves(1)) void down_one_kernel(ExpertMap m, const int32_t* ids, uint32_t top_k,
                                                                      const u16* h, const float* scale, uint32_t d, uint32_t f,
                                                                      const u16* residual, u16* y) {
  extern __shared__ f32x4 part[];
  __shared__ LiveExperts live;
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  find_live(m, ids, top_k, 2, live);
  const uint32_t c0 = blockIdx.x * 16 + (lane & 15u), col = c0 < d ? c0 : d - 1, per = (f + kChunk - 1) / kChunk;
  f32x4 acc[1][1] = {};
  if constexpr (kStaged) {
    u16* xs = reinterpret_cast<u16*>(part + waves * 64);
    stream_one<T, 1, kTail>(live.n * per, wave, waves, lds_offset(xs), [&](uint32_t c, W (&w)[1]) {
      const uint32_t j = c / per;
      w[0] = W(live.part[j], f, col, f);
      return (c - j * per) * kChunk;
    }, [&] {
      for (uint32_t j = 0; j < live.n; ++j) stage_row(xs + j * per * kChunk, h + uint64_t(live.from[j]) * f, f);
      __syncthreads();
    }, acc);
  } else {
    stream_chunks<W, 1, 1, kTail>(live.n * per, wave, waves, [&](uint32_t c, W (&w)[1], const u16* (&row)[1]) {
      const uint32_t j = c / per;
      w[0] = W(live.part[j], f, col, f);
      row[0] = h + uint64_t(live.from[j]) * f;
      return (c - j * per) * kChunk;
    }, acc);
  }
  const f32x4 v[1] = {acc[0][0]};
  join_waves<1>(part, v, wave, waves, [&](auto&& sum) {
    if (wave != 0) return;
    const float s = sum(0)[0] * (scale ? *scale : 1.0f) + (residual && c0 < d ? T::up(residual[c0]) : 0.0f);
    if (lane < 16 && c0 < d) y[c0] = T::down(s);
  });
}

// The same two with 4-bit weights by way of LDS (d and f multiples of 256, 16-byte aligned weights).
template <class T>
__global__ __launch_bounds__(64 * kQ4Waves) void gate_up_q4_kernel(ExpertMap m, const int32_t* ids, const float* weights,
                                                                   const u16* x, uint32_t d, uint32_t f, uint32_t act, held<T>* h) {
  extern __shared__ f32x4 memory[];
  __shared__ float part[kQ4Waves * 2 * 16];
  const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
  const char* p[3];
  if (!resolve(m, expert_of(m, ids, blockIdx.y), p)) {
    no_pair<T>(h + uint64_t(blockIdx.y) * f, blockIdx.x * 16, f);
    return;
  }
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
      h[uint64_t(blockIdx.y) * f + c0 + lane] = Held<T>::of((weights ? weights[blockIdx.y] : 1.0f) * activate(act, s[0]) * s[1]);
  });
}

template <class T>
__global__ __launch_bounds__(64 * kQ4Waves) void down_q4_kernel(ExpertMap m, const int32_t* ids, uint32_t top_k, const u16* h,
                                                                const float* scale, uint32_t d, uint32_t f, const u16* residual, u16* y) {
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
    if (c0 + lane < d) y[c0 + lane] = T::down(s[0] * (scale ? *scale : 1.0f) + (residual ? T::up(residual[c0 + lane]) : 0.0f));
  });
}

// A tile of at most 16 CT pairs of one expert, 16 columns of gate and up a workgroup.
template <class T, class W, int CT, bool kTail>
__global__ __launch_bounds__(64 * most_waves(CT)) void gate_up_few_kernel(Plan p, const u16* x, uint64_t x_stride, uint32_t d,
                                                                          uint32_t f, uint32_t act, held<T>* h) {
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
        if (r < t.rows && c0 < f) h[uint64_t(t.first + r) * f + c0] = Held<T>::of(activate(act, g[q]) * u[q]);
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

// ---- many rows: tiles ---------------------------------------------------------------------------------------------------
template <class T, class S>
__global__ __launch_bounds__(kTileThreads, 2) void gate_up_tile_kernel(Plan p, const u16* x, uint64_t x_stride, uint32_t d,
                                                                       uint32_t f, uint32_t act, held<T>* h) {
  extern __shared__ __attribute__((aligned(1024))) f32x4 memory[];
  constexpr int NI = S::NI, MJ = S::MJ;
  TileRows t;
  uint32_t at;
  if (!tile_of<S>(p, (f + 16 * NI - 1) / (16 * NI), t, at)) return;
  auto w = gate_up_source<NI>(p, t, d, f, at * 16 * NI);
  auto xs = mapped_rows<MJ>(t, x, x_stride, d);
  f32x4 acc[NI][MJ] = {};
  tile_product<T, NI, MJ, S::NB>(w, xs, d, lds_offset(memory), acc);
  f32x4 v[NI / 2][MJ];
#pragma unroll
  for (int i = 0; i < NI / 2; ++i)
#pragma unroll
    for (int j = 0; j < MJ; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) v[i][j][q] = activate(act, acc[i][j][q]) * acc[i + NI / 2][j][q];
  hand_out_held<T, NI / 2, MJ>(memory, v, h + uint64_t(t.first) * f, f, t.rows, at * 16 * NI, f);
}

// (With small tiles, a step of 32 rows through 8 of 128 experts of 2048 x 768: gate and up 84 us, 5.1 TB/s of weights, down 48, 4.5;
// with big ones a prompt of 4001 rows through 2 of 8 experts of 4096 x 14336: 1880 and 1060 us, 1000 and 890 TFLOP/s.)
template <class T, class S>
__global__ __launch_bounds__(kTileThreads, 2) void down_tile_kernel(Plan p, const u16* h, uint32_t d, uint32_t f, float* out) {
  extern __shared__ __attribute__((aligned(1024))) f32x4 memory[];
  constexpr int NI = S::NI, MJ = S::MJ;
  TileRows t;
  uint32_t at;
  if (!tile_of<S>(p, (d + S::kA - 1) / S::kA, t, at)) return;
  const u16* down = reinterpret_cast<const u16*>(p.part[3 * t.e + 2]);
  TileRowsSource<NI> w(f, threadIdx.x >> 6 & 1u, [&](uint32_t r) {
    const uint32_t c = at * S::kA + r;
    return down + uint64_t(c < d ? c : d - 1) * f;
  });
  auto hs = sorted_rows<MJ>(t, h, f, f);
  f32x4 acc[NI][MJ] = {};
  tile_product<T, NI, MJ, S::NB>(w, hs, f, lds_offset(memory), acc);
  FloatRows o{out + uint64_t(t.first) * d, d, t.rows, at * S::kA, d};
  hand_out<NI, MJ>(memory, acc, o);
}

// The two with 4-bit weights: 64 columns of gate and up, 128 of down a tile.
template <class T>
__global__ __launch_bounds__(kTileThreads, 2) void gate_up_q4_tile_kernel(Plan p, const u16* x, uint64_t x_stride, uint32_t d,
                                                                          uint32_t f, uint32_t act, held<T>* h) {
  extern __shared__ __attribute__((aligned(1024))) f32x4 memory[];
  TileRows t;
  uint32_t at;
  if (!tile_of<WideTile>(p, (f + 63) / 64, t, at)) return;
  const char *gate = p.part[3 * t.e], *up = p.part[3 * t.e + 1];
  TileQ4Source<T> w(d, threadIdx.x >> 6 & 1u, [&](uint32_t r) {  // of each wave's 64 rows: 32 gate, 32 up
    const uint32_t c = at * 64 + (r >> 6) * 32 + (r & 31u);
    return reinterpret_cast<const unsigned char*>(r & 32u ? up : gate) + uint64_t(c < f ? c : f - 1) * (d / kQ4Block * kQ4Bytes);
  });
  auto xs = mapped_rows<4>(t, x, x_stride, d);
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
  hand_out_held<T, 2, 4>(memory, v, h + uint64_t(t.first) * f, f, t.rows, at * 64, f);
}

template <class T>
__global__ __launch_bounds__(kTileThreads, 2) void down_q4_tile_kernel(Plan p, const u16* h, uint32_t d, uint32_t f, float* out) {
  extern __shared__ __attribute__((aligned(1024))) f32x4 memory[];
  TileRows t;
  uint32_t at;
  if (!tile_of<WideTile>(p, (d + 127) / 128, t, at)) return;
  const unsigned char* down = reinterpret_cast<const unsigned char*>(p.part[3 * t.e + 2]);
  TileQ4Source<T> w(f, threadIdx.x >> 6 & 1u, [&](uint32_t r) {
    const uint32_t c = at * 128 + r;
    return down + uint64_t(c < d ? c : d - 1) * (f / kQ4Block * kQ4Bytes);
  });
  auto hs = sorted_rows<4>(t, h, f, f);
  f32x4 acc[8][4] = {};
  tile_product<T, 8, 4, 3>(w, hs, f, lds_offset(memory), acc);
  f32x4 v[4][4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) v[i][j] = TileQ4Source<T>::whole(acc[i][j], acc[i + 4][j]);
  FloatRows o{out + uint64_t(t.first) * d, d, t.rows, at * 128, d};
  hand_out<4, 4>(memory, v, o);
}

// ---- launches ----
template <class T, int kWide>
__global__ __launch_bounds__(256) void combine_kernel(Combine c) {
  combine<T, kWide>(c, blockIdx.x);
}

struct Forward {
  Plan plan;
  u16* h;
  float *out, *scale;  // half precision: h is made in out's place, and rounded from there before out is written
};
Forward take_forward(Room& r, uint32_t n, uint32_t d, uint32_t f, uint32_t rows, uint32_t top_k, bool half) {
  const uint64_t pairs = uint64_t(rows) * top_k;
  Forward w;
  w.plan = take_plan(r, n, rows * top_k, top_k, 16);  // (the smallest tiles any path takes)
  w.h = r.take<u16>(pairs * f);
  w.out = r.take<float>(pairs * (half && f > d ? f : d));
  w.scale = r.take<float>(half ? pairs : 0);
  return w;
}
// Where a product leaves h, and the launch that makes operands of it: of the plan's pairs, or of one row's together.
template <class T>
held<T>* made(const Forward& w) {
  if constexpr (std::is_same_v<T, F16>) return w.out;
  else return w.h;
}
template <class T>
void launch_fit(const Forward& w, uint32_t f, bool one_row, hipStream_t s) {
  if constexpr (std::is_same_v<T, F16>) {
    const uint32_t n = one_row ? w.plan.pairs * f : f, parts = one_row ? (n + 8191) / 8192 : 1;
    const dim3 grid(one_row ? parts : w.plan.pairs), block(one_row ? 1024 : 256);
    const uint32_t* rows = one_row ? nullptr : w.plan.first + w.plan.n;
    if (f % 4 == 0) hipLaunchKernelGGL((fit_kernel<4>), grid, block, 0, s, w.out, w.h, w.scale, n, rows, parts);
    else hipLaunchKernelGGL((fit_kernel<1>), grid, block, 0, s, w.out, w.h, w.scale, n, rows, parts);
  }
}

template <class T>
int launch_combine(const Forward& w, uint32_t d, const tsa_ffn_args& a, hipStream_t s) {
  bool wide;
  Combine c = combine_of(w.plan, a.rows, d, w.out, a.weights, a.residual, a.residual_stride, a.y, a.y_stride, wide);
  if (std::is_same_v<T, F16>) c.scale = w.scale;
  if (wide) hipLaunchKernelGGL((combine_kernel<T, 4>), dim3(c.n_blocks), dim3(256), 0, s, c);
  else hipLaunchKernelGGL((combine_kernel<T, 1>), dim3(c.n_blocks), dim3(256), 0, s, c);
  return int(hipGetLastError());
}

template <class T, class W, bool kTail>
int forward_one(const ExpertMap& e, uint32_t d, uint32_t f, const tsa_ffn_args& a, const Forward& w, hipStream_t s) {
  constexpr bool kHalf = std::is_same_v<T, F16>;
  const uint32_t tf = (f + 15) / 16, td = (d + 15) / 16;
  const uint32_t w1 = stream_waves(uint64_t(tf) * a.top_k, chunks_of(d), 16);
  const auto up = [&](auto staged) {
    hipLaunchKernelGGL((gate_up_one_kernel<T, W, kTail, decltype(staged)::value>), dim3(tf, a.top_k), dim3(64 * w1),
                       w1 * 2048 + (staged ? staged_bytes(d) : 0), s, e, a.ids, a.weights, static_cast<const u16*>(a.x), d, f, a.act, made<T>(w));
  };
  const uint32_t w2 = stream_waves(td, uint64_t(chunks_of(f)) * a.top_k, 16);
  const auto down = [&](auto staged) {
    hipLaunchKernelGGL((down_one_kernel<T, W, kTail, decltype(staged)::value>), dim3(td), dim3(64 * w2),
                       w2 * 1024 + (staged ? a.top_k * staged_bytes(f) : 0), s, e, a.ids, a.top_k, w.h, kHalf ? w.scale : nullptr, d, f,
                       static_cast<const u16*>(a.residual), static_cast<u16*>(a.y));
  };
  constexpr std::bool_constant<std::is_same_v<W, Rows16<T>>> k16{};
  if (k16 && staged_bytes(d) <= kStagedBytes) up(k16);
  else up(std::false_type{});
  launch_fit<T>(w, f, true, s);
  if (k16 && a.top_k * staged_bytes(f) <= kStagedBytes) down(k16);
  else down(std::false_type{});
  return int(hipGetLastError());
}

template <class T>
int forward_one_q4(const ExpertMap& e, uint32_t d, uint32_t f, const tsa_ffn_args& a, const Forward& w, hipStream_t s) {
  const uint32_t tf = (f + 15) / 16, td = (d + 15) / 16;
  const uint32_t w1 = q4_waves(uint64_t(tf) * a.top_k, (d + 511) / 512);
  hipLaunchKernelGGL((gate_up_q4_kernel<T>), dim3(tf, a.top_k), dim3(64 * w1), w1 * 2 * Q4Stage<2>::kBytes, s, e, a.ids, a.weights,
                     static_cast<const u16*>(a.x), d, f, a.act, made<T>(w));
  launch_fit<T>(w, f, true, s);
  const uint32_t w2 = q4_waves(td, uint64_t((f + 1023) / 1024) * a.top_k);
  hipLaunchKernelGGL((down_q4_kernel<T>), dim3(td), dim3(64 * w2), w2 * 2 * Q4Stage<1>::kBytes, s, e, a.ids, a.top_k, w.h,
                     std::is_same_v<T, F16> ? w.scale : nullptr, d, f, static_cast<const u16*>(a.residual), static_cast<u16*>(a.y));
  return int(hipGetLastError());
}

template <class T, class W, int CT, bool kTail>
int forward_few(const ExpertMap& e, uint32_t d, uint32_t f, const tsa_ffn_args& a, const Forward& w, hipStream_t s) {
  if (int err = launch_plan(e, a.ids, w.plan, 16 * CT, s)) return err;
  const uint32_t tiles = most_tiles(w.plan.pairs, e.n, 16 * CT), tf = (f + 15) / 16, td = (d + 31) / 32;
  const uint32_t w1 = stream_waves(uint64_t(tf) * tiles, chunks_of(d), most_waves(CT));
  hipLaunchKernelGGL((gate_up_few_kernel<T, W, CT, kTail>), dim3(tf, tiles), dim3(64 * w1), w1 * CT * 2048, s, w.plan,
                     static_cast<const u16*>(a.x), a.x_stride, d, f, a.act, made<T>(w));
  launch_fit<T>(w, f, false, s);
  const uint32_t w2 = stream_waves(uint64_t(td) * tiles, chunks_of(f), most_waves(CT));
  hipLaunchKernelGGL((down_few_kernel<T, W, CT, kTail>), dim3(td, tiles), dim3(64 * w2), w2 * CT * 2048, s, w.plan, w.h, d, f,
                     w.out);
  return launch_combine<T>(w, d, a, s);
}

// Whether 4-bit weights are streamed: up to 24 pairs an expert; more where a product's workgroups, taken one after the other as in the
// linear product (11 ns a value of the sum, 256 at a time), end before its tiles (25 ns, 512 at a time), with half a tile of
// rows more for every expert. Streamed and in tiles: one expert of 4096 x 4096, 96 rows 136 and 212 us, 256 rows 272 and 213; 3 of
// 2048 x 2048, 200 rows 82 and 117; 8 of 16 of 1024 x 2048, 64 rows (32 pairs each) 122 and 107.
bool stream_few(uint32_t n, uint32_t d, uint32_t f, uint32_t rows, uint32_t top_k, bool tiles) {
  const uint64_t pairs = uint64_t(rows) * top_k, short_tiles = (n + 1) / 2;
  if (pairs <= uint64_t(tiles ? 24 : 64) * n) return true;
  if (!tiles) return false;
  const uint64_t r = pairs / 64 + short_tiles, t = pairs / 128 + short_tiles;
  const auto turns = [](uint64_t groups, uint64_t at_once) { return double(groups > at_once ? groups : at_once) / double(at_once); };
  return 11.0 * (turns(r * (f / 16), 256) * d + turns(r * (d / 32), 256) * f) <=
         25.0 * (turns(t * ((f + 63) / 64), 512) * d + turns(t * ((d + 127) / 128), 512) * f);
}

// 4-bit weights, few rows: up to so many pairs an expert (if all are asked for alike) as CT tiles of 16 hold.
template <class T, bool kTail>
int forward_few_q4(const ExpertMap& e, uint32_t d, uint32_t f, const tsa_ffn_args& a, const Forward& w, hipStream_t s) {
  typedef RowsQ4<T> W;
  const uint32_t each = w.plan.pairs / e.n;
  if (each <= 8) return forward_few<T, W, 1, kTail>(e, d, f, a, w, s);
  if (each <= 24) return forward_few<T, W, 2, kTail>(e, d, f, a, w, s);
  return forward_few<T, W, 4, kTail>(e, d, f, a, w, s);
}

template <class T, bool kQ4, class S>
int forward_tiles(const ExpertMap& e, uint32_t d, uint32_t f, const tsa_ffn_args& a, const Forward& w, hipStream_t s) {
  if (int err = launch_plan(e, a.ids, w.plan, S::kB, s)) return err;
  const uint32_t tiles = most_tiles(w.plan.pairs, e.n, S::kB);
  // Gate and up as wide as they come, 1850 us in a prompt of 4001 rows where 192 rows a tile take 1955; down, whose sums are longer
  // and whose tiles are fewer, 192 rows: 1093 us, 1240.
  typedef std::conditional_t<std::is_same_v<S, BigTile>, WideTile, S> U;
  constexpr uint32_t kF = kQ4 ? U::kA / 4 : U::kA / 2, kD = kQ4 ? S::kA / 2 : S::kA;  // columns a tile
  const dim3 up(tiles * ((f + kF - 1) / kF)), down(tiles * ((d + kD - 1) / kD));
  const u16* x = static_cast<const u16*>(a.x);
  if constexpr (kQ4) {
    hipLaunchKernelGGL((gate_up_q4_tile_kernel<T>), up, dim3(kTileThreads), S::kLds, s, w.plan, x, a.x_stride, d, f, a.act, made<T>(w));
    launch_fit<T>(w, f, false, s);
    hipLaunchKernelGGL((down_q4_tile_kernel<T>), down, dim3(kTileThreads), S::kLds, s, w.plan, w.h, d, f, w.out);
  } else {
    hipLaunchKernelGGL((gate_up_tile_kernel<T, U>), up, dim3(kTileThreads), U::kLds, s, w.plan, x, a.x_stride, d, f, a.act, made<T>(w));
    launch_fit<T>(w, f, false, s);
    hipLaunchKernelGGL((down_tile_kernel<T, S>), down, dim3(kTileThreads), S::kLds, s, w.plan, w.h, d, f, w.out);
  }
  return launch_combine<T>(w, d, a, s);
}

template <class T, bool kQ4>
int forward(const ExpertMap& e, uint32_t d, uint32_t f, const tsa_ffn_args& a, void* ws, hipStream_t s) {
  typedef std::conditional_t<kQ4, RowsQ4<T>, Rows16<T>> W;
  Room room(ws);
  const Forward w = take_forward(room, e.n, d, f, a.rows, a.top_k, kQ4 || std::is_same_v<T, F16>);
  const bool tail = d % kChunk || f % kChunk;
  if constexpr (kQ4) {
    if (a.rows == 1 && d % 256 == 0 && f % 256 == 0 && aligned16(a.x, 0) && wide_weights(e)) return forward_one_q4<T>(e, d, f, a, w, s);
    if (a.rows > 1 && stream_few(e.n, d, f, a.rows, a.top_k, wide_rows(e, d, f, true, a.x, a.x_stride)))
      return tail ? forward_few_q4<T, true>(e, d, f, a, w, s) : forward_few_q4<T, false>(e, d, f, a, w, s);
  }
  // (Two rows of 16-bit weights and more are no slower in small tiles: 32 rows, 8 of 128 experts, 146 us and 156 streamed.)
  if (a.rows == 1) return tail ? forward_one<T, W, true>(e, d, f, a, w, s) : forward_one<T, W, false>(e, d, f, a, w, s);
  if (wide_rows(e, d, f, kQ4, a.x, a.x_stride)) {
    if constexpr (!kQ4)
      if (small_tiles(a.rows, a.top_k, e.n, d, f)) return forward_tiles<T, false, SmallTile>(e, d, f, a, w, s);
    return forward_tiles<T, kQ4, std::conditional_t<kQ4, WideTile, BigTile>>(e, d, f, a, w, s);
  }
  if (int err = launch_plan(e, a.ids, w.plan, 64, s)) return err;
  const uint32_t tiles = most_tiles(w.plan.pairs, e.n, 64);
  hipLaunchKernelGGL((gate_up_any_kernel<T, kQ4>), dim3(tiles * ((f + 63) / 64)), dim3(256), 0, s, w.plan,
                     static_cast<const u16*>(a.x), a.x_stride, d, f, a.act, made<T>(w));
  launch_fit<T>(w, f, false, s);
  hipLaunchKernelGGL((down_any_kernel<T, kQ4>), dim3(tiles * ((d + 63) / 64)), dim3(256), 0, s, w.plan, w.h, d, f, w.out);
  return launch_combine<T>(w, d, a, s);
}

}  // namespace
}  // namespace op

uint64_t ffn_workspace(uint32_t n, uint32_t d, uint32_t f, uint32_t w_type, uint32_t rows, uint32_t top_k) {
  op::Room room(nullptr);
  op::take_forward(room, n, d, f, rows, top_k, w_type != TSA_BF16);  // (4-bit weights: x may be of either type)
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

}  // namespace tsa
