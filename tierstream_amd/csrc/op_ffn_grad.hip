// The gradients of the gated feed-forward blocks.
//
// b = down^T dy of every pair; with gate x and up x computed again, d w = <h, b>, dg = w b up act'(gate), du = w b act(gate) and
// w h; dx' = gate^T dg + up^T du, added over a row's pairs; d gate = dg^T x, d up = du^T x and d down = dy^T (w h) over an expert's
// pairs. dg, du and w h are rounded once to the operands' 16 bits (half precision: as what a power of two of their expert's leaves of
// them, so that none overflows or loses bits; the sums over an expert's pairs need one for all of them); b and dx' stay in 32
// bits. No sum depends on an order that changes.
#include "op_pairs.hpp"

namespace tsa {
namespace op {
namespace {

// The two largest values of a workgroup of four waves from its threads', by way of 8 places in LDS: wave by wave here, read
// behind a barrier.
__device__ __forceinline__ void leave_peaks(float (*tops)[2], float top_g, float top_h) {
  for (int s = 1; s < 64; s <<= 1) {
    top_g = fmaxf(top_g, __shfl_xor(top_g, s, 64));
    top_h = fmaxf(top_h, __shfl_xor(top_h, s, 64));
  }
  if ((threadIdx.x & 63u) == 0) {
    tops[threadIdx.x >> 6][0] = top_g;
    tops[threadIdx.x >> 6][1] = top_h;
  }
}
__device__ __forceinline__ float joint_peak(const float (*tops)[2], int i) {
  return fmaxf(fmaxf(tops[0][i], tops[1][i]), fmaxf(tops[2][i], tops[3][i]));
}

// Half precision: dg | du and w h of every pair behind the powers of two that the largest of its expert choose, whose inverses go
// to scale, one array after the other. peaks: [tile][shares][2], as the workgroups that made the values left them.
// kFitParts workgroups a tile of pairs. Bound by the bytes: 16384 pairs of 768 (226 MB) 43 us, 5.2 TB/s; 74 of 512 4 us, a launch.
constexpr uint32_t kFitParts = 16;
template <int kWide>
__device__ __forceinline__ void fit_values(const float* from, u16* to, uint32_t n, float by) {
  typedef float wide_t __attribute__((ext_vector_type(kWide)));
  typedef u16 bits_t __attribute__((ext_vector_type(kWide)));
#pragma unroll 4
  for (uint32_t i = threadIdx.x; i < n / kWide; i += 256) {
    const wide_t x = reinterpret_cast<const wide_t*>(from)[i];
    bits_t o;
#pragma unroll
    for (int q = 0; q < kWide; ++q) o[q] = F16::down(x[q] * by);
    reinterpret_cast<bits_t*>(to)[i] = o;
  }
}
template <int kWide>
__global__ __launch_bounds__(256) void fit_grads_kernel(Plan p, uint32_t rows_per_tile, uint32_t f, uint32_t shares, const float* peaks,
                                                        const float* dgu, const float* wh, u16* dgu_to, u16* wh_to, float* scale) {
  __shared__ float tops[4][2];
  TileRows t;
  if (!tile_rows(p, blockIdx.x / kFitParts, rows_per_tile, t)) return;
  const uint32_t begin = p.first[t.e], tiles = (p.first[t.e + 1] - begin + rows_per_tile - 1) / rows_per_tile;  // of the expert
  const float* mine = peaks + uint64_t(t.tile - (t.first - begin) / rows_per_tile) * shares * 2;
  float top_g = 0.0f, top_h = 0.0f;
  for (uint64_t i = threadIdx.x; i < uint64_t(tiles) * shares; i += 256) {
    top_g = fmaxf(top_g, mine[2 * i]);
    top_h = fmaxf(top_h, mine[2 * i + 1]);
  }
  leave_peaks(tops, top_g, top_h);
  __syncthreads();
  const Fit g(joint_peak(tops, 0)), h(joint_peak(tops, 1));
  for (uint32_t r = blockIdx.x % kFitParts; r < t.rows; r += kFitParts) {
    const uint64_t pos = t.first + r;
    if (threadIdx.x == 0) {
      scale[pos] = g.up;
      scale[p.pairs + pos] = h.up;
    }
    fit_values<kWide>(dgu + pos * 2 * f, dgu_to + pos * 2 * f, 2 * f, g.down);
    fit_values<kWide>(wh + pos * f, wh_to + pos * f, f, h.down);
  }
}

// Of every pair: dg | du as one row of 2 f values, w h, and this tile's share of d w (d_share[f tile][sorted position]).
template <class T>
__global__ __launch_bounds__(256) void hidden_grad_any_kernel(Plan p, const u16* x, uint64_t x_stride, const u16* dy,
                                                              uint64_t dy_stride, const float* weights, uint32_t d, uint32_t f,
                                                              uint32_t act, held<T>* dgu, held<T>* wh, float* d_share,
                                                              float* peaks) {
  __shared__ TileMemory m;
  __shared__ float share[64][2], tops[4][2];
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
  float top_g = 0.0f, top_h = 0.0f;
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
        const float dg = w * back * u[i][j][q] * slope(act, g[i][j][q]), du = w * back * a, h = w * a * u[i][j][q];
        dgu[uint64_t(pos) * 2 * f + c] = Held<T>::of(dg);
        dgu[uint64_t(pos) * 2 * f + f + c] = Held<T>::of(du);
        wh[uint64_t(pos) * f + c] = Held<T>::of(h);
        top_g = peak(peak(top_g, dg), du);
        top_h = peak(top_h, h);
      }
    sum += __shfl_xor(sum, 16, 64);
    sum += __shfl_xor(sum, 32, 64);
    if (lane < 16) share[r][wave & 1u] = sum;
  }
  if (std::is_same_v<T, F16>) leave_peaks(tops, top_g, top_h);
  __syncthreads();
  if (std::is_same_v<T, F16> && threadIdx.x < 2) peaks[(uint64_t(t.tile) * tf + ft) * 2 + threadIdx.x] = joint_peak(tops, threadIdx.x);
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
// the rows' map where left_map, right where right_map; times scale (null: 1) of the expert's first position.
template <class T>
__global__ __launch_bounds__(256) void weight_grad_any_kernel(Plan p, const u16* left, uint64_t left_stride, bool left_map,
                                                              uint32_t n_left, const u16* right, uint64_t right_stride,
                                                              bool right_map, uint32_t n_right, const float* scale, u16* out) {
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
    const float up = scale && n ? scale[first] : 1.0f;
    each64(acc, [&](uint32_t i, uint32_t j, float v) {
      if (a0 + i < n_left && b0 + j < n_right) out[(uint64_t(e) * n_right + b0 + j) * n_left + a0 + i] = T::down(v * up);
    });
    __syncthreads();
  }
}

// d w of every pair: its shares, in their order.
struct WeightShares {
  uint32_t n = 0;
  const float* share = nullptr;
  float* dweights = nullptr;
};
__device__ __forceinline__ void weights_grad(const Plan& p, const WeightShares& w, uint32_t block, uint32_t n_blocks) {
  for (uint64_t i = uint64_t(block) * 256 + threadIdx.x; i < p.pairs; i += uint64_t(n_blocks) * 256) {
    const int32_t at = p.at[i];
    float s = 0.0f;
    if (at >= 0)
#pragma unroll 4
      for (uint32_t k = 0; k < w.n; ++k) s += w.share[uint64_t(k) * p.pairs + uint32_t(at)];
    w.dweights[i] = s;
  }
}

// dx by the first blocks, d w by the others: two sums that need nothing of each other.
template <class T, int kWide>
__global__ __launch_bounds__(256) void sums_kernel(Combine c, Plan p, WeightShares w) {
  if (blockIdx.x < c.n_blocks) combine<T, kWide>(c, blockIdx.x);
  else weights_grad(p, w, blockIdx.x - c.n_blocks, gridDim.x - c.n_blocks);
}

// back = down^T dy of every pair: in 32 bits, for the kernel behind it. (One kernel for all three products needs 192 accumulators
// a lane, so one workgroup a CU: 496 us in a training step of 128 experts of 2048 x 768 with 16384 pairs, where the two take 413:
// 123 and 290. The input's gradient takes 237 there, the sums over pairs 27. All three products are bound by their loads, 2.8
// to 3.4 TB/s of weights: leaving out the empty half of short tiles changes nothing, nor do tiles of half the rows.)
template <class T, class S>
__global__ __launch_bounds__(kTileThreads, 2) void back_tile_kernel(Plan p, const u16* dy, uint64_t dy_stride, uint32_t d,
                                                                    uint32_t f, float* back) {
  extern __shared__ __attribute__((aligned(1024))) f32x4 memory[];
  constexpr int NI = S::NI, MJ = S::MJ;
  TileRows t;
  uint32_t at;
  if (!tile_of<S>(p, (f + S::kA - 1) / S::kA, t, at)) return;
  TileColumnsSource<NI, false> w(d, threadIdx.x >> 6 & 1u, reinterpret_cast<const u16*>(p.part[3 * t.e + 2]), f, at * S::kA, f);
  auto dys = mapped_rows<MJ>(t, dy, dy_stride, d);
  f32x4 acc[NI][MJ] = {};
  tile_product<T, NI, MJ, S::NB>(w, dys, d, lds_offset(memory), acc);
  FloatRows o{back + uint64_t(t.first) * f, f, t.rows, at * S::kA, f};
  hand_out<NI, MJ>(memory, acc, o);
}

// As hidden_grad_any_kernel from gate's and up's products and `back`, 16 NI columns of d_ff.
template <class T, class S>
__global__ __launch_bounds__(kTileThreads, 2) void hidden_grad_tile_kernel(Plan p, const u16* x, uint64_t x_stride,
                                                                           const float* back, const float* weights, uint32_t d,
                                                                           uint32_t f, uint32_t act, held<T>* dgu, held<T>* wh,
                                                                           float* d_share, float* peaks) {
  extern __shared__ __attribute__((aligned(1024))) f32x4 memory[];
  constexpr int NI = S::NI, MJ = S::MJ, kHalf = NI / 2;
  float* share = reinterpret_cast<float*>(memory) + S::kLds / 4 - 2 * S::kB;  // (behind what hand_out uses, as tops)
  float (*tops)[2] = reinterpret_cast<float (*)[2]>(share - 8);
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
  TileRows t;
  uint32_t at;
  if (!tile_of<S>(p, (f + 16 * NI - 1) / (16 * NI), t, at)) return;
  const uint32_t f0 = at * 16 * NI;
  f32x4 gu[NI][MJ] = {};
  auto ws = gate_up_source<NI>(p, t, d, f, f0);
  auto xs = mapped_rows<MJ>(t, x, x_stride, d);
  tile_product<T, NI, MJ, S::NB>(ws, xs, d, lds_offset(memory), gu);
  float w[MJ];
  uint32_t pos[MJ];
#pragma unroll
  for (int j = 0; j < MJ; ++j) {
    const uint32_t r = (wave >> 1) * 16 * MJ + 16 * j + (lane & 15u);
    pos[j] = t.first + (r < t.rows ? r : t.rows - 1);
    w[j] = weights ? weights[p.pair[pos[j]]] : 1.0f;
  }
  f32x4 h[kHalf][MJ];
  float top_g = 0.0f, top_h = 0.0f;
  __syncthreads();  // the product's reads are done
#pragma unroll
  for (int j = 0; j < MJ; ++j) {
    float sum = 0.0f;
    f32x4 b[kHalf];
    bool in[kHalf];  // (behind the last column stands the last one again: not part of the sum)
#pragma unroll
    for (int i = 0; i < kHalf; ++i) {
      const uint32_t c = f0 + (wave & 1u) * 8 * NI + 16 * i + (lane >> 4) * 4;
      in[i] = c < f;
      b[i] = in[i] ? *reinterpret_cast<const f32x4*>(back + uint64_t(pos[j]) * f + c) : f32x4{0, 0, 0, 0};
    }
#pragma unroll
    for (int i = 0; i < kHalf; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float g = gu[i][j][q], u = gu[i + kHalf][j][q], a = activate(act, g);
        sum += in[i] ? a * u * b[i][q] : 0.0f;
        h[i][j][q] = w[j] * a * u;
        gu[i][j][q] = w[j] * b[i][q] * u * slope(act, g);  // dg, du in the products' places
        gu[i + kHalf][j][q] = w[j] * b[i][q] * a;
        if (std::is_same_v<T, F16> && in[i] && (wave >> 1) * 16 * MJ + 16 * j + (lane & 15u) < t.rows) {
          top_g = peak(peak(top_g, gu[i][j][q]), gu[i + kHalf][j][q]);
          top_h = peak(top_h, h[i][j][q]);
        }
      }
    sum += __shfl_xor(sum, 16, 64);
    sum += __shfl_xor(sum, 32, 64);
    if (lane < 16) share[2 * ((wave >> 1) * 16 * MJ + 16 * j + lane) + (wave & 1u)] = sum;
  }
  if (std::is_same_v<T, F16>) leave_peaks(tops, top_g, top_h);
  hand_out_held<T, kHalf, MJ>(memory, h, wh + uint64_t(t.first) * f, f, t.rows, f0, f);  // (behind its barrier `share` and `tops` are whole)
  if (std::is_same_v<T, F16> && threadIdx.x < 2)
    peaks[(uint64_t(t.tile) * ((f + 16 * NI - 1) / (16 * NI)) + at) * 2 + threadIdx.x] = joint_peak(tops, threadIdx.x);
  if (threadIdx.x < t.rows) d_share[uint64_t(at) * p.pairs + t.first + threadIdx.x] = share[2 * threadIdx.x] + share[2 * threadIdx.x + 1];
#pragma unroll
  for (int half = 0; half < 2; ++half) {
#pragma unroll
    for (int i = 0; i < kHalf; ++i)
#pragma unroll
      for (int j = 0; j < MJ; ++j) h[i][j] = gu[i + kHalf * half][j];
    hand_out_held<T, kHalf, MJ>(memory, h, dgu + uint64_t(t.first) * 2 * f + half * f, uint64_t(2) * f, t.rows, f0, f);
  }
}

template <class T, class S>
__global__ __launch_bounds__(kTileThreads, 2) void input_grad_tile_kernel(Plan p, const u16* dgu, uint32_t d, uint32_t f,
                                                                          float* out) {
  extern __shared__ __attribute__((aligned(1024))) f32x4 memory[];
  constexpr int NI = S::NI, MJ = S::MJ;
  TileRows t;
  uint32_t at;
  if (!tile_of<S>(p, (d + S::kA - 1) / S::kA, t, at)) return;
  f32x4 acc[NI][MJ] = {};
  const auto add = [&](uint32_t half) {
    TileColumnsSource<NI, false> w(f, threadIdx.x >> 6 & 1u, reinterpret_cast<const u16*>(p.part[3 * t.e + half]), d, at * S::kA, d);
    auto v = sorted_rows<MJ>(t, dgu + half * f, uint64_t(2) * f, f);
    tile_product<T, NI, MJ, S::NB>(w, v, f, lds_offset(memory), acc);
  };
  add(0);
  add(1);
  FloatRows o{out + uint64_t(t.first) * d, d, t.rows, at * S::kA, d};
  hand_out<NI, MJ>(memory, acc, o);
}

// As weight_grad_any_kernel, out[e][b][a]: a tile of columns a of `left` and b of `right` a workgroup, the sum over the expert's
// pairs. One of the two is read through the rows' map (kMapLeft: left). Columns from n_right on belong to out2 (the
// gradients of gate and up are one product). 128 experts of 2048 x 768 (1.2 GB written): 454 us, 2.7 TB/s: a sum of 128 pairs is
// 4 steps, so a tile is its first loads and its stores (the matrix cores are busy 19 % of the time). Tiles of 128 x 128, three a CU: 523 for 492; an expert's on one XCD: 560.
template <class T, class S, bool kMapLeft>
__device__ __forceinline__ void weight_grad_tile(f32x4* memory, uint32_t block, const Plan& p, const u16* left, uint64_t left_stride,
                                                 uint32_t n_left, const u16* right, uint64_t right_stride, uint32_t n_right,
                                                 uint32_t n_outs, const float* scale, u16* out, u16* out2) {
  constexpr int NI = S::NI, MJ = S::MJ;
  uint32_t* map = reinterpret_cast<uint32_t*>(memory) + S::kLds / 4;
  const uint32_t wave = threadIdx.x >> 6;
  const uint32_t ta = (n_left + S::kA - 1) / S::kA, tb = (n_right + S::kB - 1) / S::kB, per = ta * tb * n_outs;
  const uint32_t e = block / per, in = block % per;
  const uint32_t a0 = in % ta * S::kA, which = in / ta / tb, b0 = in / ta % tb * S::kB;
  const uint32_t first = p.first[e], pairs = p.first[e + 1] - first;
  right += which * n_right;
  f32x4 acc[NI][MJ] = {};
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
      TileColumnsSource<NI, true> l(pairs, wave & 1u, left, left_stride, a0, n_left, map);
      TileColumnsSource<MJ, false> r(pairs, wave >> 1, right + uint64_t(first) * right_stride, right_stride, b0, n_right);
      tile_product<T, NI, MJ, S::NB>(l, r, pairs, lds_offset(memory), acc, refill);
    } else {
      TileColumnsSource<NI, false> l(pairs, wave & 1u, left + uint64_t(first) * left_stride, left_stride, a0, n_left);
      TileColumnsSource<MJ, true> r(pairs, wave >> 1, right, right_stride, b0, n_right, map);
      tile_product<T, NI, MJ, S::NB>(l, r, pairs, lds_offset(memory), acc, refill);
    }
    if constexpr (std::is_same_v<T, F16>) {
      const float up = scale[first];
#pragma unroll
      for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int j = 0; j < MJ; ++j) acc[i][j] *= up;
    }
  }
  hand_out_bits<T, NI, MJ, true>(memory, acc, (which ? out2 : out) + (uint64_t(e) * n_right + b0) * n_left + a0, n_left, n_right - b0,
                           n_left - a0);
}

// The gradients of gate and up by the first `n_up` workgroups, down's by the others.
template <class T, class S>
__global__ __launch_bounds__(kTileThreads, 2) void weight_grad_tile_kernel(Plan p, uint32_t n_up, const u16* x, uint64_t x_stride,
                                                                           const u16* dy, uint64_t dy_stride, uint32_t d,
                                                                           uint32_t f, const u16* dgu, const u16* wh, const float* scale,
                                                                           u16* dgate, u16* dup, u16* ddown) {
  extern __shared__ __attribute__((aligned(1024))) f32x4 memory[];
  if (blockIdx.x < n_up)
    weight_grad_tile<T, S, true>(memory, blockIdx.x, p, x, x_stride, d, dgu, uint64_t(2) * f, f, 2, scale, dgate, dup);
  else
    weight_grad_tile<T, S, false>(memory, blockIdx.x - n_up, p, wh, f, f, dy, dy_stride, d, 1, scale + p.pairs, ddown, nullptr);
}

// ---- launches ----
struct Backward {
  Plan plan;
  u16 *dgu, *wh;
  float *share, *out, *back;  // (back and out share their place: out is written behind back's last reader)
  float *dgu_wide, *wh_wide, *scale, *peaks;  // half precision
};
Backward take_backward(Room& r, uint32_t n, uint32_t d, uint32_t f, uint32_t rows, uint32_t top_k, bool half) {
  const uint64_t pairs = uint64_t(rows) * top_k;
  Backward w;
  w.plan = take_plan(r, n, uint32_t(pairs), top_k, 64);
  w.dgu_wide = r.take<float>(half ? pairs * 2 * f : 0);
  w.wh_wide = r.take<float>(half ? pairs * f : 0);
  w.scale = r.take<float>(half ? 2 * pairs : 0);
  w.peaks = r.take<float>(half ? uint64_t(2) * most_tiles(uint32_t(pairs), n, 64) * ((f + 31) / 32) : 0);  // (the smallest tiles')
  w.dgu = r.take<u16>(pairs * 2 * f);
  w.wh = r.take<u16>(pairs * f);
  w.share = r.take<float>(pairs * ((f + 31) / 32));  // (the narrowest tile's)
  w.out = w.back = r.take<float>(pairs * (d > f ? d : f));
  return w;
}

// Where the hidden gradients are left, and the launch that makes operands of them.
template <class T>
held<T>* made_dgu(const Backward& w) {
  if constexpr (std::is_same_v<T, F16>) return w.dgu_wide;
  else return w.dgu;
}
template <class T>
held<T>* made_wh(const Backward& w) {
  if constexpr (std::is_same_v<T, F16>) return w.wh_wide;
  else return w.wh;
}
template <class T>
void launch_fit(const Backward& w, uint32_t tiles, uint32_t rows_per_tile, uint32_t f, uint32_t shares, hipStream_t s) {
  if constexpr (std::is_same_v<T, F16>) {
    const dim3 grid(tiles * kFitParts);
    if (f % 4 == 0)
      hipLaunchKernelGGL((fit_grads_kernel<4>), grid, dim3(256), 0, s, w.plan, rows_per_tile, f, shares, w.peaks, w.dgu_wide, w.wh_wide, w.dgu, w.wh, w.scale);
    else
      hipLaunchKernelGGL((fit_grads_kernel<1>), grid, dim3(256), 0, s, w.plan, rows_per_tile, f, shares, w.peaks, w.dgu_wide, w.wh_wide, w.dgu, w.wh, w.scale);
  }
}

template <class T>
int launch_sums(const Backward& w, const tsa_ffn_grad_args& a, uint32_t d, uint32_t shares, hipStream_t s) {
  bool wide = true;
  Combine c;
  if (a.dx) {
    c = combine_of(w.plan, a.rows, d, w.out, nullptr, nullptr, 0, a.dx, a.dx_stride, wide);
    if (std::is_same_v<T, F16>) c.scale = w.scale;
  }
  WeightShares g;
  g.n = shares;
  g.share = w.share;
  g.dweights = a.dweights;
  const uint32_t n = c.n_blocks + (a.dweights ? blocks((w.plan.pairs + 255) / 256) : 0);
  if (n == 0) return 0;
  if (wide) hipLaunchKernelGGL((sums_kernel<T, 4>), dim3(n), dim3(256), 0, s, c, w.plan, g);
  else hipLaunchKernelGGL((sums_kernel<T, 1>), dim3(n), dim3(256), 0, s, c, w.plan, g);
  return int(hipGetLastError());
}

template <class T, class S, class W>
int backward_tiles(const ExpertMap& e, uint32_t d, uint32_t f, const tsa_ffn_grad_args& a, void* ws, hipStream_t s) {
  Room room(ws);
  const Backward w = take_backward(room, e.n, d, f, a.rows, a.top_k, std::is_same_v<T, F16>);
  if (int err = launch_plan(e, a.ids, w.plan, S::kB, s)) return err;
  const auto of = [](uint32_t n, uint32_t each) { return (n + each - 1) / each; };
  const uint32_t tiles = most_tiles(w.plan.pairs, e.n, S::kB), shares = of(f, S::kA / 2);
  const u16 *x = static_cast<const u16*>(a.x), *dy = static_cast<const u16*>(a.dy);
  if (tiles) {
    hipLaunchKernelGGL((back_tile_kernel<T, S>), dim3(tiles * of(f, S::kA)), dim3(kTileThreads), S::kLds, s, w.plan, dy, a.dy_stride, d,
                       f, w.back);
    hipLaunchKernelGGL((hidden_grad_tile_kernel<T, S>), dim3(tiles * shares), dim3(kTileThreads), S::kLds, s, w.plan, x, a.x_stride,
                       w.back, a.weights, d, f, a.act, made_dgu<T>(w), made_wh<T>(w), w.share, w.peaks);
    launch_fit<T>(w, tiles, S::kB, f, shares, s);
  }
  if (a.dx && tiles)
    hipLaunchKernelGGL((input_grad_tile_kernel<T, S>), dim3(tiles * of(d, S::kA)), dim3(kTileThreads), S::kLds, s, w.plan, w.dgu, d, f,
                       w.out);
  if (tiles)
    if (int err = launch_sums<T>(w, a, d, shares, s)) return err;
  if (a.dgate) {
    const uint32_t n_up = e.n * of(d, W::kA) * of(f, W::kB) * 2, n_down = e.n * of(f, W::kA) * of(d, W::kB);
    hipLaunchKernelGGL((weight_grad_tile_kernel<T, W>), dim3(n_up + n_down), dim3(kTileThreads), W::kLds + 4 * kMapRing, s, w.plan, n_up,
                       x, a.x_stride, dy, a.dy_stride, d, f, w.dgu, w.wh, w.scale, static_cast<u16*>(a.dgate), static_cast<u16*>(a.dup),
                       static_cast<u16*>(a.ddown));
  }
  return int(hipGetLastError());
}

template <class T>
int backward(const ExpertMap& e, uint32_t d, uint32_t f, const tsa_ffn_grad_args& a, void* ws, hipStream_t s) {
  if (wide_rows(e, d, f, false, a.x, a.x_stride) && aligned16(a.dy, 2 * a.dy_stride) && a.dy_stride < 1u << 24 && aligned16(a.dgate, 0) && aligned16(a.dup, 0) &&
      aligned16(a.ddown, 0)) {
    // The weights' gradients choose by themselves: 4 experts of 512 x 1024 (64 wide tiles) 173 us in all with wide tiles and 141
    // with small ones, one of 2048 x 2048 (128) 107 and 112, 8 of 4096 x 2048 (2048) 337 and 480.
    const bool small = small_tiles(a.rows, a.top_k, e.n, d, f);
    const bool small_out = uint64_t(e.n) * ((d + WideTile::kA - 1) / WideTile::kA) * ((f + WideTile::kB - 1) / WideTile::kB) < 100;
    if (small)
      return small_out ? backward_tiles<T, SmallTile, SmallTile>(e, d, f, a, ws, s) : backward_tiles<T, SmallTile, WideTile>(e, d, f, a, ws, s);
    return small_out ? backward_tiles<T, BigTile, SmallTile>(e, d, f, a, ws, s) : backward_tiles<T, BigTile, WideTile>(e, d, f, a, ws, s);
  }
  Room room(ws);
  const Backward w = take_backward(room, e.n, d, f, a.rows, a.top_k, std::is_same_v<T, F16>);
  if (int err = launch_plan(e, a.ids, w.plan, 64, s)) return err;
  const uint32_t tiles = most_tiles(w.plan.pairs, e.n, 64), tf = (f + 63) / 64, td = (d + 63) / 64;
  const u16 *x = static_cast<const u16*>(a.x), *dy = static_cast<const u16*>(a.dy);
  if (tiles) {
    hipLaunchKernelGGL((hidden_grad_any_kernel<T>), dim3(tiles * tf), dim3(256), 0, s, w.plan, x, a.x_stride, dy, a.dy_stride,
                       a.weights, d, f, a.act, made_dgu<T>(w), made_wh<T>(w), w.share, w.peaks);
    launch_fit<T>(w, tiles, 64, f, tf, s);
  }
  if (a.dx && tiles)
    hipLaunchKernelGGL((input_grad_any_kernel<T>), dim3(tiles * td), dim3(256), 0, s, w.plan, w.dgu, d, f, w.out);
  if (tiles)
    if (int err = launch_sums<T>(w, a, d, tf, s)) return err;
  if (a.dgate) {
    constexpr bool kHalf = std::is_same_v<T, F16>;
    const uint32_t g = blocks(uint64_t(e.n) * tf * td);
    for (int half = 0; half < 2; ++half)
      hipLaunchKernelGGL((weight_grad_any_kernel<T>), dim3(g), dim3(256), 0, s, w.plan, x, a.x_stride, true, d,
                         w.dgu + half * uint64_t(f), uint64_t(2) * f, false, f,
                         kHalf ? w.scale : nullptr, static_cast<u16*>(half ? a.dup : a.dgate));
    hipLaunchKernelGGL((weight_grad_any_kernel<T>), dim3(g), dim3(256), 0, s, w.plan, w.wh, uint64_t(f), false, f, dy,
                       a.dy_stride, true, d, kHalf ? w.scale + w.plan.pairs : nullptr, static_cast<u16*>(a.ddown));
  }
  return int(hipGetLastError());
}

}  // namespace
}  // namespace op

uint64_t ffn_backward_workspace(uint32_t n, uint32_t d, uint32_t f, uint32_t w_type, uint32_t rows, uint32_t top_k) {
  op::Room room(nullptr);
  op::take_backward(room, n, d, f, rows, top_k, w_type != TSA_BF16);
  return room.bytes;
}
int launch_ffn_backward(const ExpertMap& e, uint32_t d, uint32_t f, const tsa_ffn_grad_args& a, void* ws, hipStream_t stream) {
  return a.type == TSA_BF16 ? op::backward<op::Bf16>(e, d, f, a, ws, stream) : op::backward<op::F16>(e, d, f, a, ws, stream);
}

}  // namespace tsa
