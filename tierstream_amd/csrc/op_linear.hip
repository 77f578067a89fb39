// y = act(x W^T + bias) + residual.
#include "op_stream.hpp"
#include "op_tile.hpp"

namespace tsa {
namespace op {
namespace {

__device__ __forceinline__ void finish_linear(const tsa_linear_args& a, uint32_t row, uint32_t n, float v) {
  if (a.bias) v += load_as_float(a.bias, n, a.x_type);
  v = activate(a.act, v);
  if (a.residual) v += load_as_float(a.residual, uint64_t(row) * a.residual_stride + n, a.y_type);
  store_float(a.y, uint64_t(row) * a.y_stride + n, a.y_type, v);
}

// A tile's values to y, four columns at a time: in one access where the rows start so that it is aligned.
template <class T>
struct LinearOut {
  struct Fetched {
    u32x4 residual;
  };
  const tsa_linear_args& a;
  uint32_t r0, n0, n = 0;
  bool wide = false;
  f32x4 bias = {0, 0, 0, 0};

  __device__ __forceinline__ LinearOut(const tsa_linear_args& a_, uint32_t r0_, uint32_t n0_) : a(a_), r0(r0_), n0(n0_) {}
  __device__ __forceinline__ void columns(uint32_t c) {
    n = n0 + c;
    const uint64_t size = a.y_type == TSA_F32 ? 4 : 2;
    const uint64_t odd = (reinterpret_cast<uintptr_t>(a.y) | a.y_stride * size | reinterpret_cast<uintptr_t>(a.residual) |
                          a.residual_stride * size) & (4 * size - 1);
    wide = odd == 0 && n + 4 <= a.n_out;
    if (a.bias && wide)
#pragma unroll
      for (uint32_t i = 0; i < 4; ++i) bias[i] = T::up(static_cast<const u16*>(a.bias)[n + i]);
  }
  __device__ __forceinline__ Fetched fetch(uint32_t r) const {
    Fetched f = {{0, 0, 0, 0}};
    if (!a.residual || !wide || r0 + r >= a.rows) return f;
    const uint64_t at = uint64_t(r0 + r) * a.residual_stride + n;
    if (a.y_type == TSA_F32) {
      f.residual = *reinterpret_cast<const u32x4*>(static_cast<const float*>(a.residual) + at);
    } else {
      const uint2 v = *reinterpret_cast<const uint2*>(static_cast<const u16*>(a.residual) + at);
      f.residual[0] = v.x, f.residual[1] = v.y;
    }
    return f;
  }
  __device__ __forceinline__ void finish(uint32_t r, f32x4 v, const Fetched& f) const {
    const uint32_t row = r0 + r;
    if (row >= a.rows || n >= a.n_out) return;
    if (!wide) {
      for (uint32_t i = 0; i < 4; ++i)
        if (n + i < a.n_out) finish_linear(a, row, n + i, v[i]);
      return;
    }
    v += bias;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = activate(a.act, v[i]);
    const uint64_t at = uint64_t(row) * a.y_stride + n;
    if (a.y_type == TSA_F32) {
      if (a.residual) v += __builtin_bit_cast(f32x4, f.residual);
      *reinterpret_cast<f32x4*>(static_cast<float*>(a.y) + at) = v;
      return;
    }
    bits4 o;
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = T::down(v[i] + T::up(u16(f.residual[i / 2] >> (16 * (i & 1)))));
    *reinterpret_cast<bits4*>(static_cast<u16*>(a.y) + at) = o;
  }
};

// One row of 16-bit weights by 16 a workgroup, x in LDS.
template <class T, bool kTail>
__global__ __launch_bounds__(64 * most_waves(1)) void linear_one_kernel(tsa_linear_args a) {
  extern __shared__ f32x4 part[];
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  const uint32_t n = blockIdx.x * 16 + (lane & 15u);
  u16* xs = reinterpret_cast<u16*>(part + waves * 64);
  f32x4 acc[1][1] = {};
  stream_one<T, 1, kTail>((a.n_in + kChunk - 1) / kChunk, wave, waves, lds_offset(xs), [&](uint32_t c, Rows16<T> (&w)[1]) {
    w[0] = Rows16<T>(a.w, a.w_stride, n < a.n_out ? n : a.n_out - 1, a.n_in);
    return c * kChunk;
  }, [&] {
    stage_row(xs, static_cast<const u16*>(a.x), a.n_in);
    __syncthreads();
  }, acc);
  const f32x4 v[1] = {acc[0][0]};
  join_waves<1>(part, v, wave, waves, [&](auto&& sum) {
    if (wave != 0) return;
    const float s = sum(0)[0];
    if (lane < 16 && n < a.n_out) finish_linear(a, 0, n, s);
  });
}

// Few rows: a workgroup takes 16 R weight rows and 16 CT rows of x.
template <class T, class W, int R, int CT, bool kTail>
__global__ __launch_bounds__(64 * most_waves(CT)) void linear_few_kernel(tsa_linear_args a) {
  extern __shared__ f32x4 part[];
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  const uint32_t n0 = blockIdx.x * 16 * R, r0 = blockIdx.y * 16 * CT;
  f32x4 acc[R][CT] = {};
  stream_chunks<W, R, CT, kTail>((a.n_in + kChunk - 1) / kChunk, wave, waves, [&](uint32_t c, W (&w)[R], const u16* (&x)[CT]) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const uint32_t n = n0 + 16 * r + (lane & 15u);
      w[r] = W(a.w, a.w_stride, n < a.n_out ? n : a.n_out - 1, a.n_in);
    }
#pragma unroll
    for (int t = 0; t < CT; ++t) {
      const uint32_t row = a.rows == 1 ? 0 : r0 + 16 * t + (lane & 15u);
      x[t] = row < a.rows ? static_cast<const u16*>(a.x) + row * a.x_stride : nullptr;
    }
    return c * kChunk;
  }, acc);
  f32x4 v[R * CT];
#pragma unroll
  for (int i = 0; i < R * CT; ++i) v[i] = acc[i / CT][i % CT];
  join_waves<R * CT>(part, v, wave, waves, [&](auto&& sum) {
    for (uint32_t i = wave; i < R * CT; i += waves) {
      const f32x4 s = sum(i);
      const uint32_t n = n0 + 16 * (i / CT) + (lane & 15u), row = r0 + 16 * (i % CT) + (lane >> 4) * 4;
      if (n >= a.n_out) continue;
#pragma unroll
      for (uint32_t q = 0; q < 4; ++q)
        if (row + q < a.rows) finish_linear(a, row + q, n, s[q]);
    }
  });
}

// One row, 4-bit weights by way of LDS (n_in a multiple of 256).
template <class T>
__global__ __launch_bounds__(64 * kQ4Waves) void linear_q4_kernel(tsa_linear_args a) {
  extern __shared__ f32x4 memory[];
  __shared__ float part[kQ4Waves * 16];
  const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
  const uint32_t n0 = blockIdx.x * 16;
  float acc[1] = {};
  stream_q4<T, 1>((a.n_in + 1023) / 1024, wave, waves, a.n_out - n0 < 16 ? a.n_out - n0 : 16, a.n_in,
                  lds_offset(memory) + wave * 2 * Q4Stage<1>::kBytes, [&](uint32_t s, const char* (&base)[1], const u16*& x) {
                    base[0] = static_cast<const char*>(a.w) + uint64_t(n0) * (a.n_in / kQ4Block * kQ4Bytes);
                    x = static_cast<const u16*>(a.x);
                    return s * 1024;
                  }, acc);
  join_q4<1>(part, acc, wave, waves, [&](const float (&s)[1]) {
    if (n0 + lane < a.n_out) finish_linear(a, 0, n0 + lane, s[0]);
  });
}

template <class T>
int launch_q4(const tsa_linear_args& a, hipStream_t stream) {
  const uint32_t tn = (a.n_out + 15) / 16, waves = q4_waves(tn, (a.n_in + 1023) / 1024);
  hipLaunchKernelGGL((linear_q4_kernel<T>), dim3(tn), dim3(64 * waves), waves * 2 * Q4Stage<1>::kBytes, stream, a);
  return int(hipGetLastError());
}

template <class T, class W, int R, int CT>
int launch_few(const tsa_linear_args& a, hipStream_t stream) {
  const uint32_t tn = (a.n_out + 16 * R - 1) / (16 * R), tr = (a.rows + 16 * CT - 1) / (16 * CT);
  const uint32_t waves = stream_waves(uint64_t(tn) * tr, chunks_of(a.n_in), most_waves(CT));
  if (a.n_in % kChunk)
    hipLaunchKernelGGL((linear_few_kernel<T, W, R, CT, true>), dim3(tn, tr), dim3(64 * waves), waves * R * CT * 1024, stream, a);
  else
    hipLaunchKernelGGL((linear_few_kernel<T, W, R, CT, false>), dim3(tn, tr), dim3(64 * waves), waves * R * CT * 1024, stream, a);
  return int(hipGetLastError());
}

template <class T, class W>
int launch_few(const tsa_linear_args& a, hipStream_t stream) {
  if constexpr (std::is_same_v<W, RowsQ4<T>>) {
    if (a.rows > 32) return launch_few<T, W, 2, 4>(a, stream);
    if (a.rows > 16) return launch_few<T, W, 2, 2>(a, stream);
  } else if (a.rows == 1 && staged_bytes(a.n_in) <= kStagedBytes) {
    const uint32_t tn = (a.n_out + 15) / 16, waves = stream_waves(tn, chunks_of(a.n_in), most_waves(1));
    const uint32_t lds = waves * 1024 + uint32_t(staged_bytes(a.n_in));
    if (a.n_in % kChunk) hipLaunchKernelGGL((linear_one_kernel<T, true>), dim3(tn), dim3(64 * waves), lds, stream, a);
    else hipLaunchKernelGGL((linear_one_kernel<T, false>), dim3(tn), dim3(64 * waves), lds, stream, a);
    return int(hipGetLastError());
  }
  return launch_few<T, W, 1, 1>(a, stream);
}

// Many rows: big tiles, two workgroups a CU: one's products run under the other's epilogue. (Tiles of 256 x 256, one a CU,
// take less from L2 and LDS, but their epilogue stands alone: 575 us where 256 x 128 took 528, 2047 rows through 4096 x 28672
// with bias, tanh gelu and residual.)
template <class T, class S>
__global__ __launch_bounds__(kTileThreads, 2) void linear_tile_kernel(tsa_linear_args a) {
  extern __shared__ __attribute__((aligned(1024))) f32x4 memory[];
  constexpr int NI = S::NI, MJ = S::MJ;
  const uint32_t wave = threadIdx.x >> 6;
  const TileAt t = tile_at(blockIdx.x, (a.n_out + S::kA - 1) / S::kA, (a.rows + S::kB - 1) / S::kB);
  const uint32_t n0 = t.a * S::kA, r0 = t.b * S::kB;
  TileRowsSource<NI> w(a.n_in, wave & 1u, [&](uint32_t r) {
    const uint32_t n = n0 + r;
    return static_cast<const u16*>(a.w) + (n < a.n_out ? n : a.n_out - 1) * a.w_stride;
  });
  TileRowsSource<MJ> x(a.n_in, wave >> 1, [&](uint32_t r) {
    const uint32_t row = r0 + r;
    return static_cast<const u16*>(a.x) + (row < a.rows ? row : a.rows - 1) * a.x_stride;
  });
  f32x4 acc[NI][MJ] = {};
  tile_product<T, NI, MJ, S::NB>(w, x, a.n_in, lds_offset(memory), acc);
  LinearOut<T> out(a, r0, n0);
  hand_out<NI, MJ>(memory, acc, out);
}

template <class T, class S>
int launch_tile(const tsa_linear_args& a, hipStream_t stream) {
  const uint32_t tiles = (a.n_out + S::kA - 1) / S::kA * ((a.rows + S::kB - 1) / S::kB);
  hipLaunchKernelGGL((linear_tile_kernel<T, S>), dim3(tiles), dim3(kTileThreads), S::kLds, stream, a);
  return int(hipGetLastError());
}

// The same with 4-bit weights, 128 rows of them a tile.
template <class T>
__global__ __launch_bounds__(kTileThreads, 2) void linear_q4_tile_kernel(tsa_linear_args a) {
  extern __shared__ f32x4 memory[];
  const uint32_t wave = threadIdx.x >> 6;
  const TileAt t = tile_at(blockIdx.x, (a.n_out + 127) / 128, (a.rows + 127) / 128);
  const uint32_t n0 = t.a * 128, r0 = t.b * 128;
  TileQ4Source<T> w(a.n_in, wave & 1u, [&](uint32_t r) {
    const uint32_t n = n0 + r;
    return static_cast<const unsigned char*>(a.w) + uint64_t(n < a.n_out ? n : a.n_out - 1) * (a.n_in / kQ4Block * kQ4Bytes);
  });
  TileRowsSource<4> x(a.n_in, wave >> 1, [&](uint32_t r) {
    const uint32_t row = r0 + r;
    return static_cast<const u16*>(a.x) + (row < a.rows ? row : a.rows - 1) * a.x_stride;
  });
  f32x4 acc[8][4] = {};
  tile_product<T, 8, 4, 3>(w, x, a.n_in, lds_offset(memory), acc);
  f32x4 v[4][4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) v[i][j] = TileQ4Source<T>::whole(acc[i][j], acc[i + 4][j]);
  LinearOut<T> out(a, r0, n0);
  hand_out<4, 4>(memory, v, out);
}

template <class T>
int launch_q4_tile(const tsa_linear_args& a, hipStream_t stream) {
  const uint32_t tiles = (a.n_out + 127) / 128 * ((a.rows + 127) / 128);
  hipLaunchKernelGGL((linear_q4_tile_kernel<T>), dim3(tiles), dim3(kTileThreads), tile_lds(8, 4, 3), stream, a);
  return int(hipGetLastError());
}

// Rows of `from` to rows of `to_stride` values (a multiple of 8, zeros behind the n there are): what the tiles' loads take.
__global__ __launch_bounds__(256) void pack_kernel(const u16* from, uint64_t from_stride, uint32_t rows, uint32_t n, u16* to,
                                                   uint32_t to_stride) {
  const uint32_t per = to_stride / 8;
  const uint64_t total = uint64_t(rows) * per;
  for (uint64_t i = uint64_t(blockIdx.x) * 256 + threadIdx.x; i < total; i += uint64_t(gridDim.x) * 256) {
    const uint32_t row = uint32_t(i / per), c = uint32_t(i % per) * 8;
    *reinterpret_cast<bits8*>(to + uint64_t(row) * to_stride + c) = load_end(from + row * from_stride + c, int(n - c));
  }
}

bool aligned16(const void* p, uint64_t stride) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride % 8 == 0; }

}  // namespace
}  // namespace op

// Whether the weights are streamed. 16-bit ones up to 16 rows of x, above 4 only where small tiles are too few to keep up: 17 rows,
// 4096 x 28672: 73 us and 48 in tiles; 16 rows: 66 and 48, 7168 x 2048 19 and 27; 4 rows: 50 and 48. 4-bit ones by what the
// workgroups take one after the other: of 32 weight rows and 64 rows of x 11 ns a value of the sum (32 rows of x: 6), 256 of
// them at a time; a tile, half of whose time is unpacking, 25 ns, 512 at a time. Streamed and in tiles: 128 rows, 7168 x 2048
// (128 workgroups, 16 tiles) 81 and 178 us, 512 (512, 64) 152 and 178; 192 rows, 2048 x 7168 (672, 112) 69 and 60; 64 rows,
// 4096 x 28672 (896, 224) 173 and 111, 17 rows 96 and 109.
namespace {
bool streamed(const tsa_linear_args& a) {
  if (a.w_type == TSA_Q4) {
    const auto of = [](uint32_t n, uint32_t each) { return uint64_t(n + each - 1) / each; };
    const uint64_t groups = of(a.n_out, 32) * of(a.rows, a.rows > 32 ? 64 : 32), tiles = of(a.n_out, 128) * of(a.rows, 128);
    return a.rows <= 16 || (groups > 256 ? groups : 256) * (a.rows > 32 ? 10 : 6) <= (tiles > 512 ? tiles : 512) * 11;
  }
  return a.rows <= 4 || (a.rows <= 16 && (a.n_out < 16384 || a.n_in % 8 || !op::aligned16(a.x, a.x_stride) || !op::aligned16(a.w, a.w_stride)));
}
// What a call in tiles packs first: x, the weights, neither or both.
bool pack_x(const tsa_linear_args& a) { return !streamed(a) && (a.n_in % 8 || !op::aligned16(a.x, a.x_stride)); }
bool pack_w(const tsa_linear_args& a) {
  return !streamed(a) && a.w_type != TSA_Q4 && (a.n_in % 8 || !op::aligned16(a.w, a.w_stride));
}
int pack(const void* from, uint64_t stride, uint32_t rows, uint32_t n, void* to, hipStream_t stream) {
  const uint32_t wide = uint32_t(up_to(n, 8));
  const uint64_t blocks = (uint64_t(rows) * (wide / 8) + 255) / 256;
  hipLaunchKernelGGL(op::pack_kernel, dim3(uint32_t(blocks < 65536 ? blocks : 65536)), dim3(256), 0, stream,
                     static_cast<const op::u16*>(from), stride, rows, n, static_cast<op::u16*>(to), wide);
  return int(hipGetLastError());
}
}  // namespace

uint64_t linear_workspace(const tsa_linear_args& a) {
  return up_to(a.n_in, 8) * 2 * ((pack_x(a) ? a.rows : 0) + uint64_t(pack_w(a) ? a.n_out : 0));
}

int launch_linear(const tsa_linear_args& a0, void* workspace, hipStream_t stream) {
  tsa_linear_args a = a0;
  if (a.rows == 0 || a.n_out == 0) return 0;
  const bool bf16 = a.x_type == TSA_BF16, q4 = a.w_type == TSA_Q4;
  if (a.rows == 1 && q4 && a.n_in % 256 == 0 && op::aligned16(a.w, 0) && op::aligned16(a.x, 0))
    return bf16 ? op::launch_q4<op::Bf16>(a, stream) : op::launch_q4<op::F16>(a, stream);
  if (streamed(a)) {
    if (bf16) return q4 ? op::launch_few<op::Bf16, op::RowsQ4<op::Bf16>>(a, stream) : op::launch_few<op::Bf16, op::Rows16<op::Bf16>>(a, stream);
    return q4 ? op::launch_few<op::F16, op::RowsQ4<op::F16>>(a, stream) : op::launch_few<op::F16, op::Rows16<op::F16>>(a, stream);
  }
  const uint32_t wide = uint32_t(up_to(a.n_in, 8));
  const bool px = pack_x(a), pw = pack_w(a);
  op::u16* room = static_cast<op::u16*>(workspace);
  if (px) {
    if (int err = pack(a.x, a.x_stride, a.rows, a.n_in, room, stream)) return err;
    a.x = room;
    a.x_stride = wide;
    room += uint64_t(a.rows) * wide;
  }
  if (pw) {
    if (int err = pack(a.w, a.w_stride, a.n_out, a.n_in, room, stream)) return err;
    a.w = room;
    a.w_stride = wide;
  }
  a.n_in = wide;  // (packed rows end in zeros; unpacked ones are whole)
  if (q4) return bf16 ? op::launch_q4_tile<op::Bf16>(a, stream) : op::launch_q4_tile<op::F16>(a, stream);
  // Few wide tiles leave each alone on its CU, waiting for its loads. Wide and small: 1000 rows, 4096 x 4096 (128 wide tiles) 91
  // and 59 us, 256 rows, 4096 x 28672 (224) 129 and 135, 1000 rows, 4096 x 8192 (256) 104 and 126.
  if (uint64_t((a.n_out + op::WideTile::kA - 1) / op::WideTile::kA) * ((a.rows + op::WideTile::kB - 1) / op::WideTile::kB) < 224)
    return bf16 ? op::launch_tile<op::Bf16, op::SmallTile>(a, stream) : op::launch_tile<op::F16, op::SmallTile>(a, stream);
  return bf16 ? op::launch_tile<op::Bf16, op::WideTile>(a, stream) : op::launch_tile<op::F16, op::WideTile>(a, stream);
}

}  // namespace tsa
