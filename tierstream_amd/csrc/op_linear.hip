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

template <class T, bool kQ4>
__global__ __launch_bounds__(256) void linear_any_kernel(tsa_linear_args a) {
  __shared__ TileMemory m;
  const uint32_t tn = (a.n_out + 63) / 64;
  const uint64_t tiles = uint64_t(tn) * ((uint64_t(a.rows) + 63) / 64);
  const Operand x{static_cast<const u16*>(a.x), a.x_stride, 1, a.rows, a.n_in, nullptr};
  for (uint64_t tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    const uint32_t n0 = uint32_t(tile % tn) * 64, r0 = uint32_t(tile / tn) * 64;
    f32x4 acc[2][2] = {};
    if constexpr (kQ4) {
      const Q4Operand<T> w{static_cast<const unsigned char*>(a.w), weight_row_bytes(a.n_in, TSA_Q4), a.n_out, a.n_in};
      tile64<T, true>(w, n0, x, r0, a.n_in, m, acc);
    } else {
      const Operand w{static_cast<const u16*>(a.w), a.w_stride, 1, a.n_out, a.n_in, nullptr};
      tile64<T, false>(w, n0, x, r0, a.n_in, m, acc);
    }
    each64(acc, [&](uint32_t i, uint32_t j, float v) {
      if (n0 + i < a.n_out && r0 + j < a.rows) finish_linear(a, r0 + j, n0 + i, v);
    });
  }
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
  if (a.rows <= 16) return launch_few<T, W, 1, 1>(a, stream);
  if (a.rows <= 32) return launch_few<T, W, 2, 2>(a, stream);
  return launch_few<T, W, 2, 4>(a, stream);
}

// Many rows: tiles of 256 weight rows and 128 rows of x, two workgroups a CU: one's products run under the other's epilogue.
// (Tiles of 256 x 256, one a CU, take less from L2 and LDS, but their epilogue stands alone: 575 us where these take 528,
// 2047 rows through 4096 x 28672 with bias, tanh gelu and residual.)
template <class T>
__global__ __launch_bounds__(kTileThreads, 2) void linear_tile_kernel(tsa_linear_args a) {
  extern __shared__ f32x4 memory[];
  const uint32_t wave = threadIdx.x >> 6;
  const TileAt t = tile_at(blockIdx.x, (a.n_out + 255) / 256, (a.rows + 127) / 128);
  const uint32_t n0 = t.a * 256, r0 = t.b * 128;
  TileRowsSource<8> w(a.n_in, wave & 1u, [&](uint32_t r) {
    const uint32_t n = n0 + r;
    return static_cast<const u16*>(a.w) + (n < a.n_out ? n : a.n_out - 1) * a.w_stride;
  });
  TileRowsSource<4> x(a.n_in, wave >> 1, [&](uint32_t r) {
    const uint32_t row = r0 + r;
    return static_cast<const u16*>(a.x) + (row < a.rows ? row : a.rows - 1) * a.x_stride;
  });
  f32x4 acc[8][4] = {};
  tile_product<T, 8, 4, 3>(w, x, a.n_in, lds_offset(memory), acc);
  LinearOut<T> out(a, r0, n0);
  hand_out<8, 4, 2>(memory, acc, out);
}

template <class T>
int launch_tile(const tsa_linear_args& a, hipStream_t stream) {
  const uint32_t tiles = (a.n_out + 255) / 256 * ((a.rows + 127) / 128);
  hipLaunchKernelGGL((linear_tile_kernel<T>), dim3(tiles), dim3(kTileThreads), tile_lds(8, 4, 3), stream, a);
  return int(hipGetLastError());
}

bool aligned16(const void* p, uint64_t stride) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride % 8 == 0; }

}  // namespace
}  // namespace op

uint64_t linear_workspace(const tsa_linear_args&) { return 0; }

int launch_linear(const tsa_linear_args& a, void*, hipStream_t stream) {
  if (a.rows == 0 || a.n_out == 0) return 0;
  const bool wide = a.n_in % 8 == 0 && op::aligned16(a.x, a.x_stride) && (a.w_type == TSA_Q4 || op::aligned16(a.w, a.w_stride));
  if (wide && a.rows == 1 && a.w_type == TSA_Q4 && a.n_in % 256 == 0 && op::aligned16(a.w, 0))
    return a.x_type == TSA_BF16 ? op::launch_q4<op::Bf16>(a, stream) : op::launch_q4<op::F16>(a, stream);
  if (wide && a.rows <= 64) {
    if (a.x_type == TSA_BF16)
      return a.w_type == TSA_Q4 ? op::launch_few<op::Bf16, op::RowsQ4<op::Bf16>>(a, stream)
                                : op::launch_few<op::Bf16, op::Rows16<op::Bf16>>(a, stream);
    return a.w_type == TSA_Q4 ? op::launch_few<op::F16, op::RowsQ4<op::F16>>(a, stream)
                              : op::launch_few<op::F16, op::Rows16<op::F16>>(a, stream);
  }
  if (wide && a.w_type != TSA_Q4 && a.rows < (1u << 24) && a.n_out < (1u << 24)) {
    return a.x_type == TSA_BF16 ? op::launch_tile<op::Bf16>(a, stream) : op::launch_tile<op::F16>(a, stream);
  }
  const uint64_t tiles = (uint64_t(a.n_out) + 63) / 64 * ((uint64_t(a.rows) + 63) / 64);
  const dim3 grid(uint32_t(tiles < (1u << 20) ? tiles : (1u << 20)));
#define CALL(T, Q) hipLaunchKernelGGL((op::linear_any_kernel<op::T, Q>), grid, dim3(256), 0, stream, a)
  if (a.x_type == TSA_BF16) {
    if (a.w_type == TSA_Q4) CALL(Bf16, true);
    else CALL(Bf16, false);
  } else {
    if (a.w_type == TSA_Q4) CALL(F16, true);
    else CALL(F16, false);
  }
#undef CALL
  return int(hipGetLastError());
}

}  // namespace tsa
