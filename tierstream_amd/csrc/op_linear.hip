// y = act(x W^T + bias) + residual.
#include "op_device.hpp"

namespace tsa {
namespace op {
namespace {

__device__ __forceinline__ void finish_linear(const tsa_linear_args& a, uint32_t row, uint32_t n, float v) {
  if (a.bias) v += load_as_float(a.bias, n, a.x_type);
  v = activate(a.act, v);
  if (a.residual) v += load_as_float(a.residual, uint64_t(row) * a.residual_stride + n, a.y_type);
  store_float(a.y, uint64_t(row) * a.y_stride + n, a.y_type, v);
}

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

}  // namespace
}  // namespace op

uint64_t linear_workspace(const tsa_linear_args&) { return 0; }

int launch_linear(const tsa_linear_args& a, void*, hipStream_t stream) {
  if (a.rows == 0 || a.n_out == 0) return 0;
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
