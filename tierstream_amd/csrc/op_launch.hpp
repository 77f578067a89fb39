// The model operators' launches (tsa_ops.h): what the C entry points check and choose on the host, and what the kernels
// take by value. Every launch_* returns a hipError_t as an int; none synchronizes or allocates.
#pragma once

#include <hip/hip_runtime_api.h>
#include <stdint.h>

extern "C" {
#include "tierstream_amd/tsa_ops.h"
}

namespace tsa {

constexpr uint32_t kQ4Block = 32, kQ4Bytes = 18;  // values per 4-bit block, its bytes

constexpr uint64_t weight_row_bytes(uint64_t n, uint32_t type) {
  return type == TSA_Q4 ? n / kQ4Block * kQ4Bytes : 2 * n;
}
inline uint64_t up_to(uint64_t v, uint64_t a) { return (v + a - 1) / a * a; }

// Experts' weights as the kernels take them: one of the three forms.
struct ExpertMap {
  const char* part[3] = {};
  uint64_t stride[3] = {};  // stacked: bytes from expert to expert; table: offsets of the parts in a unit
  const uint64_t* table = nullptr;
  ss_dg_device_view view = {};
  uint32_t gated = 0, n = 0;
  uint32_t form = 0;  // 0 stacked, 1 table, 2 device-gated view
};

// The pairs (row, j) of a call, p = row x top_k + j, grouped by expert: in the workspace, written by the plan kernel.
struct Plan {
  const char** part = nullptr;     // [n][3]: the experts' weights (only those with pairs)
  uint32_t* first = nullptr;       // [n + 1]: an expert's first sorted position
  uint32_t* pair = nullptr;        // [pairs]: sorted position -> pair (ascending inside an expert)
  uint32_t* row = nullptr;         // [pairs]: sorted position -> row
  int32_t* at = nullptr;           // [pairs]: pair -> sorted position, -1 where the id adds nothing
  uint32_t* tile = nullptr;        // [tiles][2]: expert, first sorted position
  uint32_t* n_tiles = nullptr;
  uint32_t* counts = nullptr;      // [groups][n]: an expert's pairs in each workgroup's stretch of pairs
  uint32_t pairs = 0, top_k = 1, n = 0, groups = 1, stretch = 0;
};

int launch_route(const tsa_route_args& a, hipStream_t stream);
int launch_route_backward(const tsa_route_args& a, const float* dweights, void* dlogits, uint64_t stride,
                          hipStream_t stream);

uint64_t linear_workspace(const tsa_linear_args& a);
int launch_linear(const tsa_linear_args& a, void* workspace, hipStream_t stream);

uint64_t ffn_workspace(uint32_t n, uint32_t d, uint32_t f, uint32_t w_type, uint32_t rows, uint32_t top_k);
int launch_ffn(const ExpertMap& e, uint32_t d, uint32_t f, uint32_t w_type, const tsa_ffn_args& a, void* workspace,
               hipStream_t stream);
uint64_t ffn_backward_workspace(uint32_t n, uint32_t d, uint32_t f, uint32_t w_type, uint32_t rows, uint32_t top_k);
int launch_ffn_backward(const ExpertMap& e, uint32_t d, uint32_t f, const tsa_ffn_grad_args& a, void* workspace,
                        hipStream_t stream);

}  // namespace tsa
