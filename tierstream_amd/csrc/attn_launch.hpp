// The attention operators' launches (tsa_attn.h). Every launch_* returns a hipError_t as an int; none synchronizes or allocates.
#pragma once

#include <hip/hip_runtime_api.h>
#include <stdint.h>

extern "C" {
#include "tierstream_amd/tsa_attn.h"
}

namespace tsa {

constexpr uint32_t kPage = TSA_CACHE_PAGE;

int launch_rotate(const tsa_rotary& r, const tsa_rotate_args& a, hipStream_t stream);

int launch_cache_plan(const tsa_cache_plan_args& a, hipStream_t stream);
int launch_cache_slots(const tsa_cache_plan_args& a, hipStream_t stream);
int launch_cache_store(const tsa_cache& c, const tsa_cache_rows_args& a, hipStream_t stream);
int launch_cache_load(const tsa_cache& c, const tsa_cache_rows_args& a, hipStream_t stream);

uint64_t attend_cached_workspace(const tsa_cache& c, const tsa_attend_cached_args& a);
int launch_attend_cached(const tsa_cache& c, const tsa_attend_cached_args& a, void* workspace, hipStream_t stream);

int launch_attend(const tsa_attend_args& a, hipStream_t stream);
uint64_t attend_backward_workspace(const tsa_attend_args& f);
int launch_attend_backward(const tsa_attend_grad_args& a, void* workspace, hipStream_t stream);

}  // namespace tsa
