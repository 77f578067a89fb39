// Groups the pairs of a call by expert (one workgroup: a call has at most 2^24 pairs, a decode step a few hundred).
#include "op_pairs.hpp"

namespace tsa {
namespace op {
namespace {

constexpr uint32_t kPlanThreads = 1024, kPlanWaves = kPlanThreads / 64;

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

}  // namespace
}  // namespace op

int launch_plan(const ExpertMap& e, const int32_t* ids, const Plan& p, uint32_t rows_per_tile, hipStream_t s) {
  hipLaunchKernelGGL(op::plan_kernel, dim3(1), dim3(op::kPlanThreads), 4 * (op::kPlanThreads + op::kPlanWaves * e.n), s, e, ids, p,
                     rows_per_tile);
  return int(hipGetLastError());
}

}  // namespace tsa
