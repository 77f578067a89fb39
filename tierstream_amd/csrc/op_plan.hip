// Groups the pairs of a call by expert.
#include "op_pairs.hpp"

namespace tsa {
namespace op {
namespace {

constexpr uint32_t kPlanThreads = 1024, kPlanWaves = kPlanThreads / 64;

constexpr int kBatch = 4;  // ids of so many times 64 pairs are loaded at once

// Inclusive sum over a wave's lanes.
__device__ __forceinline__ uint32_t wave_scan(uint32_t v) {
  const uint32_t lane = threadIdx.x & 63u;
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) {
    const uint32_t o = __shfl_up(v, s, 64);
    if (lane >= uint32_t(s)) v += o;
  }
  return v;
}

// Pairs of each expert in one workgroup's stretch of pairs, for the kernel below.
__global__ __launch_bounds__(kPlanThreads) void count_kernel(ExpertMap m, const int32_t* ids, Plan p) {
  extern __shared__ uint32_t count[];  // [n]
  for (uint32_t i = threadIdx.x; i < m.n; i += kPlanThreads) count[i] = 0;
  __syncthreads();
  const uint32_t from = blockIdx.x * p.stretch, to = p.pairs - from < p.stretch ? p.pairs : from + p.stretch;
  for (uint32_t pair = from + threadIdx.x; pair < to; pair += kPlanThreads) {
    const uint32_t e = expert_of(m, ids, pair);
    if (e != ~0u) atomicAdd(&count[e], 1u);
  }
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < m.n; i += kPlanThreads) p.counts[blockIdx.x * m.n + i] = count[i];
}

// Groups the pairs by expert, stably: each wave counts its stretch of pairs per expert, the counts are summed over
// experts and waves, then each wave places its stretch 64 pairs at a time, a pair behind those of its expert in lower
// lanes. `rows_per_tile` sorted positions of one expert make a tile. A few hundred pairs: bound by its latencies (the ids', three
// barriers, a slot's look-up), 5 us. Many: by the instructions and scattered stores of a CU, so above kPlanOne pairs
// every kPlanOne of them have a workgroup, which counts on those in front of it in p.counts and writes the places of
// its own pairs, the first one also the experts' and the tiles' (16384 pairs: 13 us for both kernels, one workgroup 31).
__global__ __launch_bounds__(kPlanThreads) void plan_kernel(ExpertMap m, const int32_t* ids, Plan p, uint32_t rows_per_tile) {
  extern __shared__ uint32_t count[];  // [kPlanWaves][n]
  __shared__ uint32_t totals[kPlanWaves][2];
  const uint32_t t = threadIdx.x, lane = t & 63u, wave = t >> 6, n = m.n;
  const uint32_t stretch = (p.stretch + 64 * kPlanWaves - 1) / (64 * kPlanWaves);  // of 64 pairs, a wave
  const uint32_t from = blockIdx.x * p.stretch + wave * stretch * 64 + lane;       // (pairs are below 2^24)
  uint32_t e[kBatch];
  const auto load = [&](uint32_t i) {
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const uint32_t pair = from + (i + b) * 64;
      e[b] = i + b < stretch && pair < p.pairs ? expert_of(m, ids, pair) : ~0u;
    }
  };
  load(0);
  for (uint32_t i = t; i < kPlanWaves * n; i += kPlanThreads) count[i] = 0;
  __syncthreads();
  for (uint32_t i = 0; i < stretch; i += kBatch) {
    if (i) load(i);
#pragma unroll
    for (int b = 0; b < kBatch; ++b)
      if (e[b] != ~0u) atomicAdd(&count[wave * n + e[b]], 1u);
  }
  __syncthreads();
  uint32_t mine = 0;
  if (t < n)
    for (uint32_t w = 0; w < kPlanWaves; ++w) mine += count[w * n + t];
  uint32_t before = 0;  // of the workgroups in front
  if (p.groups > 1 && t < n) {
    mine = 0;
#pragma unroll 8
    for (uint32_t g = 0; g < p.groups; ++g) {
      const uint32_t c = p.counts[g * n + t];
      before += g < blockIdx.x ? c : 0;
      mine += c;
    }
  }
  const char* parts[3] = {};
  if (mine && blockIdx.x == 0) part_pointers(m, t, parts);
  const uint32_t n_tiles = (mine + rows_per_tile - 1) / rows_per_tile;
  uint32_t first = wave_scan(mine), tile = wave_scan(n_tiles);
  if (lane == 63) totals[wave][0] = first, totals[wave][1] = tile;
  __syncthreads();
  first -= mine;
  tile -= n_tiles;
  for (uint32_t w = 0; w < wave; ++w) first += totals[w][0], tile += totals[w][1];
  if (t < n) {
    uint32_t at = first + before;
    for (uint32_t w = 0; w < kPlanWaves; ++w) {
      const uint32_t c = count[w * n + t];
      count[w * n + t] = at;
      at += c;
    }
  }
  if (t < n && blockIdx.x == 0) {
    p.first[t] = first;
    for (uint32_t i = 0; i < n_tiles; ++i) {
      p.tile[2 * (tile + i)] = t;
      p.tile[2 * (tile + i) + 1] = first + i * rows_per_tile;
    }
    if (t == n - 1) {
      p.first[n] = first + mine;
      *p.n_tiles = tile + n_tiles;
    }
    if (mine)
      for (int i = 0; i < 3; ++i) p.part[3 * t + i] = parts[i];
  }
  __syncthreads();
  if (stretch > kBatch) load(0);
  for (uint32_t i = 0; i < stretch; i += kBatch) {
    if (i) load(i);
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const uint32_t pair = from + (i + b) * 64;
      if (i + b >= stretch || pair - lane >= p.pairs) break;
      uint64_t same = __ballot(e[b] != ~0u);
      for (uint32_t bit = 0; bit < 9; ++bit) {  // (n <= 512)
        const uint64_t set = __ballot((e[b] >> bit) & 1u);
        same &= (e[b] >> bit) & 1u ? set : ~set;
      }
      uint32_t at = 0;
      if (e[b] != ~0u) {
        at = __hip_atomic_load(&count[wave * n + e[b]], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP) +
             uint32_t(__popcll(same & ((1ull << lane) - 1)));
        p.pair[at] = pair;
        p.row[at] = pair / p.top_k;
      }
      __builtin_amdgcn_wave_barrier();
      if (e[b] != ~0u && (same >> lane) == 1)  // the last lane of its expert
        __hip_atomic_store(&count[wave * n + e[b]], at + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
      __builtin_amdgcn_wave_barrier();
      if (pair < p.pairs) p.at[pair] = e[b] != ~0u ? int32_t(at) : -1;
    }
  }
}

}  // namespace
}  // namespace op

int launch_plan(const ExpertMap& e, const int32_t* ids, const Plan& p, uint32_t rows_per_tile, hipStream_t s) {
  if (p.groups > 1) hipLaunchKernelGGL(op::count_kernel, dim3(p.groups), dim3(op::kPlanThreads), 4 * e.n, s, e, ids, p);
  hipLaunchKernelGGL(op::plan_kernel, dim3(p.groups), dim3(op::kPlanThreads), 4 * op::kPlanWaves * e.n, s, e, ids, p, rows_per_tile);
  return int(hipGetLastError());
}

}  // namespace tsa
