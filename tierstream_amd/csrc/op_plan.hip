// Groups the pairs of a call by expert (one workgroup: a call has at most 2^24 pairs, a decode step a few hundred).
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

// Groups the pairs by expert, stably: each wave counts its stretch of pairs per expert, the counts are summed over
// experts and waves, then each wave places its stretch 64 pairs at a time, a pair behind those of its expert in lower
// lanes. `rows_per_tile` sorted positions of one expert make a tile. Bound by its latencies: the ids' (twice where a stretch is
// longer than kBatch), three barriers, a slot's look-up: 256 pairs 5 us, 16384 10 us.
__global__ __launch_bounds__(kPlanThreads) void plan_kernel(ExpertMap m, const int32_t* ids, Plan p, uint32_t rows_per_tile) {
  extern __shared__ uint32_t count[];  // [kPlanWaves][n]
  __shared__ uint32_t totals[kPlanWaves][2];
  const uint32_t t = threadIdx.x, lane = t & 63u, wave = t >> 6, n = m.n;
  const uint32_t stretch = (p.pairs + 64 * kPlanWaves - 1) / (64 * kPlanWaves);  // of 64 pairs, a wave
  const uint32_t from = wave * stretch * 64 + lane;                              // (pairs are below 2^24)
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
  const char* parts[3] = {};
  if (mine) part_pointers(m, t, parts);
  const uint32_t n_tiles = (mine + rows_per_tile - 1) / rows_per_tile;
  uint32_t first = wave_scan(mine), tile = wave_scan(n_tiles);
  if (lane == 63) totals[wave][0] = first, totals[wave][1] = tile;
  __syncthreads();
  first -= mine;
  tile -= n_tiles;
  for (uint32_t w = 0; w < wave; ++w) first += totals[w][0], tile += totals[w][1];
  if (t < n) {
    p.first[t] = first;
    uint32_t at = first;
    for (uint32_t w = 0; w < kPlanWaves; ++w) {
      const uint32_t c = count[w * n + t];
      count[w * n + t] = at;
      at += c;
    }
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
  hipLaunchKernelGGL(op::plan_kernel, dim3(1), dim3(op::kPlanThreads), 4 * op::kPlanWaves * e.n, s, e, ids, p,
                     rows_per_tile);
  return int(hipGetLastError());
}

}  // namespace tsa
