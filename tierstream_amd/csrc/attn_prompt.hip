// Attention over packed sequences: O^T = V^T P^T with S^T = K Q^T, 128 queries of a head a workgroup (32 a wave), keys and values in tiles
// of 64 through LDS, the next one on its way while one is multiplied. A lane's column is its query in scores and outputs alike: the
// softmax runs in the lane's own registers, and its probabilities are the second product's operand as they stand. Four waves of 32
// queries share each tile, and two workgroups a CU fill each other's waits; the longest rows begin first.
// Measured: 8191 tokens of 32 heads on 8 of 128, causal, 511 to 540 us: 1020 to 1080 TFLOP/s (a library's large product reaches 1400); the matrix units
// are busy 57 % of the cycles, at 1.6 GHz. The next tile's scores made in the shadow of this one's exponentials took 4 % longer. 301 tokens of 4 heads: 9.1 us, latency.
#include "attn_tile.hpp"

namespace tsa {
namespace op {
namespace {

template <int kD>
struct PromptMemory {
  __attribute__((aligned(16))) unsigned char tile[2][2][TileShapes<kD>::kBytes];  // keys and values, two of each
  __attribute__((aligned(16))) float mark[kTile];
  OwnTileMemory own;
};

// A workgroup's queries.
template <class T, int kD, bool kAligned, bool kSplit>
__device__ __forceinline__ void attend_tile(const tsa_attend_args& a, float c, uint32_t head, OwnTile own, Span qs, Span ks, PromptMemory<kD>& m) {
  typedef TileShapes<kD> S;
  constexpr float kUp = std::is_same_v<T, F16> ? 7.0f : 0.0f;  // half precision: probabilities up to 2^15, so that small ones keep their bits
  const uint32_t kept = head / (a.q.heads / a.k.heads);
  const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5;
  const uint32_t row0 = own.row0 + wave * kOwn, row = row0 + (lane & 31u);
  const bool on = row < qs.count;
  // keys that a row attends to, those that every row of the workgroup does, any row of this wave, and any of the workgroup
  const int32_t ahead = a.causal ? int32_t(ks.count) - int32_t(qs.count) + 1 : 0;
  auto keys_of = [&](uint32_t r) {
    const int32_t n = a.causal ? int32_t(r) + ahead : int32_t(ks.count);
    return n < 0 ? 0u : min(uint32_t(n), ks.count);
  };
  const uint32_t limit = on ? keys_of(row) : 0, all_rows = keys_of(own.row0), any = row0 < qs.count ? keys_of(min(row0 + kOwn, qs.count) - 1) : 0;
  const uint32_t end = keys_of(min(own.row0 + kTileOwn, qs.count) - 1);

  // a negative scale turns the queries' signs, a scale of 0 takes them away
  const OwnRows<kD, kAligned> raw(a.q, uint64_t(qs.begin) + row, head, a.head_dim, on);
  bits8 q[kD / 16];
#pragma unroll
  for (uint32_t k = 0; k < kD / 16; ++k) q[k] = c == 0.0f ? bits8{0, 0, 0, 0, 0, 0, 0, 0} : raw.v[k] ^ u16(c < 0.0f ? 0x8000 : 0);
  c = c == 0.0f ? 1.0f : fabsf(c);

  const TileReads<kD> reads;
  const TileLoads<kD, kAligned> keys(a.k, ks.begin, kept, a.head_dim), values(a.v, ks.begin, kept, a.head_dim);
  const uint32_t lds = __builtin_amdgcn_readfirstlane(lds_offset(m.tile));
  f32x16 o[kD / 32];
  clear(o);
  float top = -INFINITY, total = 0.0f;
  if (end) {
    keys.fetch(0, ks.count, lds);
    values.fetch(0, ks.count, lds + S::kBytes);
  }
  for (uint32_t key0 = 0, buffer = 0; key0 < end; key0 += kTile, buffer ^= 1) {
    tile_ready();
    const uint32_t k_at = lds + buffer * 2 * S::kBytes, v_at = k_at + S::kBytes, other = lds + (buffer ^ 1) * 2 * S::kBytes;
    if (key0 + kTile < end) {
      keys.fetch(key0 + kTile, ks.count, other);
      values.fetch(key0 + kTile, ks.count, other + S::kBytes);
    }
    if (a.causal && key0 + kTile > all_rows) {
      mark_rows(clean_tile<T, kD>(v_at), m.mark);
      clean_done();
    }
    if (key0 >= any) continue;

    const auto k_rows = reads.rows(k_at);
    f32x16 s[2];
    clear(s);
#pragma unroll
    for (uint32_t k = 0; k < kD / 16; ++k)
#pragma unroll
      for (uint32_t r = 0; r < 2; ++r) s[r] = mfma32<T>(k_rows(r, k), q[k], s[r]);
    products_behind_reads<kD / 8, 4>();
    if (key0 + kTile > all_rows) {  // (by every wave that reads a cleaned tile, whether or not the mask cuts its own rows)
      if (a.causal) {
#pragma unroll
        for (uint32_t r = 0; r < 2; ++r)
#pragma unroll
          for (uint32_t i = 0; i < 4; ++i) {
            const f32x4 mark = marks_of(m.mark, r, i);
#pragma unroll
            for (uint32_t k = 0; k < 4; ++k) s[r][4 * i + k] += mark[k];
          }
      }
      const int32_t left = int32_t(limit) - int32_t(key0 + 4 * h);
#pragma unroll
      for (uint32_t r = 0; r < 2; ++r)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (int32_t(32 * r + 8 * (i / 4) + i % 4) >= left) s[r][i] = -INFINITY;
    }

    const auto v_columns = reads.columns(v_at);
    bits8 v0[kD / 32];
#pragma unroll
    for (uint32_t t = 0; t < kD / 32; ++t) v0[t] = v_columns(t, 0);
    __builtin_amdgcn_sched_barrier(0);
    // the running maximum: followed where it is passed by 2^8
    float most = -INFINITY;
#pragma unroll
    for (uint32_t r = 0; r < 2; ++r)
#pragma unroll
      for (int i = 0; i < 16; ++i) most = fmaxf(most, s[r][i]);
    most = fmaxf(most, __shfl_xor(most, 32, 64)) * c;
    if (__any(most > top + 8.0f)) {
      const float up = fmaxf(most, top), keep = top == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(top - up);
      top = up;
      total *= keep;
#pragma unroll
      for (int t = 0; t < kD / 32; ++t) o[t] *= keep;
    }
    const float base = top == -INFINITY ? 0.0f : kUp - top;
#pragma unroll
    for (uint32_t r = 0; r < 2; ++r)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        s[r][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r][i], c, base));
        total += s[r][i];
      }
#pragma unroll
    for (uint32_t u = 0; u < 4; ++u) {
      const Second<T, kSplit> p(s[u / 2], u % 2);
#pragma unroll
      for (uint32_t t = 0; t < kD / 32; ++t) p.add(u ? v_columns(t, u) : v0[t], o[t]);
    }
  }
  if (!on) return;
  total += __shfl_xor(total, 32, 64);
  put_columns<T, kD, kAligned>(a.out, uint64_t(qs.begin) + row, head, a.head_dim, o, total == 0.0f ? 0.0f : 1.0f / total);
  if (a.lse && h == 0)
    a.lse[uint64_t(head) * a.tokens + qs.begin + row] = total == 0.0f ? -INFINITY : (top - kUp + __builtin_amdgcn_logf(total)) * 0.69314718f;
}

template <class T, int kD, bool kAligned>
__global__ __launch_bounds__(64 * kTileWaves, 2) void attend_kernel(tsa_attend_args a, float c) {
  __shared__ PromptMemory<kD> m;
  OwnTile own;
  if (!find_own_tile<true>(a.first, a.sequences, a.tokens, blockIdx.x / a.q.heads, m.own, own)) return;
  const uint32_t head = head_of_group(blockIdx.x % a.q.heads, a.q.heads);
  const Span qs = span_of(a.first, own.sequence, a.tokens), ks = span_of(a.k_first ? a.k_first : a.first, own.sequence, a.k_tokens);
  if (both_parts(qs.count, ks.count)) attend_tile<T, kD, kAligned, true>(a, c, head, own, qs, ks, m);
  else attend_tile<T, kD, kAligned, false>(a, c, head, own, qs, ks, m);
}

}  // namespace
}  // namespace op

int launch_attend(const tsa_attend_args& a, hipStream_t stream) {
  using namespace op;
  const dim3 grid(uint32_t(own_tiles_at_most(a.sequences, a.tokens) * a.q.heads)), block(64 * kTileWaves);
  const float c = a.scale * 1.44269504f;
  const bool aligned = vector_heads(a.q) && vector_heads(a.out) && (a.k_tokens == 0 || (tile_heads(a.k) && tile_heads(a.v)));
#define CALL(T, D)                                                                                      \
  do {                                                                                                  \
    if (aligned) hipLaunchKernelGGL((attend_kernel<T, D, true>), grid, block, 0, stream, a, c);         \
    else hipLaunchKernelGGL((attend_kernel<T, D, false>), grid, block, 0, stream, a, c);                \
  } while (0)
  if (a.type == TSA_BF16) {
    if (a.head_dim <= 64) CALL(Bf16, 64);
    else CALL(Bf16, 128);
  } else {
    if (a.head_dim <= 64) CALL(F16, 64);
    else CALL(F16, 128);
  }
#undef CALL
  return int(hipGetLastError());
}

}  // namespace tsa
