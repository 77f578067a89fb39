// The gradients of attention over packed sequences. With p = exp(score - lse), dp = dout . v and ds = p (dp - dout . out):
//   dq = scale ds K    a workgroup has 128 queries of a head and runs over the keys,
//   dk = scale ds^T Q, dv = p^T dout    a workgroup has 128 keys of a kept head and runs over the queries of its group's heads,
// each in tiles of 64 through LDS as in the forward pass: the wave's own rows are the columns of every product, and p and ds, as they
// come out of the first products, the operand of the second. Scores are computed twice, and nothing is added up across
// workgroups: the same bits every time, without atomics or partial sums in memory. lse and dout . out go to the workspace first, a pair a row.
#include "attn_tile.hpp"

namespace tsa {
namespace op {
namespace {

// (lse / ln 2, dout . out) of each row; a row without keys has an lse of infinity, which makes its probabilities 0.
template <class T, bool kAligned>
__global__ __launch_bounds__(256) void rows_kernel(tsa_attend_grad_args g, float2* rows) {
  const tsa_attend_args& a = g.f;
  const uint32_t head = blockIdx.x % a.q.heads, t = blockIdx.x / a.q.heads * 16 + threadIdx.x / 16, value = (threadIdx.x & 15u) * 8;
  if (t >= a.tokens) return;
  float sum = 0.0f;
  if (value < a.head_dim) {
    const u16 *x = row_of<u16>(a.out, t, head) + value, *y = row_of<u16>(g.dout, t, head) + value;
    if constexpr (kAligned) {
      const bits8 u = *reinterpret_cast<const bits8*>(x), v = *reinterpret_cast<const bits8*>(y);
#pragma unroll
      for (int i = 0; i < 8; ++i) sum += T::up(u[i]) * T::up(v[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) sum += T::up(x[i]) * T::up(y[i]);
    }
  }
#pragma unroll
  for (int s = 1; s < 16; s <<= 1) sum += __shfl_xor(sum, s, 64);
  if (value == 0) {
    const uint64_t at = uint64_t(head) * a.tokens + t;
    const float lse = a.lse[at];
    rows[at] = {lse == -INFINITY ? INFINITY : lse * 1.44269504f, sum};
  }
}

// Gradients of scores on their way to 16 bits. bf16 has the range of 32 bits. Half precision has not: a column's are multiplied by
// a power of two that keeps the largest so far below 2^15 and starts it at 2^8, and what was summed before follows when that changes.
template <class T>
struct Raised {
  float by = 1.0f;
  template <int N>
  __device__ __forceinline__ void raise(const f32x16&, f32x16 (&)[N]) {}
  __device__ __forceinline__ float down() const { return 1.0f; }
};
template <>
struct Raised<F16> {
  float by = 0.0f;
  template <int N>
  __device__ __forceinline__ void raise(const f32x16& v, f32x16 (&sum)[N]) {
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) top = peak(top, v[i]);
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    if (__any(top * by > 32768.0f || (by == 0.0f && top > 0.0f))) {
      const bool on = top * by > 32768.0f || (by == 0.0f && top > 0.0f);
      const int e = 8 - (int(__builtin_bit_cast(uint32_t, top) >> 23) - 127), in = e > 126 ? 126 : e < -126 ? -126 : e;
      const float next = __builtin_bit_cast(float, uint32_t(127 + in) << 23), keep = !on ? 1.0f : by == 0.0f ? 0.0f : next / by;
      if (on) by = next;
#pragma unroll
      for (int t = 0; t < N; ++t) sum[t] *= keep;
    }
  }
  __device__ __forceinline__ float down() const { return by == 0.0f ? 0.0f : 1.0f / by; }
};

template <int N>
__device__ __forceinline__ void clear(f32x16 (&v)[N]) {
#pragma unroll
  for (int t = 0; t < N; ++t)
#pragma unroll
    for (int i = 0; i < 16; ++i) v[t][i] = 0.0f;
}

template <class T, int kD, bool kAligned>
__global__ __launch_bounds__(64 * kTileWaves, 2) void queries_kernel(tsa_attend_grad_args g, const float2* rows, float c) {
  typedef TileShapes<kD> S;
  __shared__ __attribute__((aligned(16))) unsigned char tile_s[2][2][S::kBytes];  // keys and values, two of each
  __shared__ __attribute__((aligned(16))) float mark_s[kTile];
  __shared__ OwnTileMemory own_s;
  const tsa_attend_args& a = g.f;
  OwnTile own;
  const uint32_t head = head_of_group(blockIdx.x % a.q.heads, a.q.heads), kept = head / (a.q.heads / a.k.heads);
  if (!find_own_tile<true>(a.first, a.sequences, a.tokens, blockIdx.x / a.q.heads, own_s, own)) return;
  const Span qs = span_of(a.first, own.sequence, a.tokens), ks = span_of(a.k_first ? a.k_first : a.first, own.sequence, a.k_tokens);
  const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5;
  const uint32_t row0 = own.row0 + wave * kOwn, row = row0 + (lane & 31u);
  const bool on = row < qs.count;
  const int32_t ahead = a.causal ? int32_t(ks.count) - int32_t(qs.count) + 1 : 0;
  auto keys_of = [&](uint32_t r) {  // keys that a query attends to
    const int32_t n = a.causal ? int32_t(r) + ahead : int32_t(ks.count);
    return n < 0 ? 0u : min(uint32_t(n), ks.count);
  };
  const uint32_t limit = on ? keys_of(row) : 0, all_rows = keys_of(own.row0), whole = keys_of(row0), any = row0 < qs.count ? keys_of(min(row0 + kOwn, qs.count) - 1) : 0;
  const uint32_t end = keys_of(min(own.row0 + kTileOwn, qs.count) - 1);

  const OwnRows<kD, kAligned> q(a.q, uint64_t(qs.begin) + row, head, a.head_dim, on), dout(g.dout, uint64_t(qs.begin) + row, head, a.head_dim, on);
  const float2 mine = on ? rows[uint64_t(head) * a.tokens + qs.begin + row] : float2{INFINITY, 0.0f};
  const TileReads<kD> reads;
  const TileLoads<kD, kAligned> keys(a.k, ks.begin, kept, a.head_dim), values(a.v, ks.begin, kept, a.head_dim);
  const uint32_t lds = __builtin_amdgcn_readfirstlane(lds_offset(tile_s));
  f32x16 dq[kD / 32];
  clear(dq);
  Raised<T> raised;

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
      mark_rows(clean_tile<T, kD>(k_at), mark_s);
      clean_done();
    }
    if (key0 >= any) continue;
#pragma unroll
    for (uint32_t r = 0; r < 2; ++r) {
      f32x16 one[2];  // scores, then their gradients; gradients of probabilities
      clear(one);
#pragma unroll
      for (uint32_t k = 0; k < kD / 16; ++k) {
        one[0] = mfma32<T>(reads.rows(k_at, r, k), q.v[k], one[0]);
        one[1] = mfma32<T>(reads.rows(v_at, r, k), dout.v[k], one[1]);
      }
#pragma unroll
      for (int i = 0; i < 16; ++i)
        one[0][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(one[0][i], c, -mine.x)) * (one[1][i] - mine.y);
      if (key0 + kTile > whole) {
        if (a.causal) {
#pragma unroll
          for (uint32_t i = 0; i < 4; ++i) {
            const f32x4 mark = marks_of(mark_s, r, i);
#pragma unroll
            for (uint32_t k = 0; k < 4; ++k) one[0][4 * i + k] += mark[k];
          }
        }
        const int32_t left = int32_t(limit) - int32_t(key0 + 4 * h);
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (int32_t(32 * r + 8 * (i / 4) + i % 4) >= left) one[0][i] = 0.0f;
      }
      raised.raise(one[0], dq);
      if constexpr (std::is_same_v<T, F16>) one[0] *= raised.by;
#pragma unroll
      for (uint32_t u = 0; u < 2; ++u) {
        const bits8 ds = pack8<T>(one[0], u);
#pragma unroll
        for (uint32_t t = 0; t < kD / 32; ++t) dq[t] = mfma32<T>(reads.columns(k_at, t, 2 * r + u), ds, dq[t]);
      }
    }
  }
  if (on) put_columns<T, kD, kAligned>(g.dq, uint64_t(qs.begin) + row, head, a.head_dim, dq, a.scale * raised.down());
}

template <class T, int kD, bool kAligned>
__global__ __launch_bounds__(64 * kTileWaves, kD == 64 ? 2 : 1) void keys_kernel(tsa_attend_grad_args g, const float2* rows, float c) {
  typedef TileShapes<kD> S;
  constexpr float kUp = std::is_same_v<T, F16> ? 14.0f : 0.0f;  // half precision: probabilities up to 2^14
  __shared__ __attribute__((aligned(16))) unsigned char tile_s[2][2][S::kBytes];  // queries and the outputs' gradients, two of each
  __shared__ __attribute__((aligned(16))) float2 row_s[2][kTile];
  __shared__ __attribute__((aligned(16))) float mark_s[kTile];
  __shared__ OwnTileMemory own_s;
  const tsa_attend_args& a = g.f;
  const int32_t* k_first = a.k_first ? a.k_first : a.first;
  OwnTile own;
  const uint32_t kept = head_of_group(blockIdx.x % a.k.heads, a.k.heads), group = a.q.heads / a.k.heads;
  if (!find_own_tile<false>(k_first, a.sequences, a.k_tokens, blockIdx.x / a.k.heads, own_s, own)) return;
  const Span qs = span_of(a.first, own.sequence, a.tokens), ks = span_of(k_first, own.sequence, a.k_tokens);
  const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5;
  const uint32_t row0 = own.row0 + wave * kOwn, row = row0 + (lane & 31u);
  const bool on = row < ks.count;
  // the first query that attends to a key
  auto from_of = [&](uint32_t key) {
    const int32_t n = a.causal ? int32_t(key) - int32_t(ks.count) + int32_t(qs.count) : 0;
    return n < 0 ? 0u : uint32_t(n);
  };
  const uint32_t from = from_of(row), any = from_of(row0), whole = from_of(row0 + kOwn - 1), all_rows = from_of(own.row0 + kTileOwn - 1);
  const uint32_t begin = from_of(own.row0) / kTile * kTile, tiles = begin < qs.count ? (qs.count - begin + kTile - 1) / kTile : 0, steps = tiles * group;

  const OwnRows<kD, kAligned> k(a.k, uint64_t(ks.begin) + row, kept, a.head_dim, on), v(a.v, uint64_t(ks.begin) + row, kept, a.head_dim, on);
  const TileReads<kD> reads;
  const uint32_t lds = __builtin_amdgcn_readfirstlane(lds_offset(tile_s)), row_lds = __builtin_amdgcn_readfirstlane(lds_offset(row_s));
  f32x16 dk[kD / 32], dv[kD / 32];
  clear(dk);
  clear(dv);
  Raised<T> raised;

  uint32_t head = kept * group, q0 = begin;  // of the step whose loads go next
  auto fetch = [&](uint32_t buffer) {
    const TileLoads<kD, kAligned> queries(a.q, qs.begin, head, a.head_dim), douts(g.dout, qs.begin, head, a.head_dim);
    queries.fetch(q0, qs.count, lds + buffer * 2 * S::kBytes);
    douts.fetch(q0, qs.count, lds + (buffer * 2 + 1) * S::kBytes);
    if (wave < 2) {  // 32 rows' pairs, word by word
      const uint32_t r = q0 + wave * 32 + lane / 2;
      const float2* at = rows + uint64_t(head) * a.tokens + qs.begin + min(r, qs.count - 1);
      load_words_to_lds(reinterpret_cast<const float*>(at) + (lane & 1u), row_lds + buffer * kTile * 8 + wave * 256);
    }
    q0 += kTile;
    if (q0 >= qs.count) q0 = begin, ++head;
  };
  if (steps) fetch(0);
  for (uint32_t step = 0, buffer = 0, row_at = begin; step < steps; ++step, buffer ^= 1) {
    tile_ready();
    const uint32_t q_at = lds + buffer * 2 * S::kBytes, d_at = q_at + S::kBytes, at = row_at;
    if (step + 1 < steps) fetch(buffer ^ 1);
    row_at = at + kTile >= qs.count ? begin : at + kTile;
    if (a.causal && at < all_rows) {
      const bool first = clean_tile<T, kD>(q_at), second = clean_tile<T, kD>(d_at);
      mark_rows(first || second, mark_s);
      clean_done();
    }
    if (at + kTile <= any) continue;
#pragma unroll
    for (uint32_t r = 0; r < 2; ++r) {
      f32x16 one[2];  // scores, then probabilities; their gradients, then the scores'
      clear(one);
#pragma unroll
      for (uint32_t i = 0; i < kD / 16; ++i) {
        one[0] = mfma32<T>(reads.rows(q_at, r, i), k.v[i], one[0]);
        one[1] = mfma32<T>(reads.rows(d_at, r, i), v.v[i], one[1]);
      }
#pragma unroll
      for (uint32_t i = 0; i < 4; ++i) {
        const f32x4* pair = reinterpret_cast<const f32x4*>(&row_s[buffer][32 * r + 8 * i + 4 * h]);
        const f32x4 x = pair[0], y = pair[1];
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) {
          const float lse = j < 2 ? x[2 * j] : y[2 * j - 4], mean = j < 2 ? x[2 * j + 1] : y[2 * j - 3];
          const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(one[0][4 * i + j], c, kUp - lse));
          one[0][4 * i + j] = p;
          one[1][4 * i + j] = p * (one[1][4 * i + j] - mean);
        }
      }
      if (at < whole || at + kTile > qs.count) {
        if (a.causal && at < all_rows) {
#pragma unroll
          for (uint32_t i = 0; i < 4; ++i) {
            const f32x4 mark = marks_of(mark_s, r, i);
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j) one[0][4 * i + j] += mark[j], one[1][4 * i + j] += mark[j];
          }
        }
        const int32_t lo = int32_t(from) - int32_t(at + 4 * h), hi = int32_t(qs.count) - int32_t(at + 4 * h);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int32_t x = int32_t(32 * r + 8 * (i / 4) + i % 4);
          if (x < lo || x >= hi) one[0][i] = one[1][i] = 0.0f;
        }
      }
      raised.raise(one[1], dk);
      if constexpr (std::is_same_v<T, F16>) one[1] *= raised.by;
#pragma unroll
      for (uint32_t u = 0; u < 2; ++u) {
        const bits8 p = pack8<T>(one[0], u), ds = pack8<T>(one[1], u);
#pragma unroll
        for (uint32_t t = 0; t < kD / 32; ++t) {
          dv[t] = mfma32<T>(reads.columns(d_at, t, 2 * r + u), p, dv[t]);
          dk[t] = mfma32<T>(reads.columns(q_at, t, 2 * r + u), ds, dk[t]);
        }
      }
    }
  }
  if (!on) return;
  const float back = __builtin_amdgcn_exp2f(-kUp);
  put_columns<T, kD, kAligned>(g.dk, uint64_t(ks.begin) + row, kept, a.head_dim, dk, a.scale * back * raised.down());
  put_columns<T, kD, kAligned>(g.dv, uint64_t(ks.begin) + row, kept, a.head_dim, dv, back);
}

template <class T, bool kAligned>
void rows_of(const tsa_attend_grad_args& g, float2* rows, hipStream_t stream) {
  const uint64_t n = uint64_t(g.f.tokens + 15) / 16 * g.f.q.heads;
  hipLaunchKernelGGL((rows_kernel<T, kAligned>), dim3(uint32_t(n)), dim3(256), 0, stream, g, rows);
}
template <class T, int kD, bool kAligned>
void gradients(const tsa_attend_grad_args& g, float2* rows, hipStream_t stream) {
  const tsa_attend_args& a = g.f;
  const float c = a.scale * 1.44269504f;
  if (a.tokens) rows_of<T, kAligned>(g, rows, stream);
  if (a.tokens && g.dq.p)
    hipLaunchKernelGGL((queries_kernel<T, kD, kAligned>), dim3(uint32_t(own_tiles_at_most(a.sequences, a.tokens) * a.q.heads)), dim3(64 * kTileWaves), 0,
                       stream, g, rows, c);
  if (a.k_tokens && g.dk.p)
    hipLaunchKernelGGL((keys_kernel<T, kD, kAligned>), dim3(uint32_t(own_tiles_at_most(a.sequences, a.k_tokens) * a.k.heads)), dim3(64 * kTileWaves), 0,
                       stream, g, rows, c);
}

}  // namespace
}  // namespace op

uint64_t attend_backward_workspace(const tsa_attend_args& f) { return uint64_t(f.tokens) * f.q.heads * sizeof(float2); }

int launch_attend_backward(const tsa_attend_grad_args& g, void* workspace, hipStream_t stream) {
  using namespace op;
  const tsa_attend_args& a = g.f;
  float2* rows = static_cast<float2*>(workspace);
  bool aligned = true;
  if (a.tokens) aligned = vector_heads(a.q) && vector_heads(a.out) && vector_heads(g.dout) && (!g.dq.p || vector_heads(g.dq));
  if (a.k_tokens) aligned = aligned && vector_heads(a.k) && vector_heads(a.v) && (!g.dk.p || (vector_heads(g.dk) && vector_heads(g.dv)));
#define CALL(T, D)                                                     \
  do {                                                                 \
    if (aligned) gradients<T, D, true>(g, rows, stream);               \
    else gradients<T, D, false>(g, rows, stream);                      \
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
