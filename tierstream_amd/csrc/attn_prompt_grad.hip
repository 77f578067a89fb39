// The gradients of attention over packed sequences. With p = exp(score - lse), dp = dout . v and ds = p (dp - dout . out):
//   dq = scale ds K    a workgroup has 128 queries of a head and runs over the keys,
//   dk = scale ds^T Q, dv = p^T dout    a workgroup has 128 keys of a kept head and runs over the queries of its group's heads,
// each in tiles of 64 through LDS as in the forward pass: the wave's own rows are the columns of every product, and p and ds, as they
// come out of the first products, the operand of the second. Scores are computed again in each pass. Sums over a workgroup's rows stay in
// its registers; where there are few tiles of keys their queries are cut into pieces, whose sums go to memory in 32 bits and are added
// up in order by a last launch: no atomics, the same bits every time. lse and sum p dp go to the workspace first, a pair a row.
// Measured: 8192 tokens in three sequences, 32 heads on 8 of 128, causal, after a forward pass of 239 to 250 us: the pairs 45, the gradients 861 to 907
// (ten products for the formula's seven, forward pass included: 840 TFLOP/s; alone dq takes 324, dk 364, dv 269), the joining launch 37. The matrix units
// are busy 44 to 52 % of the cycles, at 1.8 GHz. 301 tokens of 4 heads of 64: 6.7, 11.7 and 4.6, latency.
#include "attn_tile.hpp"

namespace tsa {
namespace op {
namespace {

// The queries of a workgroup, and what of the keys they attend to.
struct Queries {
  Span qs, ks;
  uint32_t head, kept;
  uint32_t row;        // this lane's
  bool on;
  uint32_t limit, all_rows, any, end;  // keys that this row; every row of the workgroup; any row of this wave; any row attends to
};
// By the whole workgroup; false: there are no more.
template <bool kFromEnd>
__device__ __forceinline__ bool find_queries(const tsa_attend_args& a, uint32_t group, OwnTileMemory& m, Queries& o) {
  OwnTile own;
  o.head = head_of_group(group % a.q.heads, a.q.heads), o.kept = o.head / (a.q.heads / a.k.heads);
  if (!find_own_tile<kFromEnd>(a.first, a.sequences, a.tokens, group / a.q.heads, m, own)) return false;
  o.qs = span_of(a.first, own.sequence, a.tokens), o.ks = span_of(a.k_first ? a.k_first : a.first, own.sequence, a.k_tokens);
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), row0 = own.row0 + wave * kOwn;
  o.row = row0 + (threadIdx.x & 31u), o.on = o.row < o.qs.count;
  const int32_t ahead = int32_t(o.ks.count) - int32_t(o.qs.count) + 1;
  auto keys_of = [&](uint32_t r) {
    const int32_t n = a.causal ? int32_t(r) + ahead : int32_t(o.ks.count);
    return n < 0 ? 0u : min(uint32_t(n), o.ks.count);
  };
  o.limit = o.on ? keys_of(o.row) : 0, o.all_rows = keys_of(own.row0);
  o.any = row0 < o.qs.count ? keys_of(min(row0 + kOwn, o.qs.count) - 1) : 0;
  o.end = keys_of(min(own.row0 + kTileOwn, o.qs.count) - 1);
  return true;
}

// The keys of a workgroup, and the piece of their queries that it has.
struct Keys {
  Span qs, ks;
  OwnTile own;
  uint32_t kept, piece;
};
__device__ __forceinline__ bool find_keys(const tsa_attend_args& a, uint32_t index, uint32_t pieces, OwnTileMemory& m, Keys& o) {
  const int32_t* k_first = a.k_first ? a.k_first : a.first;
  o.kept = head_of_group(index % a.k.heads, a.k.heads), o.piece = index / a.k.heads % pieces;
  if (!find_own_tile<false>(k_first, a.sequences, a.k_tokens, index / a.k.heads / pieces, m, o.own)) return false;
  o.qs = span_of(a.first, o.own.sequence, a.tokens), o.ks = span_of(k_first, o.own.sequence, a.k_tokens);
  return true;
}

// What is taken off the gradients of a row's probabilities, sum_j p_j dp_j. It is dout . out, but out is rounded to 16 bits, which over a
// few keys is as large an error in the gradients as their own rounding (over 10 keys they are off by 1.7 times what rounding the results
// costs, 1.4 without it; over 1000 it is lost in it): rows of workgroups that attend to no more keys than this add up p dp itself.
constexpr uint32_t kExactKeys = 512;

// (lse / ln 2, sum_j p_j dp_j) of each row; a row without keys has an lse of infinity, which makes its probabilities 0.
template <class T, int kD, bool kAligned>
__global__ __launch_bounds__(64 * kTileWaves, 2) void rows_kernel(tsa_attend_grad_args g, float2* rows, float c) {
  typedef TileShapes<kD> S;
  // (two tiles of 128 values leave room for two workgroups a CU instead of three: rows of many keys took 56 us for 45; of 64 values they do not, and
  // rows of 100 keys took 7.2 for 7.7)
  constexpr uint32_t kBuffers = kD == 64 ? 2 : 1;
  __shared__ __attribute__((aligned(16))) unsigned char tile_s[kBuffers][2][S::kBytes];  // keys and values
  __shared__ OwnTileMemory own_s;
  const tsa_attend_args& a = g.f;
  Queries o;
  if (!find_queries<false>(a, blockIdx.x, own_s, o)) return;  // (those with few keys first: they take longer)
  const uint32_t lane = threadIdx.x & 63u, h = lane >> 5;
  if (o.end > kExactKeys) {
    const uint32_t row0 = o.row - (lane & 31u) - (threadIdx.x >> 6) * kOwn, value = (lane & 15u) * 8;
#pragma unroll
    for (uint32_t j = 0; j < kTileOwn / (4 * kTileWaves); ++j) {
      const uint32_t i = j * 4 * kTileWaves + threadIdx.x / 16;
      const bool on = row0 + i < o.qs.count;
      const uint64_t t = uint64_t(o.qs.begin) + (on ? row0 + i : row0);
      float sum = 0.0f;
      if (value < a.head_dim) {
        const u16 *x = row_of<u16>(a.out, t, o.head) + value, *y = row_of<u16>(g.dout, t, o.head) + value;
        if constexpr (kAligned) {
          const bits8 u = *reinterpret_cast<const bits8*>(x), v = *reinterpret_cast<const bits8*>(y);
#pragma unroll
          for (int k = 0; k < 8; ++k) sum += T::up(u[k]) * T::up(v[k]);
        } else {
#pragma unroll
          for (int k = 0; k < 8; ++k) sum += T::up(x[k]) * T::up(y[k]);
        }
      }
#pragma unroll
      for (int s = 1; s < 16; s <<= 1) sum += __shfl_xor(sum, s, 64);
      if (on && value == 0) {
        const uint64_t at = uint64_t(o.head) * a.tokens + t;
        const float lse = a.lse[at];
        rows[at] = {lse == -INFINITY ? INFINITY : lse * 1.44269504f, sum};
      }
    }
    return;
  }
  const uint64_t at = uint64_t(o.head) * a.tokens + o.qs.begin + o.row;
  const OwnRows<kD, kAligned> q(a.q, uint64_t(o.qs.begin) + o.row, o.head, a.head_dim, o.on), dout(g.dout, uint64_t(o.qs.begin) + o.row, o.head, a.head_dim, o.on);
  float lse = o.on ? a.lse[at] : -INFINITY, sum = 0.0f;
  lse = lse == -INFINITY ? INFINITY : lse * 1.44269504f;
  const TileReads<kD> reads;
  const TileLoads<kD, kAligned> keys(a.k, o.ks.begin, o.kept, a.head_dim), values(a.v, o.ks.begin, o.kept, a.head_dim);
  const uint32_t lds = __builtin_amdgcn_readfirstlane(lds_offset(tile_s));
  auto fetch = [&](uint32_t key0, uint32_t at) {
    keys.fetch(key0, o.ks.count, at);
    values.fetch(key0, o.ks.count, at + S::kBytes);
  };
  auto other_of = [&](uint32_t tiles) { return kBuffers == 2 ? 2 * lds + 2 * S::kBytes - tiles : lds; };
  if (kBuffers == 2 && o.end) fetch(0, lds);
  for (uint32_t key0 = 0, tiles = lds; key0 < o.end; key0 += kTile, tiles = other_of(tiles)) {
    if (kBuffers == 1) {
      if (key0) tile_ready();  // the last tile's reads are done
      fetch(key0, lds);
    }
    tile_ready();
    if (kBuffers == 2 && key0 + kTile < o.end) fetch(key0 + kTile, other_of(tiles));
    if (key0 >= o.any) continue;
    const int32_t left = int32_t(o.limit) - int32_t(key0 + 4 * h);
    const auto k_rows = reads.rows(tiles), v_rows = reads.rows(tiles + S::kBytes);
#pragma unroll
    for (uint32_t r = 0; r < 2; ++r) {
      f32x16 one[2];
      clear(one);
#pragma unroll
      for (uint32_t k = 0; k < kD / 16; ++k) {
        one[0] = mfma32<T>(k_rows(r, k), q.v[k], one[0]);
        one[1] = mfma32<T>(v_rows(r, k), dout.v[k], one[1]);
      }
      products_behind_reads<kD / 8, 4>();
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (int32_t(32 * r + 8 * (i / 4) + i % 4) < left) sum += __builtin_amdgcn_exp2f(__builtin_fmaf(one[0][i], c, -lse)) * one[1][i];
    }
  }
  sum += __shfl_xor(sum, 32, 64);
  if (o.on && h == 0) rows[at] = {lse, sum};
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

template <int kD>
struct GradMemory {
  __attribute__((aligned(16))) unsigned char tile[2][2][TileShapes<kD>::kBytes];  // what a workgroup runs over, two tiles of each of two arrays
  __attribute__((aligned(16))) float2 row[2][kTile];
  __attribute__((aligned(16))) float mark[kTile];
  OwnTileMemory own;
};

template <class T, int kD, bool kAligned, bool kSplit>
__device__ __forceinline__ void queries_part(const tsa_attend_grad_args& g, const float2* rows, float c, const Queries& o, GradMemory<kD>& m) {
  typedef TileShapes<kD> S;
  const tsa_attend_args& a = g.f;
  const uint32_t h = (threadIdx.x & 63u) >> 5;
  const OwnRows<kD, kAligned> q(a.q, uint64_t(o.qs.begin) + o.row, o.head, a.head_dim, o.on), dout(g.dout, uint64_t(o.qs.begin) + o.row, o.head, a.head_dim, o.on);
  const float2 mine = o.on ? rows[uint64_t(o.head) * a.tokens + o.qs.begin + o.row] : float2{INFINITY, 0.0f};
  const TileReads<kD> reads;
  const TileLoads<kD, kAligned> keys(a.k, o.ks.begin, o.kept, a.head_dim), values(a.v, o.ks.begin, o.kept, a.head_dim);
  const uint32_t lds = __builtin_amdgcn_readfirstlane(lds_offset(m.tile));
  f32x16 dq[kD / 32];
  clear(dq);
  Raised<T> raised;

  if (o.end) {
    keys.fetch(0, o.ks.count, lds);
    values.fetch(0, o.ks.count, lds + S::kBytes);
  }
  for (uint32_t key0 = 0, buffer = 0; key0 < o.end; key0 += kTile, buffer ^= 1) {
    tile_ready();
    const uint32_t k_at = lds + buffer * 2 * S::kBytes, v_at = k_at + S::kBytes, other = lds + (buffer ^ 1) * 2 * S::kBytes;
    if (key0 + kTile < o.end) {
      keys.fetch(key0 + kTile, o.ks.count, other);
      values.fetch(key0 + kTile, o.ks.count, other + S::kBytes);
    }
    if (a.causal && key0 + kTile > o.all_rows) {
      mark_rows(clean_tile<T, kD>(k_at), m.mark);
      clean_done();
    }
    if (key0 >= o.any) continue;
    const auto k_rows = reads.rows(k_at), v_rows = reads.rows(v_at);
    const auto k_columns = reads.columns(k_at);
#pragma unroll
    for (uint32_t r = 0; r < 2; ++r) {
      f32x16 one[2];  // scores, then their gradients; gradients of probabilities
      clear(one);
#pragma unroll
      for (uint32_t k = 0; k < kD / 16; ++k) {
        one[0] = mfma32<T>(k_rows(r, k), q.v[k], one[0]);
        one[1] = mfma32<T>(v_rows(r, k), dout.v[k], one[1]);
      }
      products_behind_reads<kD / 8, 4>();
#pragma unroll
      for (int i = 0; i < 16; ++i)
        one[0][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(one[0][i], c, -mine.x)) * (one[1][i] - mine.y);
      if (key0 + kTile > o.all_rows) {  // (by every wave that reads a cleaned tile, whether or not the mask cuts its own rows)
        if (a.causal) {
#pragma unroll
          for (uint32_t i = 0; i < 4; ++i) {
            const f32x4 mark = marks_of(m.mark, r, i);
#pragma unroll
            for (uint32_t k = 0; k < 4; ++k) one[0][4 * i + k] += mark[k];
          }
        }
        const int32_t left = int32_t(o.limit) - int32_t(key0 + 4 * h);
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (int32_t(32 * r + 8 * (i / 4) + i % 4) >= left) one[0][i] = 0.0f;
      }
      raised.raise(one[0], dq);
      if constexpr (std::is_same_v<T, F16>) one[0] *= raised.by;
#pragma unroll
      for (uint32_t u = 0; u < 2; ++u) {
        const Second<T, kSplit> ds(one[0], u);
#pragma unroll
        for (uint32_t t = 0; t < kD / 32; ++t) ds.add(k_columns(t, 2 * r + u), dq[t]);
      }
    }
  }
  if (o.on) put_columns<T, kD, kAligned>(g.dq, uint64_t(o.qs.begin) + o.row, o.head, a.head_dim, dq, a.scale * raised.down());
}

// Half precision: probabilities of up to 2^14, so that small ones keep their bits.
template <class T>
constexpr float probability_up() {
  return std::is_same_v<T, F16> ? 14.0f : 0.0f;
}
// A result of the second kind to 32 bits in memory.
template <int kD>
__device__ __forceinline__ void put_part(float* p, const f32x16 (&v)[kD / 32], float by) {
#pragma unroll
  for (uint32_t t = 0; t < kD / 32; ++t)
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i)
      *reinterpret_cast<f32x4*>(p + 32 * t + 8 * i + 4 * ((threadIdx.x & 63u) >> 5)) =
          f32x4{v[t][4 * i] * by, v[t][4 * i + 1] * by, v[t][4 * i + 2] * by, v[t][4 * i + 3] * by};
}

// Both gradients of keys and values, or one. With 128 values both together need 430 registers, one wave a SIMD: they took 840 us in three
// packed sequences of 8192 together, one after the other with the scores computed again 660.
template <class T, int kD, bool kAligned, bool kSplit, bool kKeys, bool kValues>
__device__ __forceinline__ void keys_part(const tsa_attend_grad_args& g, const float2* rows, float c, const Keys& o, uint32_t pieces, float* parts, GradMemory<kD>& m) {
  typedef TileShapes<kD> S;
  constexpr float kUp = probability_up<T>();
  const tsa_attend_args& a = g.f;
  const Span qs = o.qs, ks = o.ks;
  const OwnTile own = o.own;
  const uint32_t kept = o.kept, piece = o.piece, group = a.q.heads / a.k.heads;
  const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5;
  const uint32_t row0 = own.row0 + wave * kOwn, row = row0 + (lane & 31u);
  const bool on = row < ks.count;
  // the first query that attends to a key
  auto from_of = [&](uint32_t key) {
    const int32_t n = a.causal ? int32_t(key) - int32_t(ks.count) + int32_t(qs.count) : 0;
    return n < 0 ? 0u : uint32_t(n);
  };
  const uint32_t from = from_of(row), any = from_of(row0), all_rows = from_of(own.row0 + kTileOwn - 1);
  const uint32_t begin = from_of(own.row0) / kTile * kTile, tiles = begin < qs.count ? (qs.count - begin + kTile - 1) / kTile : 0;
  // this piece's steps: a query tile of a head each
  const uint32_t step0 = uint32_t(uint64_t(tiles) * group * piece / pieces), steps = uint32_t(uint64_t(tiles) * group * (piece + 1) / pieces) - step0;

  const OwnRows<kD, kAligned> k(a.k, uint64_t(ks.begin) + row, kept, a.head_dim, on), v(a.v, uint64_t(ks.begin) + row, kept, a.head_dim, on);
  const TileReads<kD> reads;
  const uint32_t lds = __builtin_amdgcn_readfirstlane(lds_offset(m.tile)), row_lds = __builtin_amdgcn_readfirstlane(lds_offset(m.row));
  f32x16 dk[kKeys ? kD / 32 : 1], dv[kValues ? kD / 32 : 1];
  clear(dk);
  clear(dv);
  Raised<T> raised;

  uint32_t head = kept * group + (steps ? step0 / tiles : 0), q0 = begin + (steps ? step0 % tiles : 0) * kTile;  // of the step whose loads go next
  const uint32_t first_q = q0;
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
  for (uint32_t step = 0, buffer = 0, row_at = first_q; step < steps; ++step, buffer ^= 1) {
    tile_ready();
    const uint32_t q_at = lds + buffer * 2 * S::kBytes, d_at = q_at + S::kBytes, at = row_at;
    if (step + 1 < steps) fetch(buffer ^ 1);
    row_at = at + kTile >= qs.count ? begin : at + kTile;
    if (a.causal && at < all_rows) {
      const bool first = clean_tile<T, kD>(q_at), second = clean_tile<T, kD>(d_at);
      mark_rows(first || second, m.mark);
      clean_done();
    }
    if (at + kTile <= any) continue;
    const auto q_rows = reads.rows(q_at), d_rows = reads.rows(d_at);
    const auto q_columns = reads.columns(q_at), d_columns = reads.columns(d_at);
#pragma unroll
    for (uint32_t r = 0; r < 2; ++r) {
      f32x16 one[2];  // scores, then probabilities; their gradients, then the scores'
      clear(one);
      if constexpr (kKeys) {
        // reads kept four products ahead, in this order (with both kinds of sums behind them the compiler gave products_behind_reads up: 625 us
        // for 611, keys of three sequences of 2730, 32 heads on 8 of 128; 600 with one kind)
        constexpr uint32_t kProducts = kD / 8, kAhead = 4;
        bits8 ahead[kAhead];
        auto read = [&](uint32_t i) { ahead[i % kAhead] = i % 2 ? d_rows(r, i / 2) : q_rows(r, i / 2); };
#pragma unroll
        for (uint32_t i = 0; i < kAhead; ++i) read(i);
#pragma unroll
        for (uint32_t i = 0; i < kProducts; ++i) {
          __builtin_amdgcn_sched_barrier(0);
          one[i % 2] = mfma32<T>(ahead[i % kAhead], i % 2 ? v.v[i / 2] : k.v[i / 2], one[i % 2]);
          if (i + kAhead < kProducts) read(i + kAhead);
        }
      } else {
#pragma unroll
        for (uint32_t i = 0; i < kD / 16; ++i) one[0] = mfma32<T>(q_rows(r, i), k.v[i], one[0]);
      }
#pragma unroll
      for (uint32_t i = 0; i < 4; ++i) {
        const f32x4* pair = reinterpret_cast<const f32x4*>(&m.row[buffer][32 * r + 8 * i + 4 * h]);
        const f32x4 x = pair[0], y = pair[1];
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) {
          const float lse = j < 2 ? x[2 * j] : y[2 * j - 4], mean = j < 2 ? x[2 * j + 1] : y[2 * j - 3];
          const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(one[0][4 * i + j], c, kUp - lse));
          one[0][4 * i + j] = p;
          one[1][4 * i + j] = p * (one[1][4 * i + j] - mean);
        }
      }
      if (at < all_rows || at + kTile > qs.count) {  // (by every wave that reads a cleaned tile, whether or not the mask cuts its own keys)
        if (a.causal && at < all_rows) {
#pragma unroll
          for (uint32_t i = 0; i < 4; ++i) {
            const f32x4 mark = marks_of(m.mark, r, i);
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
      if constexpr (kKeys) {
        raised.raise(one[1], dk);
        if constexpr (std::is_same_v<T, F16>) one[1] *= raised.by;
      }
#pragma unroll
      for (uint32_t u = 0; u < 2; ++u) {
        const Second<T, kSplit> p(one[0], u), ds(one[1], u);
#pragma unroll
        for (uint32_t t = 0; t < kD / 32; ++t) {
          if constexpr (kValues) p.add(d_columns(t, 2 * r + u), dv[t]);
          if constexpr (kKeys) ds.add(q_columns(t, 2 * r + u), dk[t]);
        }
      }
    }
  }
  if (!on) return;
  if (pieces > 1) {
    float* const part = parts + ((uint64_t(piece) * a.k_tokens + ks.begin + row) * a.k.heads + kept) * 2 * kD;
    if constexpr (kKeys) put_part<kD>(part, dk, raised.down());
    if constexpr (kValues) put_part<kD>(part + kD, dv, 1.0f);
    return;
  }
  const float back = __builtin_amdgcn_exp2f(-kUp);
  if constexpr (kKeys) put_columns<T, kD, kAligned>(g.dk, uint64_t(ks.begin) + row, kept, a.head_dim, dk, a.scale * back * raised.down());
  if constexpr (kValues) put_columns<T, kD, kAligned>(g.dv, uint64_t(ks.begin) + row, kept, a.head_dim, dv, back);
}

// All gradients in one launch, whose parts fill what others leave idle (one launch each took 50 us more of 1000, and 9 of 21 where all is
// latency). The keys', with up to 64 values at once with the values', first: theirs are the longest workgroups.
struct GradGrid {
  uint32_t queries, keys;  // workgroups
};
template <class T, int kD, bool kAligned, bool kKeys, bool kValues>
__device__ __forceinline__ void keys_of_group(const tsa_attend_grad_args& g, const float2* rows, float c, uint32_t pieces, float* parts, GradMemory<kD>& m) {
  Keys o;
  if (!find_keys(g.f, blockIdx.x, pieces, m.own, o)) return;
  if (both_parts(o.qs.count, o.ks.count)) keys_part<T, kD, kAligned, true, kKeys, kValues>(g, rows, c, o, pieces, parts, m);
  else keys_part<T, kD, kAligned, false, kKeys, kValues>(g, rows, c, o, pieces, parts, m);
}
template <class T, int kD, bool kAligned>
__global__ __launch_bounds__(64 * kTileWaves, 2) void gradients_kernel(tsa_attend_grad_args g, const float2* rows, float c, uint32_t pieces, float* parts, GradGrid n) {
  __shared__ GradMemory<kD> m;
  if (blockIdx.y + 1 == gridDim.y) {
    Queries o;
    if (blockIdx.x >= n.queries || !find_queries<true>(g.f, blockIdx.x, m.own, o)) return;
    if (both_parts(o.qs.count, o.ks.count)) queries_part<T, kD, kAligned, true>(g, rows, c, o, m);
    else queries_part<T, kD, kAligned, false>(g, rows, c, o, m);
  } else if (blockIdx.x < n.keys) {
    if (blockIdx.y == 0) keys_of_group<T, kD, kAligned, true, kD == 64>(g, rows, c, pieces, parts, m);
    else if constexpr (kD != 64) keys_of_group<T, kD, kAligned, false, true>(g, rows, c, pieces, parts, m);
  }
}

// The pieces' sums, rounded: four values a thread.
template <class T, int kD, bool kAligned>
__global__ __launch_bounds__(256) void join_kernel(tsa_attend_grad_args g, uint32_t pieces, const float* parts) {
  const tsa_attend_args& a = g.f;
  const uint64_t i = uint64_t(blockIdx.x) * 256 + threadIdx.x;
  constexpr uint32_t kRow = 2 * kD / 4;
  const uint32_t in = uint32_t(i % kRow), d = in * 4 % kD;
  const uint64_t head_row = i / kRow, row = head_row / a.k.heads;
  if (row >= a.k_tokens || d >= a.head_dim) return;
  const int32_t* k_first = a.k_first ? a.k_first : a.first;
  const uint32_t n = sequence_of(k_first, a.sequences, uint32_t(row));
  if (n >= a.sequences) return;
  const Span ks = span_of(k_first, n, a.k_tokens);
  if (row < ks.begin || row >= uint64_t(ks.begin) + ks.count) return;
  f32x4 sum = {0, 0, 0, 0};
  for (uint32_t p = 0; p < pieces; ++p) sum += reinterpret_cast<const f32x4*>(parts)[p * (uint64_t(a.k_tokens) * a.k.heads * kRow) + i];
  const bool value = in * 4 >= kD;
  sum *= (value ? 1.0f : a.scale) * __builtin_amdgcn_exp2f(-probability_up<T>());
  put4<T, kAligned>(const_cast<u16*>(row_of<u16>(value ? g.dv : g.dk, row, uint32_t(head_row % a.k.heads))) + d, sum[0], sum[1], sum[2], sum[3]);
}

// Pieces that a workgroup's queries are cut into, as many as make twice the workgroups that run at once: with fewer the chip would idle, or
// wait for the longest (the first keys of the longest sequence have all queries, the last ones a tile). Each piece's sums go to memory in 32
// bits. In three packed sequences of 8192 together, 520 tiles: uncut 957 us, in two pieces 907 and 37 to join them, in three 945 and 49.
constexpr uint32_t kEnough = 1024, kMaxPieces = 8;
uint32_t pieces_of(const tsa_attend_args& a) {
  const uint64_t tiles = (uint64_t(a.k_tokens) / kTileOwn + 1) * a.k.heads, n = (kEnough + tiles - 1) / tiles;
  return n > kMaxPieces ? kMaxPieces : uint32_t(n);
}

template <class T, int kD, bool kAligned>
void gradients(const tsa_attend_grad_args& g, float2* rows, float* parts, hipStream_t stream) {
  const tsa_attend_args& a = g.f;
  const float c = a.scale * 1.44269504f;
  const uint32_t queries = a.tokens ? uint32_t(own_tiles_at_most(a.sequences, a.tokens) * a.q.heads) : 0, pieces = pieces_of(a);
  const bool keys = a.k_tokens && g.dk.p;
  const GradGrid n = {g.dq.p ? queries : 0, keys ? uint32_t(own_tiles_at_most(a.sequences, a.k_tokens) * a.k.heads * pieces) : 0};
  if (queries) hipLaunchKernelGGL((rows_kernel<T, kD, kAligned>), dim3(queries), dim3(64 * kTileWaves), 0, stream, g, rows, c);
  const dim3 grid(n.queries > n.keys ? n.queries : n.keys, !keys ? 1 : kD == 64 ? 2 : 3);
  hipLaunchKernelGGL((gradients_kernel<T, kD, kAligned>), grid, dim3(64 * kTileWaves), 0, stream, g, rows, c, pieces, parts, n);
  if (keys) {
    if (pieces > 1) {
      const uint64_t n = uint64_t(a.k_tokens) * a.k.heads * (2 * kD / 4);
      hipLaunchKernelGGL((join_kernel<T, kD, kAligned>), dim3(uint32_t((n + 255) / 256)), dim3(256), 0, stream, g, pieces, parts);
    }
  }
}

}  // namespace
}  // namespace op

// The rows' pairs, then the pieces (their rows together are at most kMaxPieces times the keys, and what twice kEnough tiles hold: so that
// more rows never need less).
uint64_t attend_backward_workspace(const tsa_attend_args& f) {
  const uint64_t many = uint64_t(op::kMaxPieces) * f.k_tokens * f.k.heads, most = uint64_t(2 * op::kEnough) * op::kTileOwn;
  return up_to(uint64_t(f.tokens) * f.q.heads * sizeof(float2), 16) + (many < most ? many : most) * 2 * (f.head_dim <= 64 ? 64 : 128) * sizeof(float);
}

int launch_attend_backward(const tsa_attend_grad_args& g, void* workspace, hipStream_t stream) {
  using namespace op;
  const tsa_attend_args& a = g.f;
  float2* rows = static_cast<float2*>(workspace);
  float* parts = reinterpret_cast<float*>(static_cast<char*>(workspace) + up_to(uint64_t(a.tokens) * a.q.heads * sizeof(float2), 16));
  bool aligned = true;
  if (a.tokens) aligned = tile_heads(a.q) && vector_heads(a.out) && tile_heads(g.dout) && (!g.dq.p || vector_heads(g.dq));
  if (a.k_tokens) aligned = aligned && tile_heads(a.k) && tile_heads(a.v) && (!g.dk.p || (vector_heads(g.dk) && vector_heads(g.dv)));
#define CALL(T, D)                                                  \
  do {                                                              \
    if (aligned) gradients<T, D, true>(g, rows, parts, stream);     \
    else gradients<T, D, false>(g, rows, parts, stream);            \
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
