// The paged cache of 4-bit keys and values: pages, positions and slots of a step (integers, one workgroup: latency), and keys and
// values to their slots and back (memory).
#include "attn_device.hpp"

namespace tsa {
namespace op {
namespace {

// ---- pages and slots ----
__device__ __forceinline__ uint32_t pages_of(uint32_t tokens) { return tokens / kPage + (tokens % kPage != 0); }

// Three 64-bit counts of each thread: their sums over the threads before it, and over all.
template <uint32_t kThreads>
__device__ __forceinline__ void scan(const int64_t (&v)[3], int64_t (&before)[3], int64_t (&all)[3], int64_t (&waves)[3][kThreads / 64]) {
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    int64_t upto = v[k];
#pragma unroll
    for (uint32_t s = 1; s < 64; s <<= 1) {
      const int64_t o = __shfl_up(upto, s, 64);
      if (lane >= s) upto += o;
    }
    before[k] = upto - v[k];
    if (lane == 63) waves[k][wave] = upto;
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    all[k] = 0;
#pragma unroll
    for (uint32_t w = 0; w < kThreads / 64; ++w) {
      if (w < wave) before[k] += waves[k][w];
      all[k] += waves[k][w];
    }
  }
}

// The last i with first[i] <= x, of first[0] = 0 <= ... <= first[n], x < first[n].
template <class I>
__device__ __forceinline__ uint32_t owner_of(const I* first, uint32_t n, I x) {
  uint32_t lo = 0, hi = n;
  while (hi - lo > 1) {
    const uint32_t mid = (lo + hi) / 2;
    if (first[mid] <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

// A plan's sums over the requests before each: its rows, the pages it takes and the pages it gives back; and its length before.
template <uint32_t kMost>
struct PlanSums {
  int32_t first[kMost + 1], taken[kMost + 1], given[kMost + 1], length[kMost];
};

// A plan's pages and rows by several workgroups, each of which adds up all requests itself; the first also writes what the host may have put
// in an input's place (ends over lengths). Where it has, one workgroup does all, or with more than kPlanMany rows a launch behind them does this. Pages given back and pages taken in
// one plan pass each other by: the k-th page taken is the k-th last given, or lies that far down in the stack, so that nothing waits for
// what another thread writes. 32 requests 3 us, a launch and three memory latencies (9 with 1024 threads and a barrier between giving and
// taking); 2047 requests with 65536 rows and some 10,000 pages given back 12.6, and 5.8 for the launch behind (26 together by one workgroup).
template <uint32_t kThreads, uint32_t kPer>
__global__ __launch_bounds__(kThreads) void plan_kernel(tsa_cache_plan_args a, bool work, bool finish) {
  finish = finish && blockIdx.x == 0;
  constexpr uint32_t kMost = kThreads * kPer;
  __shared__ int64_t waves[3][kThreads / 64];
  __shared__ PlanSums<kMost> sum_s;
  __shared__ uint32_t bad_s;
  const uint32_t t = threadIdx.x;
  if (t == 0) bad_s = 0;
  const int64_t n_free = a.n_free[0];
  // memory in whole lines and all at once (one request after the other a thread waited for each: 9 us for 2047), then by way of LDS
  int32_t line[2][kPer];
#pragma unroll
  for (uint32_t k = 0; k < kPer; ++k) {
    const uint32_t i = k * kThreads + t;
    line[0][k] = i < a.requests ? a.lengths[i] : 0;
    line[1][k] = i < a.requests ? a.fresh[i] : 0;
  }
#pragma unroll
  for (uint32_t k = 0; k < kPer; ++k) {
    sum_s.length[k * kThreads + t] = line[0][k];
    sum_s.first[k * kThreads + t] = line[1][k];
  }
  __syncthreads();
  int32_t length[kPer], fresh[kPer];
  int64_t add = 0, need = 0, gone = 0;
  uint32_t bad = 0;
#pragma unroll
  for (uint32_t k = 0; k < kPer; ++k) {  // thread t has requests kPer t..
    const uint32_t i = t * kPer + k;
    length[k] = sum_s.length[i];
    fresh[k] = sum_s.first[i];
  }
#pragma unroll
  for (uint32_t k = 0; k < kPer; ++k) {
    if (length[k] < 0) {
      bad |= 8;
      continue;
    }
    const uint32_t end = uint32_t(length[k]) + (fresh[k] < 0 ? 0u : uint32_t(fresh[k])), have = pages_of(uint32_t(length[k]));
    if (pages_of(end) > a.width || end > uint32_t(INT32_MAX)) bad |= 4;
    if (fresh[k] < 0) gone += have;
    else add += fresh[k], need += pages_of(end) - have;
  }
  int64_t before[3], all[3];
  scan<kThreads>({add, need, gone}, before, all, waves);
  const int64_t adds = all[0], needs = all[1], gones = all[2];
  if (n_free < 0 || n_free > a.pages || n_free + gones > a.pages) bad |= 8;
  if (needs > n_free + gones) bad |= 1;
  if (adds > a.rows) bad |= 2;
  if (bad) atomicOr(&bad_s, bad);
  __syncthreads();
  const bool ok = bad_s == 0;
  int64_t at_add = before[0], at_need = before[1], at_gone = before[2];
#pragma unroll
  for (uint32_t k = 0; k < kPer; ++k) {
    const uint32_t i = t * kPer + k;
    if (i >= a.requests) break;
    const bool over = fresh[k] < 0;
    sum_s.first[i] = ok ? int32_t(at_add) : 0;
    sum_s.taken[i] = int32_t(at_need);
    sum_s.given[i] = int32_t(at_gone);
    if (!ok) continue;
    if (over) at_gone += pages_of(uint32_t(length[k]));
    else at_add += fresh[k], at_need += pages_of(uint32_t(length[k]) + uint32_t(fresh[k])) - pages_of(uint32_t(length[k]));
  }
  const uint32_t rows = ok ? uint32_t(adds) : 0;
  if (t == 0) {
    sum_s.first[a.requests] = int32_t(rows);
    if (finish) {
      a.first[a.requests] = int32_t(rows);
      a.left[0] = int32_t(ok ? n_free + gones - needs : n_free);
      a.status[0] = int32_t(bad_s);
    }
  }
  __syncthreads();
  if (finish) {
#pragma unroll
    for (uint32_t k = 0; k < kPer; ++k) {
      const uint32_t i = k * kThreads + t;
      if (i >= a.requests) break;
      a.ends[i] = !ok ? line[0][k] : line[1][k] < 0 ? 0 : line[0][k] + line[1][k];
      a.first[i] = sum_s.first[i];
    }
  }
  if (!work) return;
  const uint32_t step = gridDim.x * kThreads, from = blockIdx.x * kThreads + t;
  // page j of those given back, and the k-th page taken
  auto given = [&](uint32_t j) {
    const uint32_t i = owner_of(sum_s.given, a.requests, int32_t(j));
    return a.table[i * a.table_stride + (j - uint32_t(sum_s.given[i]))];
  };
  auto taken = [&](uint32_t k) { return k < gones ? given(uint32_t(gones) - 1 - k) : a.free[n_free - 1 - (int64_t(k) - gones)]; };
  if (ok) {
    for (uint32_t j = from; j < uint32_t(gones); j += step) a.free[n_free + j] = given(j);
    for (uint32_t k = from; k < uint32_t(needs); k += step) {
      const uint32_t i = owner_of(sum_s.taken, a.requests, int32_t(k));
      a.table[i * a.table_stride + pages_of(uint32_t(sum_s.length[i])) + (k - uint32_t(sum_s.taken[i]))] = taken(k);
    }
  }
  for (uint32_t r = from; r < a.rows; r += step) {
    int32_t position = -1, slot = -1;
    if (r < rows) {
      const uint32_t i = owner_of(sum_s.first, a.requests, int32_t(r)), have = pages_of(uint32_t(sum_s.length[i]));
      position = sum_s.length[i] + int32_t(r - uint32_t(sum_s.first[i]));
      const uint32_t p = uint32_t(position) / kPage;
      const int32_t page = p < have ? a.table[i * a.table_stride + p] : taken(uint32_t(sum_s.taken[i]) + p - have);
      if (page >= 0 && page < (1 << 25)) slot = page * int32_t(kPage) + position % int32_t(kPage);
    }
    a.positions[r] = position;
    a.slots[r] = slot;
  }
}

// 2047 requests and 65536 rows 4.0 us, one row 1.4: a launch.
__global__ __launch_bounds__(256) void slots_kernel(tsa_cache_plan_args a) {
  const uint32_t r = blockIdx.x * 256 + threadIdx.x;
  if (r >= a.rows) return;
  const int64_t rows = a.requests ? a.first[a.requests] : 0;
  int64_t position = -1;
  int32_t slot = -1;
  if (int64_t(r) < rows && int64_t(r) >= a.first[0]) {
    const uint32_t i = owner_of(a.first, a.requests, int32_t(r));
    position = int64_t(a.ends[i]) - a.first[i + 1] + r;
    if (position < 0) {
      position = -1;
    } else if (position / kPage < a.width) {
      const int32_t page = a.table[i * a.table_stride + position / kPage];
      if (page >= 0 && page < (1 << 25)) slot = page * int32_t(kPage) + int32_t(position % kPage);
    }
  }
  a.positions[r] = int32_t(position);
  a.slots[r] = slot;
}

// ---- keys and values to their slots and back ----
// Four lanes a block of 32 values, 8 each: whole blocks are read in whole lines, and the largest of a block is two moves inside four lanes.
// 8191 tokens of 8 heads of 128: a store 14.8 us (2.9 TB/s read and written), a load 11.0 (3.9); what bounds the store are the instructions of
// the rounding, some 20 a value. 32 tokens: 3.7 and 3.1, a launch. Keys and values of a block by one thread were 0.2 and 0.7 us faster on many
// tokens and 0.7 and 0.2 slower on few. kVector: rows whose pieces of 8 values start 16-byte aligned.
__device__ __forceinline__ bits8 load8(const tsa_heads& h, uint64_t at, bool vector) {
  const u16* p = static_cast<const u16*>(h.p) + at;
  if (vector) return *reinterpret_cast<const bits8*>(p);
  bits8 v;
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = p[i];
  return v;
}

// Where a block of a head lies in its page.
struct BlockPlace {
  unsigned char* page;
  uint32_t row, nb, b;
  __device__ __forceinline__ unsigned char* key_word(uint32_t g) const { return page + row * nb * 16 + (g * nb + b) * 4; }
  __device__ __forceinline__ unsigned char* value_bytes() const { return page + nb * 1280 + (b * kPage + row) * 16; }
  __device__ __forceinline__ u16* scale(bool value) const {
    return reinterpret_cast<u16*>(page + nb * (value ? 1152 : 1024)) + row * nb + b;
  }
};
struct RowPiece {  // piece j of block b of head h of token t, of k and of v
  uint32_t t, h, b, j;
  bool on;
};
// A workgroup takes a head of as many tokens as there are threads for: tokens behind each other lie behind each other in a page, and
// its lines are written whole by one XCD (two tokens of all heads a workgroup: 17.8 us and 14.2).
__device__ __forceinline__ RowPiece row_piece(const tsa_cache& c, uint32_t tokens) {
  const uint32_t nb = c.head_dim / 32, many = 64 / nb, block = threadIdx.x >> 2;
  RowPiece p;
  p.j = threadIdx.x & 3u;
  const uint32_t t = nb == 4 ? block / 4 : block / nb;
  p.b = block - t * nb;
  p.t = blockIdx.x * many + t;
  p.h = blockIdx.y;
  p.on = t < many && p.t < tokens;
  return p;
}
__device__ __forceinline__ BlockPlace place_of(const tsa_cache& c, uint32_t slot, const RowPiece& p) {
  return {static_cast<unsigned char*>(c.pages) + (uint64_t(slot / kPage) * c.kv_heads + p.h) * (72 * c.head_dim), slot % kPage, c.head_dim / 32, p.b};
}
__device__ __forceinline__ uint64_t place_in(const tsa_heads& h, const RowPiece& p) {
  return uint64_t(p.t) * h.token_stride + uint64_t(p.h) * h.head_stride + p.b * 32 + p.j * 8;
}

// A block by its four lanes: the scale, and (in lanes 0 and 1) this lane's 8 bytes.
struct Packed {
  uint32_t lo, hi;
  u16 scale;
};
template <class T>
__device__ __forceinline__ Packed pack_block(bits8 raw) {
  constexpr uint32_t kInfinity = std::is_same_v<T, Bf16> ? 0x7F80 : 0x7C00;
  // the largest size, by its bits; then the first value that has it
  const bits8 size = raw & u16(0x7FFF);
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = size[i] > top ? size[i] : top;
#pragma unroll
  for (int s = 1; s < 4; s <<= 1) {
    const uint32_t o = __shfl_xor(top, s, 64);
    top = o > top ? o : top;
  }
  uint32_t mine = 0;
  bool there = false;
#pragma unroll
  for (int i = 7; i >= 0; --i)
    if (size[i] == top) mine = raw[i], there = true;
  const uint32_t lane = threadIdx.x & 63u, quad = lane & 60u;
  const uint32_t has = uint32_t(__ballot(there) >> quad) & 15u, minus = uint32_t(__ballot(there && (mine & 0x8000u)) >> quad) & 15u;
  const bool finite = top < kInfinity, negative = (minus & has & (0u - has)) != 0;
  // (-big / 8 is exact; a scale beyond half precision is an infinity and 0 times it is NaN, as it should be)
  const float big = T::up(u16(top));
  const u16 scale = finite ? F16::down(negative ? big * 0.125f : big * -0.125f) : u16(0x7E00);
  const float step = F16::up(scale), each = finite && big != 0.0f && step != 0.0f ? 1.0f / step : 0.0f;
  uint32_t lo = 0, hi = 0;  // 8 half bytes, one a byte
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    // The nearest whole step, ties to even. The quotient of a 16-bit value and a half-precision step lies on a border between two
    // steps or 2^-15 of itself away from it: taken through the reciprocal it is off by 2^-23, which moves it over none, but may move it off one
    // that it lies on. What is left of it is exact, and is half a step on a border alone.
    const float x = T::up(raw[i]);
    float q = each == 0.0f ? 0.0f : rintf(x * each);
    const float left = 2.0f * __builtin_fmaf(-q, step, x);
    if (fabsf(left) == fabsf(step) && (int(q) & 1)) q += (left < 0.0f) == (step < 0.0f) ? 1.0f : -1.0f;
    q = __builtin_amdgcn_fmed3f(q, -8.0f, 7.0f);
    const uint32_t n = uint32_t(int(q) + 8);
    if (i < 4) lo |= n << (8 * i);
    else hi |= n << (8 * (i - 4));
  }
  // values 16.. of the block go to the high halves of bytes 0..
  lo |= __shfl_xor(lo, 2, 64) << 4;
  hi |= __shfl_xor(hi, 2, 64) << 4;
  return {lo, hi, scale};
}

// What a thread reads is on its way before its slot is known.
template <class T>
__global__ __launch_bounds__(256) void store_kernel(tsa_cache c, tsa_cache_rows_args a, bool vector) {
  const RowPiece p = row_piece(c, a.tokens);
  if (!p.on) return;
  const bool value = blockIdx.z;
  const uint32_t slot = uint32_t(a.slots[p.t]);
  const tsa_heads& h = value ? a.v : a.k;
  const bits8 raw = load8(h, place_in(h, p), vector);
  if (slot >= c.n_pages * kPage) return;  // (a block's four lanes go together)
  const BlockPlace at = place_of(c, slot, p);
  const Packed w = pack_block<T>(raw);
  if (p.j == 3) *at.scale(value) = w.scale;
  if (p.j >= 2) return;
  if (value) {
    *reinterpret_cast<uint2*>(at.value_bytes() + 8 * p.j) = uint2{w.lo, w.hi};
  } else {
    *reinterpret_cast<uint32_t*>(at.key_word(2 * p.j)) = w.lo;
    *reinterpret_cast<uint32_t*>(at.key_word(2 * p.j + 1)) = w.hi;
  }
}

template <class T>
__global__ __launch_bounds__(256) void load_kernel(tsa_cache c, tsa_cache_rows_args a, bool vector) {
  const RowPiece p = row_piece(c, a.tokens);
  const uint32_t slot = p.on ? uint32_t(a.slots[p.t]) : ~0u;
  if (slot >= c.n_pages * kPage) return;
  const bool value = blockIdx.z;
  const BlockPlace at = place_of(c, slot, p);
  uint2 w;
  const uint32_t half = p.j & 1u;
  if (value) w = *reinterpret_cast<const uint2*>(at.value_bytes() + 8 * half);
  else w = uint2{*reinterpret_cast<const uint32_t*>(at.key_word(2 * half)), *reinterpret_cast<const uint32_t*>(at.key_word(2 * half + 1))};
  const float step = F16::up(*at.scale(value));
  bits8 out;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t n = ((i < 4 ? w.x : w.y) >> (8 * (i & 3) + (p.j >= 2 ? 4 : 0))) & 15u;
    out[i] = T::down(float(int(n) - 8) * step);
  }
  const tsa_heads& h = value ? a.v : a.k;
  u16* to = static_cast<u16*>(h.p) + place_in(h, p);
  if (vector) {
    *reinterpret_cast<bits8*>(to) = out;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) to[i] = out[i];
  }
}

dim3 row_grid(const tsa_cache& c, uint32_t tokens) {
  const uint32_t many = 64 / (c.head_dim / 32);
  return dim3((tokens + many - 1) / many, c.kv_heads, 2);
}

}  // namespace
}  // namespace op

namespace op {
namespace {
constexpr uint32_t kPlanMany = 8192;  // rows that one workgroup writes faster than a second launch begins

template <uint32_t kThreads, uint32_t kPer>
void plan(const tsa_cache_plan_args& a, hipStream_t stream) {
  const bool in_place = (a.requests && a.ends == a.lengths) || a.left == a.n_free;
  const uint32_t many = a.rows / (2 * kThreads) + 1, groups = in_place && a.rows <= kPlanMany ? 1 : many < 256 ? many : 256;
  const bool behind = in_place && groups > 1;
  hipLaunchKernelGGL((plan_kernel<kThreads, kPer>), dim3(groups), dim3(kThreads), 0, stream, a, true, !behind);
  if (behind) hipLaunchKernelGGL((plan_kernel<kThreads, kPer>), dim3(1), dim3(kThreads), 0, stream, a, false, true);
}
}  // namespace
}  // namespace op

int launch_cache_plan(const tsa_cache_plan_args& a, hipStream_t stream) {
  // the fewest threads that hold the requests, and do not take many turns over the rows
  if (a.requests <= 64 && (a.rows <= 256 || a.rows > op::kPlanMany)) op::plan<64, 1>(a, stream);
  else if (a.requests <= 256 && (a.rows <= 1024 || a.rows > op::kPlanMany)) op::plan<256, 1>(a, stream);
  else op::plan<512, TSA_CACHE_MAX_REQUESTS / 512>(a, stream);
  return int(hipGetLastError());
}

int launch_cache_slots(const tsa_cache_plan_args& a, hipStream_t stream) {
  hipLaunchKernelGGL(op::slots_kernel, dim3((a.rows + 255) / 256), dim3(256), 0, stream, a);
  return int(hipGetLastError());
}

int launch_cache_store(const tsa_cache& c, const tsa_cache_rows_args& a, hipStream_t stream) {
  const bool vector = op::vector_heads(a.k) && op::vector_heads(a.v);
  const dim3 grid = op::row_grid(c, a.tokens);
  if (a.type == TSA_BF16) hipLaunchKernelGGL(op::store_kernel<op::Bf16>, grid, dim3(256), 0, stream, c, a, vector);
  else hipLaunchKernelGGL(op::store_kernel<op::F16>, grid, dim3(256), 0, stream, c, a, vector);
  return int(hipGetLastError());
}

int launch_cache_load(const tsa_cache& c, const tsa_cache_rows_args& a, hipStream_t stream) {
  const bool vector = op::vector_heads(a.k) && op::vector_heads(a.v);
  const dim3 grid = op::row_grid(c, a.tokens);
  if (a.type == TSA_BF16) hipLaunchKernelGGL(op::load_kernel<op::Bf16>, grid, dim3(256), 0, stream, c, a, vector);
  else hipLaunchKernelGGL(op::load_kernel<op::F16>, grid, dim3(256), 0, stream, c, a, vector);
  return int(hipGetLastError());
}

}  // namespace tsa
