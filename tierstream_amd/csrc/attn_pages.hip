// The paged cache of 4-bit keys and values: pages, positions and slots of a step (integers, one workgroup: latency), and keys and
// values to their slots and back (memory).
#include "attn_device.hpp"

namespace tsa {
namespace op {
namespace {

// ---- pages and slots ----
constexpr uint32_t kPlanThreads = 1024, kPlanPer = TSA_CACHE_MAX_REQUESTS / kPlanThreads;
constexpr uint32_t kPlanRows = 8192;  // rows that the planning workgroup writes itself: a second launch costs more below

__device__ __forceinline__ uint32_t pages_of(int64_t tokens) { return uint32_t((tokens + kPage - 1) / kPage); }

// Inclusive sums of 64-bit counts over the workgroup's threads; `all`: the whole sum.
__device__ __forceinline__ int64_t scan(int64_t v, int64_t* waves, int64_t& all) {
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
#pragma unroll
  for (uint32_t s = 1; s < 64; s <<= 1) {
    const int64_t o = __shfl_up(v, s, 64);
    if (lane >= s) v += o;
  }
  __syncthreads();  // the last scan's sums are read
  if (lane == 63) waves[wave] = v;
  __syncthreads();
  all = 0;
  int64_t before = 0;
#pragma unroll
  for (uint32_t w = 0; w < kPlanThreads / 64; ++w) {
    if (w == wave) before = all;
    all += waves[w];
  }
  return before + v;
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

// Row r's position and slot, from the requests' rows (first) and ends.
__device__ __forceinline__ void write_slot(const tsa_cache_plan_args& a, const int32_t* first, int64_t rows, const int32_t* ends, uint32_t r) {
  int64_t position = -1;
  int32_t slot = -1;
  if (int64_t(r) < rows) {
    const uint32_t i = owner_of(first, a.requests, int32_t(r));
    position = int64_t(ends[i]) - first[i + 1] + r;
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

__global__ __launch_bounds__(kPlanThreads) void plan_kernel(tsa_cache_plan_args a, uint32_t write_rows) {
  __shared__ int64_t waves[kPlanThreads / 64];
  __shared__ int32_t first_s[TSA_CACHE_MAX_REQUESTS + 1], end_s[TSA_CACHE_MAX_REQUESTS];
  __shared__ int32_t taken_s[TSA_CACHE_MAX_REQUESTS + 1], given_s[TSA_CACHE_MAX_REQUESTS + 1];
  __shared__ uint32_t bad_s;
  const uint32_t t = threadIdx.x;
  if (t == 0) bad_s = 0;
  int32_t length[kPlanPer], fresh[kPlanPer];
  int64_t add = 0, need = 0, gone = 0;
  uint32_t bad = 0;
#pragma unroll
  for (uint32_t k = 0; k < kPlanPer; ++k) {  // thread t has requests 4 t..
    const uint32_t i = t * kPlanPer + k;
    length[k] = i < a.requests ? a.lengths[i] : 0;
    fresh[k] = i < a.requests ? a.fresh[i] : 0;
    if (length[k] < 0) {
      bad |= 8;
      continue;
    }
    const int64_t end = int64_t(length[k]) + fresh[k];
    if (fresh[k] < 0) {
      gone += pages_of(length[k]);
      if (pages_of(length[k]) > a.width) bad |= 4;
    } else {
      add += fresh[k];
      if (pages_of(end) > a.width || end > INT32_MAX) bad |= 4;
      else need += pages_of(end) - pages_of(length[k]);
    }
  }
  int64_t adds, needs, gones;
  const int64_t add0 = scan(add, waves, adds) - add, need0 = scan(need, waves, needs) - need, gone0 = scan(gone, waves, gones) - gone;
  const int64_t n_free = a.n_free[0];
  if (n_free < 0 || n_free > a.pages || n_free + gones > a.pages) bad |= 8;
  if (needs > n_free + gones) bad |= 1;
  if (adds > a.rows) bad |= 2;
  if (bad) atomicOr(&bad_s, bad);
  __syncthreads();
  const bool ok = bad_s == 0;
  const int32_t count = int32_t(ok ? n_free + gones : n_free);
  int64_t at_add = add0, at_need = need0, at_gone = gone0;
#pragma unroll
  for (uint32_t k = 0; k < kPlanPer; ++k) {
    const uint32_t i = t * kPlanPer + k;
    if (i >= a.requests) break;
    const bool over = fresh[k] < 0;
    const int32_t end = !ok ? length[k] : over ? 0 : length[k] + fresh[k];
    first_s[i] = ok ? int32_t(at_add) : 0;
    end_s[i] = end;
    taken_s[i] = int32_t(at_need);
    given_s[i] = int32_t(at_gone);
    a.ends[i] = end;
    a.first[i] = first_s[i];
    if (!ok) continue;
    if (over) at_gone += pages_of(length[k]);
    else at_add += fresh[k], at_need += pages_of(end) - pages_of(length[k]);
  }
  const int32_t rows = ok ? int32_t(adds) : 0;
  if (t == 0) {
    first_s[a.requests] = rows;
    a.first[a.requests] = rows;
    a.left[0] = ok ? int32_t(count - needs) : count;
    a.status[0] = int32_t(bad_s);
  }
  __syncthreads();
  if (ok) {
    for (uint32_t j = t; j < uint32_t(gones); j += kPlanThreads) {
      const uint32_t i = owner_of(given_s, a.requests, int32_t(j));
      a.free[n_free + j] = a.table[i * a.table_stride + (j - given_s[i])];
    }
    __syncthreads();  // the stack is whole before pages are taken
    for (uint32_t j = t; j < uint32_t(needs); j += kPlanThreads) {
      const uint32_t i = owner_of(taken_s, a.requests, int32_t(j));
      const uint32_t next = i + 1 < a.requests ? taken_s[i + 1] : uint32_t(needs);
      a.table[i * a.table_stride + (pages_of(end_s[i]) - (next - j))] = a.free[count - 1 - int32_t(j)];
    }
    __syncthreads();
  }
  for (uint32_t r = t; r < write_rows; r += kPlanThreads) write_slot(a, first_s, rows, end_s, r);
}

__global__ __launch_bounds__(256) void slots_kernel(tsa_cache_plan_args a) {
  const uint32_t r = blockIdx.x * 256 + threadIdx.x;
  if (r < a.rows) write_slot(a, a.first, a.requests ? a.first[a.requests] : 0, a.ends, r);
}

// ---- keys and values to their slots and back ----
// Four lanes a block of 32 values, 8 each. kVector: rows whose pieces of 8 values start 16-byte aligned.
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
struct RowPiece {  // piece j of block b of head h of k (0) or v (1) of token t
  uint32_t t, which, h, b, j;
  bool on;
};
__device__ __forceinline__ RowPiece row_piece(const tsa_cache& c, uint32_t tokens) {
  const uint64_t i = uint64_t(blockIdx.x) * 256 + threadIdx.x;
  const uint32_t nb = c.head_dim / 32, row = 2 * c.kv_heads * nb;
  RowPiece p;
  const uint64_t block = i >> 2;
  p.j = uint32_t(i) & 3u;
  p.t = uint32_t(block / row);
  uint32_t in = uint32_t(block % row);
  p.b = in % nb;
  in /= nb;
  p.h = in % c.kv_heads;
  p.which = in / c.kv_heads;
  p.on = p.t < tokens;
  return p;
}
__device__ __forceinline__ BlockPlace place_of(const tsa_cache& c, uint32_t slot, const RowPiece& p) {
  return {static_cast<unsigned char*>(c.pages) + (uint64_t(slot / kPage) * c.kv_heads + p.h) * (72 * c.head_dim), slot % kPage, c.head_dim / 32, p.b};
}

template <class T>
__global__ __launch_bounds__(256) void store_kernel(tsa_cache c, tsa_cache_rows_args a, bool vector) {
  const RowPiece p = row_piece(c, a.tokens);
  const uint32_t slot = p.on ? uint32_t(a.slots[p.t]) : ~0u;
  if (slot >= c.n_pages * kPage) return;  // (a block's four lanes go together)
  const tsa_heads& h = p.which ? a.v : a.k;
  const bits8 raw = load8(h, uint64_t(p.t) * h.token_stride + uint64_t(p.h) * h.head_stride + p.b * 32 + p.j * 8, vector);
  float x[8], top = 0.0f;
  bool finite = true;
  float big = 0.0f;  // the value of the largest size, the first of equal ones
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    x[i] = T::up(raw[i]);
    finite = finite && fabsf(x[i]) < INFINITY;
    if (fabsf(x[i]) > top) top = fabsf(x[i]), big = x[i];
  }
#pragma unroll
  for (int s = 1; s < 4; s <<= 1) {
    const float other = __shfl_xor(big, s, 64);
    finite = finite & (__shfl_xor(int(finite), s, 64) != 0);
    const bool lower = (p.j & s) != 0;  // the other lane's values stand before this one's
    if (fabsf(other) > fabsf(big) || (lower && fabsf(other) == fabsf(big))) big = other;
  }
  // (-big / 8 is exact; a scale beyond half precision is an infinity and 0 times it is NaN, as it should be)
  const u16 scale = finite ? F16::down(big * -0.125f) : u16(0x7E00);
  const float step = F16::up(scale);
  uint32_t lo = 0, hi = 0;  // 8 half bytes, one a byte
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    // The quotient of a 16-bit value and a half-precision step is no nearer than 2^-15 of itself to a border between two steps
    // unless it is on it, so that its rounding to 32 bits takes none over.
    float q = step == 0.0f || !finite ? 0.0f : rintf(x[i] / step);
    q = fminf(fmaxf(q, -8.0f), 7.0f);
    const uint32_t n = uint32_t(int(q) + 8);
    if (i < 4) lo |= n << (8 * i);
    else hi |= n << (8 * (i - 4));
  }
  // values 16.. of the block go to the high halves of bytes 0..
  lo |= __shfl_xor(lo, 2, 64) << 4;
  hi |= __shfl_xor(hi, 2, 64) << 4;
  const BlockPlace at = place_of(c, slot, p);
  if (p.j == 3) *at.scale(p.which) = scale;
  if (p.j >= 2) return;
  if (p.which) {
    *reinterpret_cast<uint2*>(at.value_bytes() + 8 * p.j) = uint2{lo, hi};
  } else {
    *reinterpret_cast<uint32_t*>(at.key_word(2 * p.j)) = lo;
    *reinterpret_cast<uint32_t*>(at.key_word(2 * p.j + 1)) = hi;
  }
}

template <class T>
__global__ __launch_bounds__(256) void load_kernel(tsa_cache c, tsa_cache_rows_args a, bool vector) {
  const RowPiece p = row_piece(c, a.tokens);
  const uint32_t slot = p.on ? uint32_t(a.slots[p.t]) : ~0u;
  if (slot >= c.n_pages * kPage) return;
  const BlockPlace at = place_of(c, slot, p);
  uint2 w;
  const uint32_t half = p.j & 1u;
  if (p.which) w = *reinterpret_cast<const uint2*>(at.value_bytes() + 8 * half);
  else w = uint2{*reinterpret_cast<const uint32_t*>(at.key_word(2 * half)), *reinterpret_cast<const uint32_t*>(at.key_word(2 * half + 1))};
  const float step = F16::up(*at.scale(p.which));
  bits8 out;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t n = ((i < 4 ? w.x : w.y) >> (8 * (i & 3) + (p.j >= 2 ? 4 : 0))) & 15u;
    out[i] = T::down(float(int(n) - 8) * step);
  }
  const tsa_heads& h = p.which ? a.v : a.k;
  u16* to = static_cast<u16*>(h.p) + uint64_t(p.t) * h.token_stride + uint64_t(p.h) * h.head_stride + p.b * 32 + p.j * 8;
  if (vector) {
    *reinterpret_cast<bits8*>(to) = out;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) to[i] = out[i];
  }
}

uint32_t row_grid(const tsa_cache& c, uint32_t tokens) {
  return uint32_t((uint64_t(tokens) * 2 * c.kv_heads * (c.head_dim / 32) * 4 + 255) / 256);
}

}  // namespace
}  // namespace op

int launch_cache_plan(const tsa_cache_plan_args& a, hipStream_t stream) {
  const bool one = a.rows <= op::kPlanRows;
  hipLaunchKernelGGL(op::plan_kernel, dim3(1), dim3(op::kPlanThreads), 0, stream, a, one ? a.rows : 0u);
  if (!one) hipLaunchKernelGGL(op::slots_kernel, dim3((a.rows + 255) / 256), dim3(256), 0, stream, a);
  return int(hipGetLastError());
}

int launch_cache_slots(const tsa_cache_plan_args& a, hipStream_t stream) {
  hipLaunchKernelGGL(op::slots_kernel, dim3((a.rows + 255) / 256), dim3(256), 0, stream, a);
  return int(hipGetLastError());
}

int launch_cache_store(const tsa_cache& c, const tsa_cache_rows_args& a, hipStream_t stream) {
  const bool vector = op::vector_heads(a.k) && op::vector_heads(a.v);
  const dim3 grid(op::row_grid(c, a.tokens));
  if (a.type == TSA_BF16) hipLaunchKernelGGL(op::store_kernel<op::Bf16>, grid, dim3(256), 0, stream, c, a, vector);
  else hipLaunchKernelGGL(op::store_kernel<op::F16>, grid, dim3(256), 0, stream, c, a, vector);
  return int(hipGetLastError());
}

int launch_cache_load(const tsa_cache& c, const tsa_cache_rows_args& a, hipStream_t stream) {
  const bool vector = op::vector_heads(a.k) && op::vector_heads(a.v);
  const dim3 grid(op::row_grid(c, a.tokens));
  if (a.type == TSA_BF16) hipLaunchKernelGGL(op::load_kernel<op::Bf16>, grid, dim3(256), 0, stream, c, a, vector);
  else hipLaunchKernelGGL(op::load_kernel<op::F16>, grid, dim3(256), 0, stream, c, a, vector);
  return int(hipGetLastError());
}

}  // namespace tsa
