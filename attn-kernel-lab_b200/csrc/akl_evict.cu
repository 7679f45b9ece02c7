// Eviction by accumulated weight: the first and last positions of a request and the heaviest of the
// others move to the front of its page-table row in position order.
//
// The weights are compared as 32-bit keys in the order of the floats (NaN as -inf, -0 as 0).  The key
// of the lightest position that stays is found digit by digit, eight bits a pass, from a histogram of
// the keys that share the digits found so far; of the positions with exactly that key the lowest stay.
#include "akl_common.cuh"

namespace akl {

namespace {

constexpr int kThreads = 1024, kWarps = kThreads / 32;

__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) w = -INFINITY;
  w = w + 0.f;
  const uint32_t u = __float_as_uint(w);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// Exclusive count of `flag` before this thread in the CTA, and the total.
__device__ __forceinline__ int cta_rank(bool flag, int* sm, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const unsigned ballot = __ballot_sync(0xffffffffu, flag);
  if (lane == 0) sm[warp] = __popc(ballot);
  __syncthreads();
  if (warp == 0) {
    const int v = sm[lane];
    int s = v;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, s, d);
      if (lane >= d) s += up;
    }
    sm[lane] = s - v;
    if (lane == 31) sm[32] = s;
  }
  __syncthreads();
  const int rank = sm[warp] + __popc(ballot & ((1u << lane) - 1u));
  total = sm[32];
  __syncthreads();
  return rank;
}

// One CTA per request.
template <typename Slot>
__global__ void __launch_bounds__(kThreads) evict_kernel(akl_evict_t c) {
  __shared__ int sm_scan[33];
  __shared__ int hist[256];
  __shared__ uint32_t sm_prefix;
  __shared__ int sm_need;
  const int b = blockIdx.x, tid = threadIdx.x;
  const long long row = c.rows != nullptr ? load_index(c.rows, c.rows_dtype, b) : b;
  long long len = load_index(c.kv_lens, c.lens_dtype, b);
  len = len < 0 ? 0 : (len > c.table_width ? c.table_width : len);
  if (row < 0 || row >= c.table_rows) len = 0;
  const int n = static_cast<int>(len);
  const bool full = n > c.keep;
  const Slot* slots = static_cast<const Slot*>(c.page_table) + row * c.table_stride;
  const float* weights = c.weights + row * c.weights_stride;
  Slot* slots_out = static_cast<Slot*>(c.page_table_out) + row * c.table_out_stride;
  float* weights_out = c.weights_out + row * c.weights_out_stride;
  Slot* freed = static_cast<Slot*>(c.freed) + b * c.freed_stride;

  uint32_t threshold = 0;
  int need = c.keep - c.first - c.last;         // how many of the middle stay
  if (full && need > 0) {
    if (tid == 0) { sm_prefix = 0; sm_need = need; }
    for (int shift = 24; shift >= 0; shift -= 8) {
      if (tid < 256) hist[tid] = 0;
      __syncthreads();
      const uint32_t prefix = sm_prefix, mask = shift == 24 ? 0u : ~0u << (shift + 8);
      for (int i = c.first + tid; i < n - c.last; i += kThreads) {
        const uint32_t k = weight_key(weights[i]);
        if ((k & mask) == prefix) atomicAdd(&hist[(k >> shift) & 255u], 1);
      }
      __syncthreads();
      if (tid == 0) {
        int left = sm_need, d = 255;
        while (d > 0 && hist[d] < left) left -= hist[d--];
        sm_need = left;
        sm_prefix = prefix | (static_cast<uint32_t>(d) << shift);
      }
      __syncthreads();
    }
    threshold = sm_prefix;
    need = sm_need;                             // how many of those with exactly this key stay
  }
  int stay0 = 0, go0 = 0, equal0 = 0;
  for (int base = 0; base < n; base += kThreads) {
    const int i = base + tid;
    const bool in = i < n;
    const bool middle = in && full && i >= c.first && i < n - c.last;
    const Slot slot = in ? slots[i] : Slot(0);
    const float w = in ? weights[i] : 0.f;
    const uint32_t key = weight_key(w);
    const bool equal = middle && key == threshold;
    int total;
    const int rank = cta_rank(equal, sm_scan, total);
    const bool stay = in && (!middle || (c.keep > c.first + c.last && (key > threshold || (equal && equal0 + rank < need))));
    equal0 += total;
    const int at = cta_rank(stay, sm_scan, total);      // ends with a barrier: the chunk is in registers
    if (stay) { slots_out[stay0 + at] = slot; weights_out[stay0 + at] = w; }
    const int before = min(tid, n - base) - at;
    if (in && !stay) freed[go0 + before] = slot;
    stay0 += total;
    go0 += min(kThreads, n - base) - total;
    __syncthreads();
  }
  for (int i = stay0 + tid; i < n; i += kThreads) weights_out[i] = 0.f;
  if (tid == 0) {
    if (c.lens_dtype == AKL_IDX_I64) static_cast<long long*>(c.kv_lens_out)[b] = stay0;
    else static_cast<int*>(c.kv_lens_out)[b] = stay0;
    c.freed_lens[b] = go0;
  }
}

}  // namespace
}  // namespace akl

using namespace akl;

extern "C" int akl_evict_lightest(const akl_evict_t* c, void* stream) {
  if (c == nullptr || c->page_table == nullptr || c->weights == nullptr || c->kv_lens == nullptr ||
      c->page_table_out == nullptr || c->weights_out == nullptr || c->kv_lens_out == nullptr || c->freed == nullptr ||
      c->freed_lens == nullptr)
    return AKL_ERR_INVALID;
  if (c->batch < 1 || c->table_rows < 1 || c->table_width < 1 || c->keep < 1 || c->first < 0 || c->last < 0)
    return AKL_ERR_INVALID;
  if (static_cast<int64_t>(c->first) + c->last > c->keep) return AKL_ERR_INVALID;
  if (!known_index(c->idx_dtype) || !known_index(c->lens_dtype) || !known_index(c->rows_dtype)) return AKL_ERR_INVALID;
  if (c->rows == nullptr && c->table_rows < c->batch) return AKL_ERR_INVALID;
  if (c->table_stride < c->table_width || c->table_out_stride < c->table_width || c->weights_stride < c->table_width ||
      c->weights_out_stride < c->table_width || c->freed_stride < c->freed_width)
    return AKL_ERR_INVALID;
  if (c->freed_width < c->table_width - c->keep) return AKL_ERR_CAPACITY;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (c->idx_dtype == AKL_IDX_I64) evict_kernel<long long><<<c->batch, kThreads, 0, s>>>(*c);
  else evict_kernel<int><<<c->batch, kThreads, 0, s>>>(*c);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) { note_cuda_error(e, "evict_kernel"); return AKL_ERR_CUDA; }
  return AKL_OK;
}
