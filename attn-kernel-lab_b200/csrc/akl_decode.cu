// Decode attention: one new token per request over the paged pool.
//   x = c <q, k>, c = sm_scale log2 e;  m = max x;  l = sum 2^(x - m);  out = sum 2^(x - m) v / l;
//   lse = m + log2 l;   weights += sum over the q heads of 2^(x - lse)
#include <cstring>

#include "akl_common.cuh"
#include "akl_sm100_ptx.cuh"

namespace akl {

namespace {

constexpr int kChunk = 64;          // positions per chunk of recorded scores
constexpr int kMaxGroup = 8;        // query heads per kv head
constexpr float kLog2e = 1.4426950408889634f;

inline uint64_t align1k(uint64_t x) { return (x + 1023) / 1024 * 1024; }

int decode_layout(const akl_decode_plan_t& p, akl_decode_layout_t* o) {
  if (p.max_requests < 1 || p.q_heads < 1 || p.kv_heads < 1 || p.max_weight_tokens < 0) return AKL_ERR_INVALID;
  if (p.q_heads % p.kv_heads || p.q_heads / p.kv_heads > kMaxGroup) return AKL_ERR_UNSUPPORTED;
  std::memset(o, 0, sizeof(*o));
  uint64_t off = 0;
  o->off_status = off;
  off += 1024;
  o->off_parts = off;
  o->off_lse = off;
  off += align1k(static_cast<uint64_t>(p.max_requests) * p.q_heads * 4);
  o->off_scores = off;
  o->total_bytes = off;
  return AKL_OK;
}

__device__ __forceinline__ void request_of(const akl_decode_t& c, int b, long long& row, int& n) {
  row = c.rows != nullptr ? load_index(c.rows, c.rows_dtype, b) : b;
  long long len = load_index(c.kv_lens, c.lens_dtype, b);
  len = len < 0 ? 0 : (len > c.table_width ? c.table_width : len);
  if (row < 0 || row >= c.table_rows) { row = 0; len = 0; }
  n = static_cast<int>(len);
}

// One CTA per (request, kv head); a warp takes every eighth position, a lane eight channels.
template <int KV>
__global__ void __launch_bounds__(256) decode_kernel(akl_decode_t c, float* lse_ws) {
  __shared__ float sm_m[8][kMaxGroup], sm_l[8][kMaxGroup];
  __shared__ float sm_o[8][256];
  const int b = blockIdx.x, j = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int group = c.q_heads / c.kv_heads;
  long long row;
  int n;
  request_of(c, b, row, n);
  float q[kMaxGroup][8], o[kMaxGroup][8], m[kMaxGroup], l[kMaxGroup];
#pragma unroll
  for (int h = 0; h < kMaxGroup; ++h) {
    m[h] = -INFINITY;
    l[h] = 0.f;
    if (h < group) {
      const uint4 raw = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(c.q) + b * c.q_stride + (j * group + h) * 256 + lane * 8);
      unpack8<AKL_KV_BF16>(raw, q[h]);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      q[h][i] = h < group ? q[h][i] * (c.sm_scale * kLog2e) : 0.f;
      o[h][i] = 0.f;
    }
  }
  for (int i = warp; i < n; i += 8) {
    const long long slot = load_index(c.page_table, c.idx_dtype, row * c.table_stride + i);
    if (slot < 0 || slot >= c.pool_rows) continue;
    float k[8], v[8];
    unpack8<KV>(*reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(c.k_pool) + slot * c.k_stride + j * 256 + lane * 8), k);
    unpack8<KV>(*reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(c.v_pool) + slot * c.v_stride + j * 256 + lane * 8), v);
#pragma unroll
    for (int h = 0; h < kMaxGroup; ++h) {
      if (h >= group) break;
      float x = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) x = fmaf(q[h][e], k[e], x);
#pragma unroll
      for (int s = 16; s > 0; s >>= 1) x += __shfl_xor_sync(0xffffffffu, x, s);
      const float top = fmaxf(m[h], x), a = exp2f(m[h] - top), p = exp2f(x - top);
      m[h] = top;
      l[h] = l[h] * a + p;
#pragma unroll
      for (int e = 0; e < 8; ++e) o[h][e] = fmaf(p, v[e], o[h][e] * a);
    }
  }
  for (int h = 0; h < group; ++h) {
    float mh = 0.f, lh = 0.f;
#pragma unroll
    for (int k = 0; k < kMaxGroup; ++k)
      if (k == h) { mh = m[k]; lh = l[k]; }
    if (lane == 0) { sm_m[warp][h] = mh; sm_l[warp][h] = lh; }
    __syncthreads();
    float top = -INFINITY, total = 0.f;
    for (int w = 0; w < 8; ++w) top = fmaxf(top, sm_l[w][h] != 0.f ? sm_m[w][h] : -INFINITY);
    for (int w = 0; w < 8; ++w) total += sm_l[w][h] != 0.f ? sm_l[w][h] * exp2f(sm_m[w][h] - top) : 0.f;
    const float f = lh != 0.f ? exp2f(mh - top) : 0.f;
#pragma unroll
    for (int k = 0; k < kMaxGroup; ++k)
      if (k == h) {
#pragma unroll
        for (int e = 0; e < 8; ++e) sm_o[warp][lane * 8 + e] = lh != 0.f ? o[k][e] * f : 0.f;
      }
    __syncthreads();
    float sum = 0.f;
    for (int w = 0; w < 8; ++w) sum += sm_o[w][threadIdx.x];
    const int head = j * group + h;
    const bool none = total == 0.f;
    reinterpret_cast<__nv_bfloat16*>(c.out)[(static_cast<long long>(b) * c.q_heads + head) * 256 + threadIdx.x] =
        __float2bfloat16_rn(none ? 0.f : sum / total);
    if (threadIdx.x == 0) {
      const float lse = none ? -INFINITY : top + log2f(total);
      if (c.lse_out != nullptr) c.lse_out[b * c.q_heads + head] = lse;
      lse_ws[b * c.q_heads + head] = lse;
    }
    __syncthreads();
  }
}

// One warp per position.
template <int KV>
__global__ void __launch_bounds__(256) decode_weights_kernel(akl_decode_t c, const float* lse_ws) {
  const int b = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, group = c.q_heads / c.kv_heads;
  long long row;
  int n;
  request_of(c, b, row, n);
  for (int i = blockIdx.y * 8 + warp; i < n; i += gridDim.y * 8) {
    const long long slot = load_index(c.page_table, c.idx_dtype, row * c.table_stride + i);
    float total = 0.f;
    for (int j = 0; slot >= 0 && slot < c.pool_rows && j < c.kv_heads; ++j) {
      float k[8];
      unpack8<KV>(*reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(c.k_pool) + slot * c.k_stride + j * 256 + lane * 8), k);
      for (int h = j * group; h < (j + 1) * group; ++h) {
        float q[8], x = 0.f;
        unpack8<AKL_KV_BF16>(*reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(c.q) + b * c.q_stride + h * 256 + lane * 8), q);
#pragma unroll
        for (int e = 0; e < 8; ++e) x = fmaf(q[e] * (c.sm_scale * kLog2e), k[e], x);
#pragma unroll
        for (int s = 16; s > 0; s >>= 1) x += __shfl_xor_sync(0xffffffffu, x, s);
        total += exp2f(x - lse_ws[b * c.q_heads + h]);
      }
    }
    float* w = c.weights + row * c.weights_stride + i;
    if (lane == 0) *w = c.weight_decay == 0.f ? total : fmaf(c.weight_decay, *w, total);
  }
}

int check_decode(const akl_decode_t* c, akl_decode_layout_t* L) {
  if (c == nullptr || c->q == nullptr || c->k_pool == nullptr || c->v_pool == nullptr || c->page_table == nullptr ||
      c->kv_lens == nullptr || c->out == nullptr || c->workspace == nullptr)
    return AKL_ERR_INVALID;
  if (c->batch < 1 || c->q_heads < 1 || c->kv_heads < 1 || c->table_rows < 1 || c->table_width < 1 || c->pool_rows < 1)
    return AKL_ERR_INVALID;
  if (c->kv_dtype != AKL_KV_BF16 && c->kv_dtype != AKL_KV_FP16) return AKL_ERR_INVALID;
  if (!known_index(c->idx_dtype) || !known_index(c->lens_dtype) || !known_index(c->rows_dtype)) return AKL_ERR_INVALID;
  if (!(c->sm_scale > 0.f) || !(c->weight_decay >= 0.f && c->weight_decay <= 1.f)) return AKL_ERR_INVALID;
  if (c->rows == nullptr && c->table_rows < c->batch) return AKL_ERR_INVALID;
  if (c->q_heads % c->kv_heads || c->q_heads / c->kv_heads > kMaxGroup) return AKL_ERR_UNSUPPORTED;
  if (c->kv_heads != 1 && c->kv_heads != 2 && c->kv_heads != 4 && c->kv_heads != 8) return AKL_ERR_UNSUPPORTED;
  if (c->k_stride < c->kv_heads * 256 || c->v_stride < c->kv_heads * 256 || c->q_stride < c->q_heads * 256 ||
      c->table_stride < c->table_width)
    return AKL_ERR_INVALID;
  if (c->weights != nullptr && c->weights_stride < c->table_width) return AKL_ERR_INVALID;
  int rc = decode_layout(c->plan, L);
  if (rc != AKL_OK) return rc;
  if (c->workspace_bytes < L->total_bytes || c->batch > c->plan.max_requests || c->q_heads != c->plan.q_heads ||
      c->kv_heads != c->plan.kv_heads || (c->weights != nullptr && c->plan.max_weight_tokens < 1))
    return AKL_ERR_CAPACITY;
  const uintptr_t mask = reinterpret_cast<uintptr_t>(c->q) | reinterpret_cast<uintptr_t>(c->k_pool) |
                         reinterpret_cast<uintptr_t>(c->v_pool) | reinterpret_cast<uintptr_t>(c->out);
  if ((mask & 15u) || ((c->k_stride | c->v_stride | c->q_stride) & 7) || (reinterpret_cast<uintptr_t>(c->workspace) & 1023u))
    return AKL_ERR_ALIGN;
  return AKL_OK;
}

}  // namespace
}  // namespace akl

using namespace akl;

extern "C" {

int akl_decode_layout(const akl_decode_plan_t* plan, akl_decode_layout_t* out) {
  if (plan == nullptr || out == nullptr) return AKL_ERR_INVALID;
  return decode_layout(*plan, out);
}

int akl_paged_decode(const akl_decode_t* c, void* stream) {
  akl_decode_layout_t L;
  int rc = check_decode(c, &L);
  if (rc != AKL_OK) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  float* lse = reinterpret_cast<float*>(static_cast<uint8_t*>(c->workspace) + L.off_lse);
  const dim3 grid(c->batch, c->kv_heads), grid_w(c->batch, 64);
  if (c->kv_dtype == AKL_KV_BF16) decode_kernel<AKL_KV_BF16><<<grid, 256, 0, s>>>(*c, lse);
  else decode_kernel<AKL_KV_FP16><<<grid, 256, 0, s>>>(*c, lse);
  if (c->weights != nullptr) {
    if (c->kv_dtype == AKL_KV_BF16) decode_weights_kernel<AKL_KV_BF16><<<grid_w, 256, 0, s>>>(*c, lse);
    else decode_weights_kernel<AKL_KV_FP16><<<grid_w, 256, 0, s>>>(*c, lse);
  }
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) { note_cuda_error(e, "decode_kernel"); return AKL_ERR_CUDA; }
  return AKL_OK;
}

}  // extern "C"
