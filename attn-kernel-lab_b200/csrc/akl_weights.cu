// Attention weights of an extend: weights[i] (+)= sum over rows t and q heads h with i <= prefix + t of
// 2^(c <q[t][h], k_i> - lse[t][h]), c = sm_scale log2 e.
#include <cstring>

#include "akl_common.cuh"
#include "akl_sm100_ptx.cuh"

namespace akl {

namespace {

constexpr int kMaxGroup = 8;
constexpr float kLog2e = 1.4426950408889634f;

int weights_layout(const akl_weights_plan_t& p, akl_weights_layout_t* o) {
  if (p.max_kv_len < 1 || p.max_q_len < 1 || p.q_heads < 1 || p.kv_heads < 1) return AKL_ERR_INVALID;
  if (p.q_heads % p.kv_heads || p.q_heads / p.kv_heads > kMaxGroup) return AKL_ERR_UNSUPPORTED;
  std::memset(o, 0, sizeof(*o));
  o->total_bytes = 1024;
  return AKL_OK;
}

// One warp per position, a lane eight channels.
template <int KV>
__global__ void __launch_bounds__(256) extend_weights_kernel(akl_weights_t c) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, group = c.q_heads / c.kv_heads;
  const int i = blockIdx.x * 8 + warp;
  if (i >= c.N) return;
  const long long slot = load_index(c.idx, c.idx_dtype, i);
  float total = 0.f;
  for (int j = 0; slot >= 0 && slot < c.pool_rows && j < c.kv_heads; ++j) {
    float k[8];
    unpack8<KV>(*reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(c.k_pool) + slot * c.k_stride + j * 256 + lane * 8), k);
    float head = 0.f;
    for (int t = max(0, i - c.prefix); t < c.T; ++t) {
      float part = 0.f;
      for (int h = j * group; h < (j + 1) * group; ++h) {
        float q[8], x = 0.f;
        unpack8<AKL_KV_BF16>(*reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(c.q) + t * c.q_stride + h * 256 + lane * 8), q);
#pragma unroll
        for (int e = 0; e < 8; ++e) x = fmaf(q[e], k[e], x);
#pragma unroll
        for (int s = 16; s > 0; s >>= 1) x += __shfl_xor_sync(0xffffffffu, x, s);
        const float lse = c.lse[static_cast<long long>(t) * c.q_heads + h];
        if (!isinf(lse)) part += exp2f(fmaf(x, c.sm_scale * kLog2e, -lse));
      }
      head += part;
    }
    total += head;
  }
  if (lane == 0) c.weights[i] = c.weight_decay == 0.f ? total : fmaf(c.weight_decay, c.weights[i], total);
}

int check_weights(const akl_weights_t* c, akl_weights_layout_t* L) {
  if (c == nullptr || c->q == nullptr || c->k_pool == nullptr || c->idx == nullptr || c->lse == nullptr ||
      c->weights == nullptr || c->workspace == nullptr)
    return AKL_ERR_INVALID;
  if (c->T < 1 || c->N < 1 || c->q_heads < 1 || c->kv_heads < 1 || c->pool_rows < 1) return AKL_ERR_INVALID;
  if (c->prefix < 0 || c->prefix > c->N - c->T) return AKL_ERR_INVALID;
  if (c->kv_dtype != AKL_KV_BF16 && c->kv_dtype != AKL_KV_FP16) return AKL_ERR_INVALID;
  if (!known_index(c->idx_dtype)) return AKL_ERR_INVALID;
  if (!(c->sm_scale > 0.f) || !(c->weight_decay >= 0.f && c->weight_decay <= 1.f)) return AKL_ERR_INVALID;
  if (c->q_heads % c->kv_heads || c->q_heads / c->kv_heads > kMaxGroup) return AKL_ERR_UNSUPPORTED;
  if (c->kv_heads != 1 && c->kv_heads != 2 && c->kv_heads != 4 && c->kv_heads != 8) return AKL_ERR_UNSUPPORTED;
  if (c->k_stride < c->kv_heads * 256 || c->q_stride < c->q_heads * 256) return AKL_ERR_INVALID;
  int rc = weights_layout(c->plan, L);
  if (rc != AKL_OK) return rc;
  if (c->workspace_bytes < L->total_bytes || c->N > c->plan.max_kv_len || c->T > c->plan.max_q_len ||
      c->q_heads != c->plan.q_heads || c->kv_heads != c->plan.kv_heads)
    return AKL_ERR_CAPACITY;
  const uintptr_t mask = reinterpret_cast<uintptr_t>(c->q) | reinterpret_cast<uintptr_t>(c->k_pool);
  if ((mask & 15u) || ((c->k_stride | c->q_stride) & 7) || (reinterpret_cast<uintptr_t>(c->workspace) & 1023u))
    return AKL_ERR_ALIGN;
  return AKL_OK;
}

}  // namespace
}  // namespace akl

using namespace akl;

extern "C" {

int akl_weights_layout(const akl_weights_plan_t* plan, akl_weights_layout_t* out) {
  if (plan == nullptr || out == nullptr) return AKL_ERR_INVALID;
  return weights_layout(*plan, out);
}

int akl_extend_weights(const akl_weights_t* c, void* stream) {
  akl_weights_layout_t L;
  int rc = check_weights(c, &L);
  if (rc != AKL_OK) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const unsigned blocks = (static_cast<unsigned>(c->N) + 7) / 8;
  if (c->kv_dtype == AKL_KV_BF16) extend_weights_kernel<AKL_KV_BF16><<<blocks, 256, 0, s>>>(*c);
  else extend_weights_kernel<AKL_KV_FP16><<<blocks, 256, 0, s>>>(*c);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) { note_cuda_error(e, "extend_weights_kernel"); return AKL_ERR_CUDA; }
  return AKL_OK;
}

}  // extern "C"
