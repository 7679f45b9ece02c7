// Merge of per-split partial attention states for a KV-axis split of one long request:
//   lse = log2 sum_i 2^lse_i,   O = sum_i 2^(lse_i - lse) O_i.
// Each O_i is a normalised BF16 output that already carries the V channel mean; the weights
// sum to one, so the mean is counted once.  The reference exposes the base-2 LSE for this
// composition (docs/OPERATOR_CONTRACT.md:57,238-242) but has no merge of its own.
//
// And the step that makes an LSE over centred keys one over the pool's own, so that it can be composed with others.
//
// HBM-bound: one warp per (row, head) vector of 256 channels, one 16-byte load per lane per
// part, one 16-byte store.  The part pointers may address memory that a collective has
// already landed in this GPU's HBM; the kernel issues plain loads only.
#include "akl_common.cuh"

namespace akl {

namespace {

constexpr int kMaxParts = 64;

__global__ void __launch_bounds__(256) merge_states_kernel(akl_merge_t m) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long row = static_cast<long long>(blockIdx.x) * 8 + warp;
  if (row >= m.rows) return;
  float mx = -INFINITY;
  for (int i = 0; i < m.nparts; ++i) mx = fmaxf(mx, m.parts_lse[i][row]);
  float acc[8];
#pragma unroll
  for (int c = 0; c < 8; ++c) acc[c] = 0.f;
  float den = 0.f;
  if (mx == -INFINITY) {
    // no split saw a key for this row: every part holds the V mean; pass part 0 through
    const uint4 raw = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(m.parts_o[0]) + row * kD + lane * 8);
    *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(m.out) + row * kD + lane * 8) = raw;
    if (m.lse_out != nullptr && lane == 0) m.lse_out[row] = -INFINITY;
    return;
  }
  for (int i = 0; i < m.nparts; ++i) {
    const float li = m.parts_lse[i][row];
    if (li == -INFINITY) continue;
    const float w = exp2f(li - mx);
    den += w;
    const uint4 raw = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(m.parts_o[i]) + row * kD + lane * 8);
    float x[8];
    unpack8<AKL_KV_BF16>(raw, x);
#pragma unroll
    for (int c = 0; c < 8; ++c) acc[c] = fmaf(w, x[c], acc[c]);
  }
  const float inv = 1.0f / den;
  uint32_t pk[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    __nv_bfloat162 t = __floats2bfloat162_rn(acc[2 * e] * inv, acc[2 * e + 1] * inv);
    pk[e] = *reinterpret_cast<uint32_t*>(&t);
  }
  *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(m.out) + row * kD + lane * 8) = make_uint4(pk[0], pk[1], pk[2], pk[3]);
  if (m.lse_out != nullptr && lane == 0) m.lse_out[row] = mx + log2f(den);
}

// lse[t][h] += c <q[t][h], kmean[h / group]>, c = sm_scale log2 e: from the log-sum-exp over the centred keys, which is
// what the attention launch sums, to that over the pool's own.  512 bytes of q per (row, head), read once: 25 MB and
// 10 to 12 us (2.3 TB/s, its launch included) for 2048 rows of 24 heads, beside the 182 us of their extend over 4096
// positions.  The mean is taken before the rotation, so it meets the q of the call.
__device__ __forceinline__ void add_mean_term(const Geom& g, long long row, int lane) {
  const int head = static_cast<int>(row % g.Hq);
  const uint4 raw = __ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(g.q) + row * kD + lane * 8));
  const float4* mean = reinterpret_cast<const float4*>(g.kmean + head / (g.Hq / g.Hkv) * kD + lane * 8);
  const float4 m0 = mean[0], m1 = mean[1];
  float x[8];
  unpack8<AKL_KV_BF16>(raw, x);
  float sum = fmaf(x[0], m0.x, fmaf(x[1], m0.y, fmaf(x[2], m0.z, x[3] * m0.w))) +
              fmaf(x[4], m1.x, fmaf(x[5], m1.y, fmaf(x[6], m1.z, x[7] * m1.w)));
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, s);
  if (lane == 0) g.lse_out[row] = fmaf(g.sm_scale * 1.4426950408889634f, sum, g.lse_out[row]);
}

__global__ void __launch_bounds__(256) pool_lse_kernel(const Geom g) {
  const long long row = static_cast<long long>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  if (row < static_cast<long long>(g.T) * g.Hq) add_mean_term(g, row, threadIdx.x & 31);
}

// The same for a batch: groups of eight (row, head) pairs of all requests, dealt to the CTAs in turn.
__global__ void __launch_bounds__(256) pool_lse_batch_kernel(const BatchRef b) {
  const int n = batch_header(b)->n_requests;
  const Geom* geoms = reinterpret_cast<const Geom*>(b.table + b.off_geoms);
  long long turn = blockIdx.x;                       // groups from here to this CTA's next one
  for (int r = 0; r < n; ++r) {
    const Geom& g = geoms[r];
    const long long rows = static_cast<long long>(g.T) * g.Hq, groups = (rows + 7) / 8;
    for (; turn < groups; turn += gridDim.x) {
      const long long row = turn * 8 + (threadIdx.x >> 5);
      if (g.lse_out != nullptr && row < rows) add_mean_term(g, row, threadIdx.x & 31);
    }
    turn -= groups;
  }
}

}  // namespace

int launch_pool_lse(const Geom& g, cudaStream_t s) {
  if (!(g.flags & AKL_FLAG_POOL_LSE) || !(g.flags & AKL_FLAG_CENTER_K) || g.lse_out == nullptr) return AKL_OK;
  const long long blocks = (static_cast<long long>(g.T) * g.Hq + 7) / 8;
  if (blocks >= (1ll << 31)) return AKL_ERR_UNSUPPORTED;
  pool_lse_kernel<<<static_cast<unsigned>(blocks), 256, 0, s>>>(g);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) { note_cuda_error(e, "pool_lse_kernel"); return AKL_ERR_CUDA; }
  return AKL_OK;
}

int launch_batch_pool_lse(const BatchRef& b, int sm_count, cudaStream_t s) {
  pool_lse_batch_kernel<<<static_cast<unsigned>(sm_count * 8), 256, 0, s>>>(b);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) { note_cuda_error(e, "pool_lse_batch_kernel"); return AKL_ERR_CUDA; }
  return AKL_OK;
}

int launch_merge(const akl_merge_t& m, cudaStream_t s) {
  if (m.nparts < 1 || m.nparts > kMaxParts || m.rows < 1) return AKL_ERR_INVALID;
  const unsigned blocks = static_cast<unsigned>((static_cast<long long>(m.rows) + 7) / 8);
  merge_states_kernel<<<blocks, 256, 0, s>>>(m);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) { note_cuda_error(e, "merge_states_kernel"); return AKL_ERR_CUDA; }
  return AKL_OK;
}

}  // namespace akl
