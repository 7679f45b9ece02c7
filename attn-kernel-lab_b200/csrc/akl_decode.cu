// Decode attention: one new token per request over the paged pool.
//   x = c <q, k>, c = sm_scale log2 e;  m = max x;  l = sum 2^(x - m);  out = sum 2^(x - m) v / l;
//   lse = m + log2 l;   weights (+)= sum over the q heads of 2^(x - lse)
//
// K and V are read once, 1 KiB per position and kv head for 4 * 256 * group operations: HBM bound for
// every group up to 8.  So the kernel is a copy pipeline with arithmetic that keeps out of its way:
//
//   * one CTA per SM; the positions of all requests, cut into tiles of 64 KiB of K and V, form one
//     sequence of which every CTA takes an equal share, whatever the lengths (they are read here, on
//     the device).  A CTA meets a run of requests: those it holds whole it finishes itself, of the
//     first and the last it may hold a part, whose (m, l, unnormalised out) goes to the workspace for
//     the join launch.  No atomics: partial states are joined in position order.
//   * four producer warps gather the rows (the kv heads of a position are neighbours in the pool: 2 KiB
//     at four heads) into a ring of three tiles with 16-byte asynchronous copies, 512 bytes a warp
//     instruction, with the page-table entries four tiles ahead.  Rows lie 16 bytes off a multiple of 128 in
//     shared memory, so that matrix loads meet no bank twice.  (Bulk copies of a row each were measured
//     first: about 75 cycles of the copy unit apiece, 94 us for 136 MB in rows of 512 bytes.)
//   * eight warps: four (kv head, 16 positions) tasks times two halves of the channels.  A pair of warps
//     forms the scores, half the products each, S^T = K Q^T as m16n8k16 with the positions on M and the (up to eight) q
//     heads of the kv head on N -- with the heads on M half to three quarters of the tensor work would
//     be padding.  Out^T = V^T P^T takes P^T in the operand layout that an 8x8 transpose of the score
//     fragment gives, so P never touches shared memory.  mma.sync, not tcgen05: 8192
//     multiply-adds per position and kv head (2048 for eight heads' scores, three times that for the parts of P; two
//     times for an FP16 pool) against the ~43 cycles that its bytes take per SM (the tensor pipe is 12 to 17 % busy);
//     tcgen05's 128 rows would be 6 to 25 % filled and its TMEM round trip longer.
//
// Measured (a call in a CUDA graph): 64 ragged requests, 2.2 GB of K and V, 359 us, 95 % of the
// copy bandwidth; one request of 139264 positions, 571 MB, 103 to 106 us; 8 requests, 137 MB, 36 us; one of 1000, 4 MB,
// 9.0 us.  The short ones are bound by three dependent trips to memory (lengths, page table, rows) and the join,
// the long ones by HBM and by the SMs that get their equal share up to 8 % later than the median.
//
// Rounding: scores, m, l and both sums are 32-bit, and so is P: it enters the second product as a sum of three BF16
// numbers, or of two FP16 ones, 24 and 22 bits.  (With one the error of the outputs was 1.77e-3 instead of 1.66e-3, which
// is the BF16 rounding of the result; with two of BF16, 17 bits, one output in 1000 was not the correctly rounded one,
// with three one in 4000.  The third takes 1 % of the time.)  The tensor pipe cuts its
// 32-bit sums off where it should round, always towards zero, and over a thousand tiles that adds up; so it sums
// within a tile only, from zero, and the tiles are added up by FMAs that round.  (Distance of the outputs from the
// correctly rounded ones in the long cases: 1.3e-4 to 1.5e-4 with one running sum and two parts, below 0.5e-4 now, for 0 to
// 0.6 % of the time.)  For an FP16 pool P is
// scaled by 2^14, so that small probabilities stay normal numbers, and Q (BF16) is brought to FP16 by the power
// of two of its row's largest element: exact down to 2^-17 of that element, 2^-25 of it below.
#include <algorithm>
#include <atomic>
#include <cstring>

#include "akl_common.cuh"
#include "akl_sm100_ptx.cuh"

namespace akl {

namespace {

using namespace ptx;

constexpr int kChunk = 64;          // positions per chunk of recorded scores
constexpr int kMaxGroup = 8;        // query heads per kv head
constexpr int kMaxCtas = 160;       // CTAs whose partial states the workspace holds (two each)
constexpr int kStages = 3;
constexpr int kWarps = 8;           // consumers
constexpr int kProducers = 4;       // and the warps that gather for them
constexpr int kThreads = (kWarps + kProducers) * 32;
constexpr int kAhead = 4;           // tiles whose page-table entries are on their way
constexpr float kLog2e = 1.4426950408889634f;
constexpr long long kWaitCycles = 4000000000ll;      // ~2 s: a wait that long is a defect

inline uint64_t align1k(uint64_t x) { return (x + 1023) / 1024 * 1024; }

// Heads per CTA and what follows from them.
template <int HB>
struct Tile {
  static constexpr int kRow = HB * 512;              // bytes of one position's heads in one plane
  static constexpr int kPitch = kRow + 16;
  static constexpr int kPos = 64 / HB;               // positions per tile
  static constexpr int kPlane = kPos * kPitch;
  static constexpr int kStage = 2 * kPlane;
  static constexpr int kRing = kStages * kStage;
  static constexpr int kGroups = 4 / HB;             // 16-position groups of a tile
  static constexpr int kMerge = kGroups > 1 ? 16384 : 0;
  static constexpr int kOffMerge = kRing;
  static constexpr int kOffMl = kOffMerge + kMerge;  // [8 warps][8 heads] {m, l}
  static constexpr int kOffMeet = kOffMl + 512;      // [2][8 warps][32 lanes] float4: half scores of a warp for its partner
  static constexpr int kOwn = kPos / kProducers;     // positions of a tile that one producer warp gathers
  static constexpr int kOffMask = kOffMeet + 8192;      // [kStages][kProducers] u32: which of them are there
  static constexpr int kOffBar = kOffMask + 16 * kStages;
  static constexpr int kSmem = kOffBar + 16 * kStages + 16;
};
static_assert(Tile<1>::kSmem <= 232448 && Tile<2>::kSmem <= 232448 && Tile<4>::kSmem <= 232448, "shared memory");

// Workspace, behind off_parts: who holds which request, then the partial states.
constexpr int kSlotHeads = 4 * kMaxGroup;
inline uint64_t info_bytes(const akl_decode_plan_t& p) { return align1k(static_cast<uint64_t>(p.max_requests) * 2 * 16); }
constexpr uint64_t kMlBytes = static_cast<uint64_t>(2 * kMaxCtas) * kSlotHeads * 8;
constexpr uint64_t kPartBytes = static_cast<uint64_t>(2 * kMaxCtas) * kSlotHeads * 1024;

int decode_layout(const akl_decode_plan_t& p, akl_decode_layout_t* o) {
  if (p.max_requests < 1 || p.q_heads < 1 || p.kv_heads < 1 || p.max_weight_tokens < 0) return AKL_ERR_INVALID;
  if (p.q_heads % p.kv_heads || p.q_heads / p.kv_heads > kMaxGroup) return AKL_ERR_UNSUPPORTED;
  if (p.max_weight_tokens >= (1ll << 40)) return AKL_ERR_UNSUPPORTED;      // beyond any memory, and the bytes stay within 64 bits
  std::memset(o, 0, sizeof(*o));
  uint64_t off = 1024;
  o->off_parts = off;
  off += info_bytes(p) + align1k(kMlBytes) + kPartBytes;
  o->off_lse = off;
  off += align1k(static_cast<uint64_t>(p.max_requests) * p.q_heads * 4);
  o->off_scores = off;
  off += align1k((static_cast<uint64_t>(p.max_weight_tokens) + kChunk - 1) / kChunk * kChunk * p.q_heads * 4);
  o->total_bytes = off;
  return AKL_OK;
}

// CTAs that add a request's weights, 256 positions at a time.
inline int weight_blocks(const akl_decode_t& c) { return c.weights != nullptr ? std::min((c.table_width + 255) / 256, 64) : 0; }

// What the kernels get besides the call.
struct Work {
  int* status;
  int4* info;            // [request][head block] {first slot, first CTA, last CTA, -}
  float2* ml;            // [slot][kSlotHeads]
  float* parts;          // [slot][kSlotHeads][256]
  float* lse;            // [batch][Hq], for the weights
  float* scores;         // [chunk][Hq][64] or NULL
  long long max_chunks;
};

// Cached positions of request b and its table row; 0 where there is nothing to read.
__device__ __forceinline__ int request_of(const akl_decode_t& c, int b, long long& row) {
  row = c.rows != nullptr ? load_index(c.rows, c.rows_dtype, b) : b;
  long long len = load_index(c.kv_lens, c.lens_dtype, b);
  len = len < 0 ? 0 : (len > c.table_width ? c.table_width : len);
  if (row < 0 || row >= c.table_rows) { row = 0; len = 0; }
  return static_cast<int>(len);
}

__device__ __forceinline__ long long warp_sum(long long v) {
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) v += __shfl_xor_sync(0xffffffffu, v, s);
  return v;
}

// A warp's place in the sequence of tiles: request b, head block hb, tile t of nt.  The lengths of 32
// requests at a time are spread over the lanes.
template <int HB>
struct Cursor {
  static constexpr int kPos = Tile<HB>::kPos;
  const akl_decode_t& c;
  const int lane, blocks;           // head blocks
  int base, lane_n;
  long long lane_row;
  int b, n, nt, hb, t;
  long long row, chunk0;            // chunk0: score chunks of the requests before b

  __device__ __forceinline__ Cursor(const akl_decode_t& call, int l) : c(call), lane(l), blocks(call.kv_heads / HB) {}

  __device__ __forceinline__ long long total() const {
    long long tiles = 0;
#pragma unroll 4
    for (int i = lane; i < c.batch; i += 32) {
      long long r;
      tiles += (request_of(c, i, r) + kPos - 1) / kPos;
    }
    return warp_sum(tiles) * blocks;
  }
  __device__ __forceinline__ void window(int at) {
    base = at;
    lane_n = 0;
    lane_row = 0;
    if (at + lane < c.batch) lane_n = request_of(c, at + lane, lane_row);
  }
  __device__ __forceinline__ void take(int i) {
    b = base + i;
    n = __shfl_sync(0xffffffffu, lane_n, i);
    row = __shfl_sync(0xffffffffu, lane_row, i);
    nt = (n + kPos - 1) / kPos;
  }
  // Tile `at` of the sequence; there is one.
  __device__ __forceinline__ void seek(long long at) {
    chunk0 = 0;
    for (window(0);; window(base + 32)) {
      const int tiles = (lane_n + kPos - 1) / kPos * blocks;
      long long upto = tiles;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const long long v = __shfl_up_sync(0xffffffffu, upto, d);
        if (lane >= d) upto += v;
      }
      const unsigned past = __ballot_sync(0xffffffffu, upto > at);
      const int chunks = (lane_n + kChunk - 1) / kChunk;
      if (past != 0u) {
        const int i = __ffs(past) - 1;
        take(i);
        const int in = static_cast<int>(at - __shfl_sync(0xffffffffu, upto - tiles, i));
        hb = in / nt;
        t = in - hb * nt;
        chunk0 += warp_sum(lane < i ? chunks : 0);
        return;
      }
      at -= __shfl_sync(0xffffffffu, upto, 31);
      chunk0 += warp_sum(chunks);
      if (base + 32 >= c.batch) { b = c.batch; n = nt = hb = t = 0; return; }   // not reached
    }
  }
  // On to the next tile; only where there is one.
  __device__ __forceinline__ void next() {
    if (++t < nt) return;
    t = 0;
    if (++hb < blocks) return;
    hb = 0;
    do {
      chunk0 += (n + kChunk - 1) / kChunk;
      if (b + 1 >= c.batch) { n = nt = 0; return; }                            // not reached
      if (b + 1 == base + 32) window(base + 32);
      take(b + 1 - base);
    } while (n == 0);
  }
};

struct Wait {
  int* status;
  volatile int* aborted;   // shared memory
  // Every waiter observes every phase of its barriers in order.  False after ~2 s, or once another
  // thread of the CTA gave up; the status word then says so.
  __device__ __forceinline__ bool operator()(uint32_t bar, uint32_t parity) const {
    if (mbar_try_wait(bar, parity)) return true;
    long long t0 = 0;
    for (uint32_t spin = 1;; ++spin) {
      if (mbar_try_wait(bar, parity)) return true;
      if ((spin & 0x3FFu) == 0) {
        if (t0 == 0) t0 = clock64();
        if (*aborted || clock64() - t0 > kWaitCycles) {
          *aborted = 1;
          atomicCAS(status, 0, AKL_ERR_TIMEOUT);
          return false;
        }
      }
    }
  }
};

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
// D[16 x 8] += A[16 x 16] B[16 x 8], 16-bit operands of the pool's type, 32-bit sums.
template <int KV>
__device__ __forceinline__ void mma16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (KV == AKL_KV_BF16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Two floats as sums of numbers of the pool's type, the largest first.
template <int KV, int kParts>
__device__ __forceinline__ void split2(float a, float b, uint32_t (&out)[kParts][2], int at) {
#pragma unroll
  for (int i = 0; i < kParts; ++i) {
    if (KV == AKL_KV_BF16) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
      const float2 f = __bfloat1622float2(h);
      out[i][at] = *reinterpret_cast<const uint32_t*>(&h);
      a -= f.x;
      b -= f.y;
    } else {
      const __half2 h = __floats2half2_rn(a, b);
      const float2 f = __half22float2(h);
      out[i][at] = *reinterpret_cast<const uint32_t*>(&h);
      a -= f.x;
      b -= f.y;
    }
  }
}

// Queries of one kv head as the B operand, channels 128 half ..: thread (g, q) = (lane / 4, lane % 4) holds head g,
// channels 16 k + 2 q, + 1 and the same + 8.  cs: what scores of the heads 2 q and 2 q + 1 are multiplied by.
template <int KV>
__device__ __forceinline__ void load_q(const akl_decode_t& c, int b, int head0, int group, int half, int lane, uint32_t (&q)[8][2], float (&cs)[2]) {
  const int g = lane >> 2, quad = lane & 3;
  const uint32_t* src = reinterpret_cast<const uint32_t*>(static_cast<const uint16_t*>(c.q) + b * c.q_stride + (head0 + g) * 256) + quad;
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    q[k][0] = g < group ? __ldg(src + half * 64 + k * 8) : 0u;
    q[k][1] = g < group ? __ldg(src + half * 64 + k * 8 + 4) : 0u;
  }
  cs[0] = cs[1] = c.sm_scale * kLog2e;
  if (KV == AKL_KV_FP16) {
    float top = 0.f;
    auto larger = [&](uint32_t v) { top = fmaxf(top, fmaxf(fabsf(bf16_bits_to_float(v & 0xFFFFu)), fabsf(bf16_bits_to_float(v >> 16)))); };
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      larger(q[k][0]);
      larger(q[k][1]);
      larger(g < group ? __ldg(src + (half ^ 1) * 64 + k * 8) : 0u);
      larger(g < group ? __ldg(src + (half ^ 1) * 64 + k * 8 + 4) : 0u);
    }
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    // 2^e <= top < 2^(e+1), with both 2^e and 2^-e normal; 1 for a row of zeros or of infinities
    int e = static_cast<int>((__float_as_uint(top) >> 23) & 0xFFu) - 127;
    e = (top == 0.f || e == 128) ? 0 : max(-126, min(126, e));
    const float down = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
    const float up = __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const __half2 h = __floats2half2_rn(bf16_bits_to_float(q[k][i] & 0xFFFFu) * down, bf16_bits_to_float(q[k][i] >> 16) * down);
        q[k][i] = *reinterpret_cast<const uint32_t*>(&h);
      }
    }
    cs[0] *= __shfl_sync(0xffffffffu, up, quad * 8);
    cs[1] *= __shfl_sync(0xffffffffu, up, quad * 8 + 4);
  }
}

__device__ __forceinline__ void copy16(uint32_t dst, const void* src, uint32_t bytes) {   // bytes: 16, or 0 to clear
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}

// A producer warp: its positions of every tile of this CTA's share.  A row of 512 bytes is one
// instruction of the warp; rows that are not there are cleared, for 0 * NaN is not 0.
template <int HB>
__device__ __forceinline__ void produce(const akl_decode_t& c, uint32_t smem, uint8_t* smem_gen, const Wait& wait,
                                        Cursor<HB>& at, long long first, int count, int own, int lane) {
  using T = Tile<HB>;
  // The page-table entry of this lane's position in the tile the cursor is at, as it was loaded: anything that looks
  // at it here, a sign extension even, would wait for the load (0.7 us a tile).  Negative: nothing to read.
  int2 slot[kAhead];
  int block[kAhead];
  const bool wide = c.idx_dtype == AKL_IDX_I64;
  auto look = [&](int2& s, int& hb) {
    hb = at.hb;
    s = make_int2(-1, -1);
    const int i = at.t * T::kPos + own * T::kOwn + lane;
    if (lane < T::kOwn && i < at.n) {
      const long long e = at.row * c.table_stride + i;
      if (wide) s = __ldg(reinterpret_cast<const int2*>(c.page_table) + e);
      else s.x = __ldg(reinterpret_cast<const int*>(c.page_table) + e);
    }
  };
  at.seek(first);
#pragma unroll
  for (int s = 0; s < kAhead; ++s) {
    if (s < count) {
      if (s > 0) at.next();
      look(slot[s], block[s]);
    }
  }
  const uint32_t bars = smem + T::kOffBar;
  const uint32_t dst0 = smem + own * T::kOwn * T::kPitch + lane * 16;
  for (int it = 0; it < count; ++it) {
    const int st = it % kStages;
    const bool free = it < kStages || (wait(bars + (kStages + st) * 8, ((it / kStages) - 1) & 1) && !*wait.aborted);
    if (!__all_sync(0xffffffffu, free)) break;
    const bool there = slot[0].x >= 0 && slot[0].x < c.pool_rows && (!wide || slot[0].y == 0);
    const int now = there ? slot[0].x : -1;
    const unsigned mask = __ballot_sync(0xffffffffu, now >= 0);
    const long long head0 = static_cast<long long>(block[0]) * (HB * 256) + lane * 8;
    const uint32_t dst = dst0 + st * T::kStage;
#pragma unroll
    for (int i = 0; i < T::kOwn; ++i) {
      const int s = __shfl_sync(0xffffffffu, now, i);
      const long long row = s < 0 ? 0 : s;
      const uint32_t bytes = s < 0 ? 0u : 16u;
      const uint16_t* k = static_cast<const uint16_t*>(c.k_pool) + row * c.k_stride + head0;
      const uint16_t* v = static_cast<const uint16_t*>(c.v_pool) + row * c.v_stride + head0;
#pragma unroll
      for (int e = 0; e < HB; ++e) {
        copy16(dst + i * T::kPitch + e * 512, k + e * 256, bytes);
        copy16(dst + T::kPlane + i * T::kPitch + e * 512, v + e * 256, bytes);
      }
    }
    // one arrival per thread once its copies landed, and one that publishes the mask
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bars + st * 8) : "memory");
    if (lane == 0) {
      reinterpret_cast<volatile uint32_t*>(smem_gen + T::kOffMask + st * 16)[own] = mask;
      mbar_arrive(bars + st * 8);
    }
#pragma unroll
    for (int s = 0; s + 1 < kAhead; ++s) {
      block[s] = block[s + 1];
      slot[s] = slot[s + 1];
    }
    if (it + kAhead < count) {
      at.next();
      look(slot[kAhead - 1], block[kAhead - 1]);
    }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");       // no copy outlives its thread
}

template <int KV, int HB>
__global__ void __launch_bounds__(kThreads, 1) decode_kernel(const akl_decode_t c, const Work w) {
  using T = Tile<HB>;
  extern __shared__ __align__(128) uint8_t smem_gen[];
  __shared__ int sm_aborted;
  const uint32_t smem = smem_u32(smem_gen);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (threadIdx.x == 0) {
    sm_aborted = 0;
    for (int i = 0; i < kStages; ++i) {
      mbar_init(smem + T::kOffBar + i * 8, kProducers * 33);
      mbar_init(smem + T::kOffBar + (kStages + i) * 8, kWarps);
    }
    mbar_init_fence();
  }
  Cursor<HB> at(c, lane);
  const long long total = at.total();
  // (at least two tiles a CTA made one request of 1000 positions 10.1 us instead of 8.7, and nothing faster)
  const long long ctas = min(total, static_cast<long long>(gridDim.x));
  if (blockIdx.x >= ctas) return;                    // the whole CTA: nothing waits for it
  const long long first = total * blockIdx.x / ctas;
  const int count = static_cast<int>(total * (blockIdx.x + 1) / ctas - first);
  __syncthreads();
  const Wait wait{w.status, &sm_aborted};

  if (warp >= kWarps) {
    produce<HB>(c, smem, smem_gen, wait, at, first, count, warp - kWarps, lane);
    return;
  }

  // ---- consumers: kv head `unit` of the block, positions 16 tg .. of the tile, channels 128 half ..
  const int unit = (warp & 3) % HB, tg = (warp & 3) / HB, half = warp >> 2;
  const int g = lane >> 2, quad = lane & 3, group = c.q_heads / c.kv_heads;
  const uint32_t bars = smem + T::kOffBar;
  constexpr float kShift = KV == AKL_KV_FP16 ? 14.f : 0.f;   // P carries 2^kShift
  constexpr int kParts = KV == AKL_KV_BF16 ? 3 : 2;          // numbers of the pool's type that make up one of P
  const uint32_t k_lane = (tg * 16 + (lane & 15)) * T::kPitch + unit * 512 + half * 256 + (lane >> 4) * 16;
  const uint32_t v_lane = T::kPlane + (tg * 16 + (lane & 7) + ((lane >> 4) & 1) * 8) * T::kPitch + unit * 512 + half * 256 +
                          ((lane >> 3) & 1) * 16;
  float4* const meet = reinterpret_cast<float4*>(smem_gen + T::kOffMeet) + lane;      // [tile & 1][warp][lane]
  uint32_t q[8][2];
  float cs[2], m[2], l[2], o[8][4];
  bool ok = true, new_piece = true;
  int t_begin = 0;
  at.seek(first);
  for (int it = 0; it < count; ++it) {
    if (new_piece) {
      load_q<KV>(c, at.b, (at.hb * HB + unit) * group, group, half, lane, q, cs);
      m[0] = m[1] = -INFINITY;
      l[0] = l[1] = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
      t_begin = at.t;
      new_piece = false;
    }
    const int st = it % kStages;
    const uint32_t stage = smem + st * T::kStage;
    if (ok) ok = __all_sync(0xffffffffu, wait(bars + st * 8, (it / kStages) & 1));
    unsigned there = 0;                 // positions of this warp's sixteen that are there
    if (ok) {
#pragma unroll
      for (int i = 0; i < 16 / T::kOwn; ++i)
        there |= reinterpret_cast<volatile uint32_t*>(smem_gen + T::kOffMask + st * 16)[tg * (16 / T::kOwn) + i] << (i * T::kOwn);
    }
    // Scores of 16 positions x 8 heads: thread has positions g, g + 8 of heads 2 quad, 2 quad + 1.  Each of the
    // pair of warps multiplies half the channels; two chains keep the sums short, in time and in rounding.
    float x[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
    float4* const buf = meet + (it & 1) * (kWarps * 32);    // its next use is two tiles on, behind the next tile's barrier
    float4 own = make_float4(0.f, 0.f, 0.f, 0.f);
    if (there != 0u) {
      float s[2][4];
#pragma unroll
      for (int i = 0; i < 2; ++i) s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.f;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        uint32_t a[4];
        ldsm4(stage + k_lane + k * 32, a);
        mma16<KV>(s[k & 1], a, q[k][0], q[k][1]);
      }
      own = make_float4(s[0][0] + s[1][0], s[0][1] + s[1][1], s[0][2] + s[1][2], s[0][3] + s[1][3]);
      buf[warp * 32] = own;
    }
    // (by every warp for every tile, whatever it found: nobody waits here for one that gave up)
    asm volatile("bar.sync %0, 64;" ::"r"(2 + (warp & 3)) : "memory");
    if (ok) {
      if (there != 0u) {
        const float4 other = buf[(warp ^ 4) * 32];
        x[0] = (own.x + other.x) * cs[0];
        x[1] = (own.y + other.y) * cs[1];
        x[2] = (own.z + other.z) * cs[0];
        x[3] = (own.w + other.w) * cs[1];
        if (there != 0xFFFFu) {
          if (!((there >> g) & 1u)) x[0] = x[1] = -INFINITY;
          if (!((there >> (g + 8)) & 1u)) x[2] = x[3] = -INFINITY;
        }
      }
      if (w.scores != nullptr && half == 0) {
        const long long chunk = at.chunk0 + (at.t * T::kPos + tg * 16) / kChunk;
        if (chunk < w.max_chunks) {
          float* dst = w.scores + (chunk * c.q_heads + (at.hb * HB + unit) * group) * kChunk + (at.t * T::kPos + tg * 16) % kChunk + g;
#pragma unroll
          for (int e = 0; e < 2; ++e)
            if (quad * 2 + e < group) {
              dst[(quad * 2 + e) * kChunk] = x[e];
              dst[(quad * 2 + e) * kChunk + 8] = x[e + 2];
            }
        }
      }
      if (there != 0u) {
        float safe[2];
        float alpha[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float top = fmaxf(x[e], x[e + 2]);
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
          const float m_new = fmaxf(m[e], top);
          safe[e] = m_new == -INFINITY ? 0.f : m_new;      // nothing but scores of -inf so far: they weigh 0
          alpha[e] = ex2(m[e] - safe[e]);                  // 1 where the maximum stays
          m[e] = m_new;
        }
        float p[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) p[i] = ex2(x[i] - safe[i & 1] + kShift);
        l[0] = fmaf(l[0], alpha[0], p[0] + p[2]);
        l[1] = fmaf(l[1], alpha[1], p[1] + p[3]);
        uint32_t pt[kParts][2];
        split2<KV>(p[0], p[1], pt, 0);
        split2<KV>(p[2], p[3], pt, 1);
#pragma unroll
        for (int i = 0; i < kParts; ++i) {
          pt[i][0] = transpose8x8(pt[i][0]);
          pt[i][1] = transpose8x8(pt[i][1]);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          uint32_t a[4];
          ldsm4_trans(stage + v_lane + i * 32, a);
          float t[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int k = kParts - 1; k >= 0; --k) mma16<KV>(t, a, pt[k][0], pt[k][1]);
          o[i][0] = fmaf(o[i][0], alpha[0], t[0]);
          o[i][1] = fmaf(o[i][1], alpha[1], t[1]);
          o[i][2] = fmaf(o[i][2], alpha[0], t[2]);
          o[i][3] = fmaf(o[i][3], alpha[1], t[3]);
        }
      }
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(bars + (kStages + st) * 8);
    if (at.t + 1 < at.nt && it + 1 < count) {
      ++at.t;
      continue;
    }

    // ---- end of this CTA's piece of (request, head block)
    new_piece = true;
    if (*wait.aborted) ok = false;
    ok = __all_sync(0xffffffffu, ok);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      l[e] += __shfl_xor_sync(0xffffffffu, l[e], 4);
      l[e] += __shfl_xor_sync(0xffffffffu, l[e], 8);
      l[e] += __shfl_xor_sync(0xffffffffu, l[e], 16);
    }
    if (!ok) {                        // a bounded wait ran out: leave nothing that looks like a result
      l[0] = l[1] = __int_as_float(0x7FC00000);
      m[0] = m[1] = 0.f;
    }
    if (T::kGroups > 1) {
      // join the position groups of each kv head: a common maximum, then pairwise sums through shared memory
      float2* ml = reinterpret_cast<float2*>(smem_gen + T::kOffMl);
      float* buf = reinterpret_cast<float*>(smem_gen + T::kOffMerge);
      if (g == 0) {
        ml[warp * 8 + quad * 2] = make_float2(m[0], l[0]);
        ml[warp * 8 + quad * 2 + 1] = make_float2(m[1], l[1]);
      }
      asm volatile("bar.sync 1, 256;" ::: "memory");
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float top = -INFINITY, sum = 0.f;
#pragma unroll
        for (int k = 0; k < T::kGroups; ++k) top = fmaxf(top, ml[(half * 4 + k * HB + unit) * 8 + quad * 2 + e].x);
        const float safe = top == -INFINITY ? 0.f : top;
#pragma unroll
        for (int k = 0; k < T::kGroups; ++k) {
          const float2 v = ml[(half * 4 + k * HB + unit) * 8 + quad * 2 + e];
          sum += v.y * ex2(v.x - safe);
        }
        const float f = ex2(m[e] - safe);
#pragma unroll
        for (int i = 0; i < 8; ++i) { o[i][e] *= f; o[i][e + 2] *= f; }
        m[e] = top;
        l[e] = sum;
      }
#pragma unroll
      for (int step = T::kGroups / 2; step > 0; step >>= 1) {
        // groups step .. 2 step - 1 hand theirs to groups 0 .. step - 1
        const int pair = (half * step + (tg % step)) * HB + unit;       // at most 4 pairs of 4 KiB
        if (tg >= step && tg < 2 * step) {
#pragma unroll
          for (int i = 0; i < 32; ++i) buf[(pair * 32 + i) * 32 + lane] = o[i >> 2][i & 3];
        }
        asm volatile("bar.sync 1, 256;" ::: "memory");
        if (tg < step) {
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i >> 2][i & 3] += buf[(pair * 32 + i) * 32 + lane];
        }
        asm volatile("bar.sync 1, 256;" ::: "memory");
      }
    }
    const bool whole = t_begin == 0 && at.t + 1 == at.nt;
    const int piece_slot = 2 * blockIdx.x + (first + it - (at.t - t_begin) == first ? 0 : 1);
    if (warp == 0 && lane == 0) {
      int* info = reinterpret_cast<int*>(w.info + at.b * 2 + at.hb);
      if (t_begin == 0) { info[0] = piece_slot; info[1] = blockIdx.x; }
      if (at.t + 1 == at.nt) info[2] = blockIdx.x;
    }
    if (tg == 0) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int h = quad * 2 + e;
        if (h >= group) break;
        const int head = (at.hb * HB + unit) * group + h;
        if (whole) {
          const float inv = l[e] == 0.f ? 0.f : 1.f / l[e];
          __nv_bfloat16* dst = reinterpret_cast<__nv_bfloat16*>(c.out) + (static_cast<long long>(at.b) * c.q_heads + head) * 256 + half * 128 + g;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            dst[i * 16] = __float2bfloat16_rn(o[i][e] * inv);
            dst[i * 16 + 8] = __float2bfloat16_rn(o[i][e + 2] * inv);
          }
          if (half == 0 && g == 0) {
            const float lse = l[e] == 0.f ? -INFINITY : m[e] + (log2f(l[e]) - kShift);
            w.lse[static_cast<long long>(at.b) * c.q_heads + head] = lse;
            if (c.lse_out != nullptr) c.lse_out[static_cast<long long>(at.b) * c.q_heads + head] = lse;
          }
        } else {
          const int at_head = piece_slot * kSlotHeads + unit * group + h;
          float* dst = w.parts + static_cast<long long>(at_head) * 256 + half * 128 + g;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            dst[i * 16] = o[i][e];
            dst[i * 16 + 8] = o[i][e + 2];
          }
          if (half == 0 && g == 0) w.ml[at_head] = make_float2(m[e] - kShift, l[e]);
        }
      }
    }
    if (it + 1 < count) at.next();
  }
}

// Join of the partial states of a (request, q head): lse = log2 sum_i l_i 2^m_i, out = sum_i 2^(m_i - lse) O_i,
// in position order.  A request without positions gets its zeros here; one that a single CTA held
// has its result already.  Latency bound (a request's parts are read from L2 once): what counts is how
// many of the loads are in flight together.

// Few requests, so up to all 148 parts of one: a CTA takes 64 channels, sixteen sets of sixteen threads
// every sixteenth part, all of whose loads are issued before the factors that they wait for.
__device__ __forceinline__ void join_wide(const akl_decode_t& c, const Work& w, int hb_heads, int block) {
  constexpr int kSets = 16, kEach = kMaxCtas / kSets;
  __shared__ float sm_f[kMaxCtas];
  __shared__ float sm_red[16];
  __shared__ __align__(16) float sm_o[kSets][64];       // read and written as float4
  const int head_of = block >> 2, b = head_of / c.q_heads, head = head_of - b * c.q_heads, ch0 = (block & 3) * 64;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  long long row;
  const int n = request_of(c, b, row);
  const int hb = head / hb_heads, h = head - hb * hb_heads;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const long long at = static_cast<long long>(b) * c.q_heads + head;
  __nv_bfloat16* out = reinterpret_cast<__nv_bfloat16*>(c.out) + at * 256 + ch0;
  if (n == 0) {
    if (tid < 64) out[tid] = __float2bfloat16_rn(0.f);
    if (tid == 0 && ch0 == 0) {
      w.lse[at] = -INFINITY;
      if (c.lse_out != nullptr) c.lse_out[at] = -INFINITY;
    }
    return;
  }
  const int4 info = w.info[b * 2 + hb];
  const int parts = info.z - info.y + 1;
  if (parts == 1) return;
  auto slot = [&](int i) { return (i == 0 ? info.x : 2 * (info.y + i)) * kSlotHeads + h; };
  const int set = tid >> 4, ch = (tid & 15) * 4;
  float4 v[kEach];
#pragma unroll
  for (int k = 0; k < kEach; ++k)
    if (set + k * kSets < parts) v[k] = *reinterpret_cast<const float4*>(w.parts + static_cast<long long>(slot(set + k * kSets)) * 256 + ch0 + ch);
  float2 mine = make_float2(-INFINITY, 0.f);
  if (tid < parts) mine = w.ml[slot(tid)];
  float top = warp_max(mine.x);
  if (lane == 0) sm_red[warp] = top;
  __syncthreads();
  top = sm_red[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) top = fmaxf(top, sm_red[i]);
  const float safe = top == -INFINITY ? 0.f : top;
  const float f = ex2(mine.x - safe);
  if (tid < parts) sm_f[tid] = f;
  float sum = mine.y * f;
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, s);
  if (lane == 0) sm_red[8 + warp] = sum;
  __syncthreads();
  sum = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) sum += sm_red[8 + i];
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int k = 0; k < kEach; ++k)
    if (set + k * kSets < parts) {
      const float fi = sm_f[set + k * kSets];
      o.x = fmaf(fi, v[k].x, o.x);
      o.y = fmaf(fi, v[k].y, o.y);
      o.z = fmaf(fi, v[k].z, o.z);
      o.w = fmaf(fi, v[k].w, o.w);
    }
  *reinterpret_cast<float4*>(&sm_o[set][ch]) = o;
  __syncthreads();
  if (tid < 64) {
    float total = 0.f;
#pragma unroll
    for (int i = 0; i < kSets; ++i) total += sm_o[i][tid];
    out[tid] = __float2bfloat16_rn(sum == 0.f ? 0.f : total / sum);
  }
  if (tid == 0 && ch0 == 0) {
    const float lse = sum == 0.f ? -INFINITY : top + log2f(sum);
    w.lse[at] = lse;
    if (c.lse_out != nullptr) c.lse_out[at] = lse;
  }
}

// All 256 channels of one (request, q head) by a CTA: four sets of 64 threads take every fourth part, a few of them
// in flight.  (Registers count here: the weights of a batch are added by this kernel too, and its whole call takes
// 3 % longer at 80 registers than at 40.)
__device__ __forceinline__ void join_block(const akl_decode_t& c, const Work& w, long long at, int h, const int4 info) {
  constexpr int kSets = 4, kFlight = 4;
  __shared__ float sm_f[kMaxCtas];
  __shared__ float sm_red[16];
  __shared__ __align__(16) float sm_o[kSets][256];      // read and written as float4
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int parts = info.z - info.y + 1;
  auto slot = [&](int i) { return (i == 0 ? info.x : 2 * (info.y + i)) * kSlotHeads + h; };
  float2 mine = make_float2(-INFINITY, 0.f);
  if (tid < parts) mine = w.ml[slot(tid)];
  float top = warp_max(mine.x);
  if (lane == 0) sm_red[warp] = top;
  __syncthreads();
  top = warp_max(sm_red[lane & 7]);
  const float f = ex2(mine.x - (top == -INFINITY ? 0.f : top));
  if (tid < parts) sm_f[tid] = f;
  float sum = mine.y * f;
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, s);
  if (lane == 0) sm_red[8 + warp] = sum;
  __syncthreads();
  const int set = tid >> 6, ch = (tid & 63) * 4;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i = set; i < parts; i += kSets * kFlight) {
    float4 v[kFlight];
#pragma unroll
    for (int k = 0; k < kFlight; ++k)
      if (i + k * kSets < parts) v[k] = *reinterpret_cast<const float4*>(w.parts + static_cast<long long>(slot(i + k * kSets)) * 256 + ch);
#pragma unroll
    for (int k = 0; k < kFlight; ++k)
      if (i + k * kSets < parts) {
        const float fi = sm_f[i + k * kSets];
        o.x = fmaf(fi, v[k].x, o.x);
        o.y = fmaf(fi, v[k].y, o.y);
        o.z = fmaf(fi, v[k].z, o.z);
        o.w = fmaf(fi, v[k].w, o.w);
      }
  }
  *reinterpret_cast<float4*>(&sm_o[set][ch]) = o;
  __syncthreads();
  sum = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) sum += sm_red[8 + i];
  const float total = (sm_o[0][tid] + sm_o[1][tid]) + (sm_o[2][tid] + sm_o[3][tid]);
  reinterpret_cast<__nv_bfloat16*>(c.out)[at * 256 + tid] = __float2bfloat16_rn(sum == 0.f ? 0.f : total / sum);
  if (tid == 0) {
    const float lse = sum == 0.f ? -INFINITY : top + log2f(sum);
    w.lse[at] = lse;
    if (c.lse_out != nullptr) c.lse_out[at] = lse;
  }
  __syncthreads();                                      // the shared memory is the next one's
}

// Many requests: a warp per (request, q head), a lane eight channels, one part after the other with a running
// maximum.  That is half a microsecond a part, and a long request among short ones still has a part in nearly every
// CTA; so a pair of more than kSerial parts is left to the whole CTA (true).  (24:4, one request of 131072 among twelve of 3:
// 182 us when the warp walked through all its parts, 114 now, and 109 with the wide join of one request fewer; of 8192:
// 81, 25 and 17 us.)
constexpr int kSerial = 8;
__device__ __forceinline__ bool join_warp(const akl_decode_t& c, const Work& w, int hb_heads, long long at) {
  const int lane = threadIdx.x & 31;
  const bool in = at < static_cast<long long>(c.batch) * c.q_heads;
  const int b = in ? static_cast<int>(at / c.q_heads) : 0, head = in ? static_cast<int>(at - static_cast<long long>(b) * c.q_heads) : 0;
  const int hb = head / hb_heads, h = head - hb * hb_heads;
  long long row;
  const int n = request_of(c, b, row);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (!in) return false;
  __nv_bfloat16* out = reinterpret_cast<__nv_bfloat16*>(c.out) + at * 256 + lane * 8;
  float m = -INFINITY, l = 0.f, o[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) o[i] = 0.f;
  if (n > 0) {
    const int4 info = w.info[b * 2 + hb];
    const int parts = info.z - info.y + 1;
    if (parts == 1) return false;
    if (parts > kSerial) return true;
#pragma unroll 2
    for (int i = 0; i < parts; ++i) {
      const int s = (i == 0 ? info.x : 2 * (info.y + i)) * kSlotHeads + h;
      const float2 ml = w.ml[s];
      const float4* src = reinterpret_cast<const float4*>(w.parts + static_cast<long long>(s) * 256 + lane * 8);
      const float4 v0 = src[0], v1 = src[1];
      const float v[8] = {v0.x, v0.y, v0.z, v0.w, v1.x, v1.y, v1.z, v1.w};
      const float top = fmaxf(m, ml.x), safe = top == -INFINITY ? 0.f : top;
      const float keep = ex2(m - safe), add = ex2(ml.x - safe);
      m = top;
      l = l * keep + ml.y * add;
#pragma unroll
      for (int e = 0; e < 8; ++e) o[e] = o[e] * keep + v[e] * add;
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  uint32_t pk[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const __nv_bfloat162 t = __floats2bfloat162_rn(o[2 * e] * inv, o[2 * e + 1] * inv);
    pk[e] = *reinterpret_cast<const uint32_t*>(&t);
  }
  *reinterpret_cast<uint4*>(out) = make_uint4(pk[0], pk[1], pk[2], pk[3]);
  if (lane == 0) {
    const float lse = l == 0.f ? -INFINITY : m + log2f(l);
    w.lse[at] = lse;
    if (c.lse_out != nullptr) c.lse_out[at] = lse;
  }
  return false;
}

// The pairs of a CTA lie `joins` apart, so that the q heads of one long request fall to different CTAs.
__device__ __forceinline__ void join_many(const akl_decode_t& c, const Work& w, int hb_heads, int block, int joins) {
  __shared__ bool sm_long[8];
  const int warp = threadIdx.x >> 5;
  const bool left = join_warp(c, w, hb_heads, block + static_cast<long long>(warp) * joins);
  if ((threadIdx.x & 31) == 0) sm_long[warp] = left;
  __syncthreads();
  for (int i = 0; i < 8; ++i) {
    if (!sm_long[i]) continue;
    const long long at = block + static_cast<long long>(i) * joins;
    const int b = static_cast<int>(at / c.q_heads), head = static_cast<int>(at - static_cast<long long>(b) * c.q_heads);
    const int hb = head / hb_heads, h = head - hb * hb_heads;
    join_block(c, w, at, h, w.info[b * 2 + hb]);
  }
}

// weights[row][i] = decay weights[row][i] + sum_h 2^(x[h][i] - lse[h]), from the scores the decode launch
// recorded: 4 bytes per position and q head written and read, against the K and V rows' 1024 per kv
// head.  A thread per position, 256 positions at a time.  The log-sum-exps are put together here
// once more from the parts (a few floats a head), so that this needs no launch behind the joins'.
__device__ __forceinline__ void add_weights(const akl_decode_t& c, const Work& w, int hb_heads, int block, int blocks) {
  __shared__ long long sm_chunks[8];
  __shared__ float sm_lse[64];
  const int b = block / blocks, part = block - b * blocks, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  long long row, before = 0;
  for (int i = tid; i < b; i += 256) before += (request_of(c, i, row) + kChunk - 1) / kChunk;
  before = warp_sum(before);
  if (lane == 0) sm_chunks[warp] = before;
  const int n = request_of(c, b, row);
  if (part * 256 >= n) return;                        // the whole CTA
  asm volatile("griddepcontrol.wait;" ::: "memory");
  for (int head = warp; head < c.q_heads; head += 8) {
    const int hb = head / hb_heads, h = head - hb * hb_heads;
    const int4 info = w.info[b * 2 + hb];
    const int parts = info.z - info.y + 1;
    float lse;
    if (parts == 1) {
      lse = w.lse[static_cast<long long>(b) * c.q_heads + head];
    } else {
      float m = -INFINITY, l = 0.f;
      for (int i = lane; i < parts; i += 32) {
        const float2 ml = w.ml[(i == 0 ? info.x : 2 * (info.y + i)) * kSlotHeads + h];
        const float top = fmaxf(m, ml.x), safe = top == -INFINITY ? 0.f : top;
        l = l * ex2(m - safe) + ml.y * ex2(ml.x - safe);
        m = top;
      }
      const float top = warp_max(m);
      l *= ex2(m - (top == -INFINITY ? 0.f : top));
#pragma unroll
      for (int s = 16; s > 0; s >>= 1) l += __shfl_xor_sync(0xffffffffu, l, s);
      lse = l == 0.f ? -INFINITY : top + log2f(l);
    }
    if (lane == 0) sm_lse[head] = lse;
  }
  __syncthreads();
  long long chunk0 = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) chunk0 += sm_chunks[i];
  if (chunk0 + (n + kChunk - 1) / kChunk > w.max_chunks) {
    // not all of the request's scores were recorded: its row stays as it was, from the first position to the last
    if (tid == 0) atomicCAS(w.status, 0, AKL_ERR_CAPACITY);
    return;
  }
  for (int i = part * 256 + tid; i < n; i += blocks * 256) {
    const float* x = w.scores + (chunk0 + i / kChunk) * c.q_heads * kChunk + i % kChunk;
    float total = 0.f;
#pragma unroll 8
    for (int h = 0; h < c.q_heads; ++h) {
      const float v = x[h * kChunk];
      total += v == -INFINITY ? 0.f : ex2(v - sm_lse[h]);
    }
    float* dst = c.weights + row * c.weights_stride + i;
    *dst = c.weight_decay == 0.f ? total : fmaf(c.weight_decay, *dst, total);
  }
}

// What follows the decode launch: the joins, and behind them in the grid the weights.
template <bool kWide>
__global__ void __launch_bounds__(256) decode_finish_kernel(const akl_decode_t c, const Work w, int hb_heads, int joins, int blocks) {
  const int block = blockIdx.x;
  if (block >= joins) add_weights(c, w, hb_heads, block - joins, blocks);
  else if (kWide) join_wide(c, w, hb_heads, block);
  else join_many(c, w, hb_heads, block, joins);
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
  if (c->pool_rows >= (1ll << 31)) return AKL_ERR_UNSUPPORTED;      // slots travel in 32 bits
  if (c->table_width >= (1 << 30)) return AKL_ERR_UNSUPPORTED;      // positions too, and loops step past the end
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
  // the second launch's CTAs, counted before the first one runs (a wide join has few requests)
  if ((static_cast<int64_t>(c->batch) * c->q_heads + 7) / 8 + static_cast<int64_t>(c->batch) * weight_blocks(*c) >= (1ll << 31))
    return AKL_ERR_UNSUPPORTED;
  const int64_t batch = c->batch, heads = c->q_heads, dense = static_cast<int64_t>(c->kv_heads) * 512;
  const Span outputs[3] = {{c->out, 1, batch * heads * 512, 1}, {c->lse_out, 1, batch * heads * 4, 1},
                           {c->weights, c->table_rows, static_cast<int64_t>(c->table_width) * 4, c->weights_stride * 4}};
  const Span inputs[6] = {{c->q, batch, heads * 512, c->q_stride * 2},
                          {c->k_pool, c->pool_rows, dense, c->k_stride * 2},
                          {c->v_pool, c->pool_rows, dense, c->v_stride * 2},
                          {c->page_table, c->table_rows, static_cast<int64_t>(c->table_width) * index_bytes(c->idx_dtype),
                           c->table_stride * index_bytes(c->idx_dtype)},
                          {c->rows, 1, batch * index_bytes(c->rows_dtype), 1},
                          {c->kv_lens, 1, batch * index_bytes(c->lens_dtype), 1}};
  return outputs_meet(outputs, 3, inputs, 6) ? AKL_ERR_INVALID : AKL_OK;
}

template <int KV, int HB>
int launch_decode(const akl_decode_t& c, const Work& w, int ctas, cudaStream_t s) {
  static std::atomic<bool> configured[64];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && !(dev >= 0 && dev < 64 && configured[dev].load(std::memory_order_acquire))) {
    e = cudaFuncSetAttribute(decode_kernel<KV, HB>, cudaFuncAttributeMaxDynamicSharedMemorySize, Tile<HB>::kSmem);
    if (e == cudaSuccess && dev >= 0 && dev < 64) configured[dev].store(true, std::memory_order_release);
  }
  if (e == cudaSuccess) {
    decode_kernel<KV, HB><<<ctas, kThreads, Tile<HB>::kSmem, s>>>(c, w);
    e = cudaGetLastError();
  }
  if (e != cudaSuccess) { note_cuda_error(e, "decode_kernel"); return AKL_ERR_CUDA; }
  return AKL_OK;
}

// A launch that may be set up while the one before it still runs (it waits for its results itself).
template <typename... Args>
int launch_after(void (*kernel)(Args...), dim3 grid, cudaStream_t s, const char* name, Args... args) {
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(256);
  cfg.stream = s;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
  if (e != cudaSuccess) { note_cuda_error(e, name); return AKL_ERR_CUDA; }
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
  int sms = 0;
  if ((rc = device_sm_count(&sms)) != AKL_OK) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  uint8_t* ws = static_cast<uint8_t*>(c->workspace);
  Work w;
  w.status = reinterpret_cast<int*>(ws + L.off_status);
  w.info = reinterpret_cast<int4*>(ws + L.off_parts);
  w.ml = reinterpret_cast<float2*>(ws + L.off_parts + info_bytes(c->plan));
  w.parts = reinterpret_cast<float*>(ws + L.off_parts + info_bytes(c->plan) + align1k(kMlBytes));
  w.lse = reinterpret_cast<float*>(ws + L.off_lse);
  w.scores = c->weights != nullptr ? reinterpret_cast<float*>(ws + L.off_scores) : nullptr;
  w.max_chunks = (c->plan.max_weight_tokens + kChunk - 1) / kChunk;
  const int ctas = std::min(sms, kMaxCtas), hb = std::min(c->kv_heads, 4);
  if (c->kv_dtype == AKL_KV_BF16)
    rc = hb == 4 ? launch_decode<AKL_KV_BF16, 4>(*c, w, ctas, s)
                 : (hb == 2 ? launch_decode<AKL_KV_BF16, 2>(*c, w, ctas, s) : launch_decode<AKL_KV_BF16, 1>(*c, w, ctas, s));
  else
    rc = hb == 4 ? launch_decode<AKL_KV_FP16, 4>(*c, w, ctas, s)
                 : (hb == 2 ? launch_decode<AKL_KV_FP16, 2>(*c, w, ctas, s) : launch_decode<AKL_KV_FP16, 1>(*c, w, ctas, s));
  if (rc != AKL_OK) return rc;
  // the wide join while its CTAs fit the GPU in about two waves; past that most requests have few parts, and join_many
  // looks which have not
  const int64_t pairs = static_cast<int64_t>(c->batch) * c->q_heads;
  const bool wide = pairs * 4 <= 8 * sms;
  const int64_t joins = wide ? pairs * 4 : (pairs + 7) / 8;
  const int blocks = weight_blocks(*c);
  const int64_t grid = joins + static_cast<int64_t>(c->batch) * blocks;
  const int hb_heads = hb * (c->q_heads / c->kv_heads);
  return launch_after(wide ? decode_finish_kernel<true> : decode_finish_kernel<false>, dim3(static_cast<unsigned>(grid)), s,
                      "decode_finish_kernel", *c, w, hb_heads, static_cast<int>(joins), blocks);
}

}  // extern "C"
