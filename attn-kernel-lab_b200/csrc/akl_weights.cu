// Attention weights of an extend: weights[i] (+)= sum over rows t and q heads h with i <= prefix + t of
// 2^(c <q[t][h], k_i> - lse[t][h]), c = sm_scale log2 e.
//
// One product of 256 multiply-adds and one exponential per (position, row, head), and a sum over rows and
// heads: tensor pipe (4096 multiply-adds a cycle and SM) and exponential unit (16 a cycle and SM) need
// the same time, everything else is small.  The product is formed transposed, D = K Q^T, so that
//
//   * a TMEM lane is a position and the sum over rows and heads runs along the columns: every thread
//     adds up numbers of its own, nothing is exchanged, and the scores are never written;
//   * K is the A operand and stays in TMEM (256 positions, 256 columns) while the packed (row, head) pairs
//     of the kv head stream through shared memory as B, 128 at a time.  With K in shared memory an
//     M128 N128 K16 product reads 8 KiB in its 64 cycles, all that shared memory gives.
//
// The rows are packed once per call into swizzled images of 128 rows (row = t group + head, so short
// windows fill their tiles), with the factor and the LSE of each; a tile is then one bulk copy.
// A unit is (256 positions, kv head, 128 rows).  The units, position tile by position tile and head by
// head, are one sequence of which every CTA takes an equal share; tiles above the diagonal are not
// in it.  A CTA's first piece may continue the one of the CTA before it and then goes to a place of its own; the last launch
// adds the pieces of a position in a fixed order.
//
// Measured (a call in a CUDA graph, 24:4 heads): 2048 rows over 10240 positions 172 to 174 us, 1340 TFLOP/s of the
// product; tensor pipe and exponential unit 75 % busy in the main launch, the packing in front of it 8 us.  32 rows
// over 4097: 12.7 us, the latency of three launches.
//
// Rounding: scores and sums are 32-bit.  BF16 queries meet a BF16 pool unchanged; for an FP16 pool
// a row is divided by the power of two of its largest element and rounded to FP16: exact down to
// 2^-17 of that element, 2^-25 of it below.
#include <algorithm>
#include <atomic>
#include <cstring>

#include "akl_common.cuh"
#include "akl_sm100_ptx.cuh"

namespace akl {

namespace {

using namespace ptx;

constexpr int kMaxGroup = 8, kMaxHeads = 8;         // q heads per kv head, kv heads
constexpr int kMaxCtas = 160;
constexpr int kRows = 128;                          // packed rows of a tile
constexpr int kPos = 256;                           // positions of a unit: two TMEM lane sets
constexpr int kImage = 4 * kPlaneBytes;             // four planes of 64 channels, 128-byte swizzle
constexpr int kTileBytes = kImage + 2 * kRows * 4;  // and per row {factor}[128], {-lse}[128]
constexpr int kStages = 3;
constexpr int kEpiWarps = 16;
constexpr int kThreads = (kEpiWarps + 3) * 32;      // + two warps that issue products, one that fetches rows
constexpr uint32_t kTmemCols = 512, kColD = 0, kColK = 256;
constexpr float kLog2e = 1.4426950408889634f;
// The tensor pipe drops what its running 32-bit sum cannot hold: sixteen additions take about 2^-22 off a score,
// always towards zero, and off the heavy weights about 1e-6 of themselves.  The factor gives it back on average
// (error of the weights against 64 bits, eight cases: 6e-7 .. 1.2e-6 without, 0.5e-7 .. 2.8e-7 with).  A row whose
// products the pipe adds up exactly, of a few channels, lost nothing and is 2^-22 of its score too high instead: 4.4e-4
// of a weight at scores of 2600, where half a step of the score and of the LSE are 1.7e-4.
constexpr float kGiveBack = 1.f + 0x1p-22f;
constexpr long long kWaitCycles = 4000000000ll;     // ~2 s: a wait that long is a defect

inline uint64_t align1k(uint64_t x) { return (x + 1023) / 1024 * 1024; }

int weights_layout(const akl_weights_plan_t& p, akl_weights_layout_t* o) {
  if (p.max_kv_len < 1 || p.max_q_len < 1 || p.q_heads < 1 || p.kv_heads < 1) return AKL_ERR_INVALID;
  if (p.q_heads % p.kv_heads || p.q_heads / p.kv_heads > kMaxGroup) return AKL_ERR_UNSUPPORTED;
  if (p.max_q_len >= (1 << 27) || p.max_kv_len >= (1 << 30)) return AKL_ERR_UNSUPPORTED;    // 32-bit packed rows and positions
  std::memset(o, 0, sizeof(*o));
  const uint64_t tiles = (static_cast<uint64_t>(p.max_q_len) * (p.q_heads / p.kv_heads) + kRows - 1) / kRows;
  const uint64_t pos = (static_cast<uint64_t>(p.max_kv_len) + kPos - 1) / kPos * kPos;
  uint64_t off = 1024;
  o->off_q = off;
  off += align1k(tiles * p.kv_heads * kTileBytes);
  o->off_parts = off;
  off += align1k(pos * p.kv_heads * 4) + align1k(static_cast<uint64_t>(kMaxCtas) * kPos * 4);
  o->total_bytes = off;
  return AKL_OK;
}

// The sequence of units, from the call alone.  A (position tile, kv head) costs its row tiles and
// `piece` more for the K that has to come in first.
struct Units {
  int group, heads, tiles, ptiles, full, prefix;    // full: position tiles that every row tile sees
  int piece;
  long long total;                                  // cost of everything
  long long ctas;
  __host__ __device__ int first_tile(int p) const { // row tiles before this one see nothing of position tile p
    const long long n0 = static_cast<long long>(p) * kPos - prefix;
    return n0 <= 0 ? 0 : static_cast<int>(n0 * group / kRows);
  }
  __host__ __device__ int count(int p) const {
    const int f = first_tile(p);
    return f < tiles ? tiles - f : 0;
  }
  __host__ __device__ int cost(int p) const {
    const int n = count(p);
    return n > 0 ? n + piece : 0;
  }
  __host__ __device__ long long start(int p) const {
    long long u = static_cast<long long>(p < full ? p : full) * (tiles + piece);
    for (int i = full; i < p; ++i) {
      const int n = cost(i);
      if (n == 0) break;                            // seen by no row, as are all behind it
      u += n;
    }
    return u * heads;
  }
  // Where cost `at` (below total) falls, and how many units lie before it.
  __device__ __forceinline__ long long locate(long long at, int& p, int& j, int& skip) const {
    const long long per = static_cast<long long>(heads) * (tiles + piece);
    long long before;
    if (at < per * full) {
      p = static_cast<int>(at / per);
      at -= per * p;
      before = static_cast<long long>(p) * heads * tiles;
    } else {
      at -= per * full;
      before = static_cast<long long>(full) * heads * tiles;
      for (p = full; p + 1 < ptiles; ++p) {
        const long long n = static_cast<long long>(heads) * cost(p);
        if (at < n) break;
        at -= n;
        before += static_cast<long long>(heads) * count(p);
      }
    }
    const int n = count(p), each = n + piece;
    j = static_cast<int>(at / each);
    skip = static_cast<int>(at - static_cast<long long>(j) * each) - piece;
    skip = skip < 0 ? 0 : skip;
    return before + static_cast<long long>(j) * n + skip;
  }
};

struct Work {
  const uint8_t* images;     // [kv head][tile][kTileBytes]
  float* sums;               // [kv head][position]: pieces that begin a (position tile, kv head)
  float* more;               // [CTA][kPos]: first pieces that continue one
  int* status;
  int pos_cap;               // positions between two kv heads of sums
};

// One CTA per tile of packed rows, a warp every 16 of them: image rows in the pool's type, factors and -lse.
template <int KV>
__global__ void __launch_bounds__(256) pack_rows_kernel(const akl_weights_t c, uint8_t* images, int tiles) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int group = c.q_heads / c.kv_heads, j = blockIdx.y, lane = threadIdx.x & 31;
  const int row0 = (threadIdx.x >> 5) * 16, r0 = blockIdx.x * kRows + row0;
  uint8_t* image = images + (static_cast<long long>(j) * tiles + blockIdx.x) * kTileBytes;
  // words 4 q .. 4 q + 3 of every 16 go to 2 q, 2 q + 1, 8 + 2 q and 9 + 2 q, the order of K in TMEM
  uint8_t* plane = image + (lane >> 3) * kPlaneBytes;
  const int col = ((lane >> 2) & 1) * 64 + (lane & 3) * 8;
  int t = r0 / group, h = r0 - t * group;
#pragma unroll 1
  for (int half = 0; half < 16; half += 8) {
    uint4 raw[8];
    float lse[8];
    int tt = t, hh = h;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      raw[i] = make_uint4(0u, 0u, 0u, 0u);
      lse[i] = INFINITY;
      if (tt < c.T) {
        raw[i] = __ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(c.q) + tt * c.q_stride + (j * group + hh) * 256 + lane * 8));
        lse[i] = __ldg(c.lse + static_cast<long long>(tt) * c.q_heads + j * group + hh);
      }
      if (++hh == group) { hh = 0; ++tt; }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int row = row0 + half + i;
      float factor = c.sm_scale * (kLog2e * kGiveBack);
      if (isinf(lse[i])) raw[i] = make_uint4(0u, 0u, 0u, 0u);     // saw no key, or is no row: whatever it holds, its scores are 0
      uint4 out = raw[i];
      if (KV == AKL_KV_FP16) {
        float x[8], top = 0.f;
        unpack8<AKL_KV_BF16>(raw[i], x);
#pragma unroll
        for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(x[e]));
        top = warp_max(top);
        // 2^e <= top < 2^(e+1), with both 2^e and 2^-e normal; 1 for a row of zeros or of infinities
        int e = static_cast<int>((__float_as_uint(top) >> 23) & 0xFFu) - 127;
        e = (top == 0.f || e == 128) ? 0 : max(-126, min(126, e));
        const float down = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
        factor *= __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
        uint32_t pk[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const __half2 v = __floats2half2_rn(x[2 * k] * down, x[2 * k + 1] * down);
          pk[k] = *reinterpret_cast<const uint32_t*>(&v);
        }
        out = make_uint4(pk[0], pk[1], pk[2], pk[3]);
      }
      *reinterpret_cast<uint2*>(plane + swz128(row, col)) = make_uint2(out.x, out.y);
      *reinterpret_cast<uint2*>(plane + swz128(row, col + 32)) = make_uint2(out.z, out.w);
      if (lane == 0) {
        float* f = reinterpret_cast<float*>(image + kImage);
        f[row] = factor;
        f[kRows + row] = isinf(lse[i]) ? -INFINITY : -lse[i];      // and add nothing
      }
    }
    for (int i = 0; i < 8; ++i)
      if (++h == group) { h = 0; ++t; }
  }
}

struct Bars {
  uint32_t base;
  __device__ uint32_t q_full(int s) const { return base + s * 8; }
  __device__ uint32_t q_empty(int s) const { return base + (kStages + s) * 8; }
  __device__ uint32_t d_full(int s) const { return base + (2 * kStages + s) * 8; }
  __device__ uint32_t d_empty(int s) const { return base + (2 * kStages + 2 + s) * 8; }
  __device__ uint32_t k_full() const { return base + (2 * kStages + 4) * 8; }
};
constexpr int kBars = 2 * kStages + 5;
constexpr int kOffRed = kStages * kTileBytes;       // [2][3][kPos] floats, behind the row tiles
constexpr int kOffBar = kOffRed + 6 * kPos * 4;
constexpr int kOffMisc = kOffBar + kBars * 8 + 8;
constexpr int kSmem = kOffMisc + 64 + 1024;         // + alignment slack
static_assert(kSmem <= 232448 && kTileBytes % 1024 == 0, "shared memory");

struct Wait {
  int* status;
  volatile int* aborted;     // shared memory
  // Every waiter observes every phase of its barriers in order.  False after ~2 s, or once another
  // thread of the CTA gave up; the status word then says so.
  __device__ __forceinline__ bool operator()(uint32_t bar, uint32_t parity) const {
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

// Instruction descriptor of kind::f16: both operands K-major and of one type (f16 or bf16), fp32 D.
template <int KV>
__host__ __device__ constexpr uint32_t idesc_16(int m, int n) {
  return (1u << 4) | ((KV == AKL_KV_BF16 ? 1u : 0u) << 7) | ((KV == AKL_KV_BF16 ? 1u : 0u) << 10) |
         (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}
// D[tmem] (+)= A[tmem] * B[smem]^T; one thread issues.
__device__ __forceinline__ void mma_16_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%5, %5, %5, %5}, p;\n\t}"
      ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(0u)
      : "memory");
}

// Sixteen TMEM lanes x 32 columns: thread (g, q) = (lane / 4, lane % 4) stores, of each group of eight
// columns, columns 2 q, 2 q + 1 of lanes g (v[0], v[1]) and g + 8 (v[2], v[3]).
__device__ __forceinline__ void tmem_st_16x256b_x4(uint32_t taddr, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.16x256b.x4.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};"
      ::AKL_I8(v, 0), AKL_I8(v, 8), "r"(taddr)
      : "memory");
}
// Values of an asynchronous TMEM load exist from here on (behind its wait).
__device__ __forceinline__ void pin32(uint32_t (&v)[32]) {
#pragma unroll
  for (int i = 0; i < 32; ++i) asm volatile("" : "+r"(v[i]));
}

// What this CTA's share holds next: position tile p, kv head j, row tiles [r, r_end).
struct Piece {
  int p, j, r, r_end;
  bool begins;
};
// The CTA's first piece and the number of units in its share.
__device__ __forceinline__ Piece first_piece(const Units& u, long long from, long long to, int& count) {
  Piece x;
  int p, j, skip;
  const long long begin = u.locate(from, x.p, x.j, skip);
  if (to < u.total) {
    int more;
    count = static_cast<int>(u.locate(to, p, j, more) - begin);
  } else {
    int last;
    count = static_cast<int>(u.locate(u.total - 1, p, j, last) + 1 - begin);      // the sequence ends with a unit
  }
  x.begins = skip == 0;
  x.r = u.first_tile(x.p) + skip;
  x.r_end = static_cast<int>(min(static_cast<long long>(u.tiles), static_cast<long long>(x.r) + count));
  return x;
}
// The piece behind x; `left` units of the share remain, at least one.
__device__ __forceinline__ Piece next_piece(const Units& u, Piece x, long long left) {
  if (++x.j == u.heads) { x.j = 0; ++x.p; }
  x.begins = true;
  x.r = u.first_tile(x.p);
  x.r_end = static_cast<int>(min(static_cast<long long>(u.tiles), x.r + left));
  return x;
}

// 2^(s factor - lse) of 32 columns, added up; columns outside [low, high) count nothing.  The exponential
// unit is busy 75 % of the time, as the tensor pipe is.  (Every fourth pair, or every eighth, as a polynomial
// on the FMA pipe was measured: 172 us became 179 and 173, the issue slots then bind.)
template <int KV, bool kMask>
__device__ __forceinline__ float add_columns(const uint32_t (&v)[32], const float* rows, float factor, int low, int high) {
  f2 acc[2] = {pack2(0.f, 0.f), pack2(0.f, 0.f)};
#pragma unroll
  for (int i = 0; i < 32; i += 4) {
    const float4 l = *reinterpret_cast<const float4*>(rows + kRows + i);
    float4 f = make_float4(factor, factor, factor, factor);
    if (KV == AKL_KV_FP16) f = *reinterpret_cast<const float4*>(rows + i);
    float p[4];
    unpack2(fma2p(pack2(__uint_as_float(v[i]), __uint_as_float(v[i + 1])), pack2(f.x, f.y), pack2(l.x, l.y)), p[0], p[1]);
    unpack2(fma2p(pack2(__uint_as_float(v[i + 2]), __uint_as_float(v[i + 3])), pack2(f.z, f.w), pack2(l.z, l.w)), p[2], p[3]);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      p[e] = ex2(p[e]);
      if (kMask && !(i + e >= low && i + e < high)) p[e] = 0.f;
    }
    acc[0] = add2p(acc[0], pack2(p[0], p[1]));
    acc[1] = add2p(acc[1], pack2(p[2], p[3]));
  }
  float a, b;
  unpack2(add2p(acc[0], acc[1]), a, b);
  return a + b;
}

template <int KV>
__global__ void __launch_bounds__(kThreads, 1) extend_weights_kernel(const akl_weights_t c, const Units u, const Work w) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* const smem_gen = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const uint32_t smem = smem_u32(smem_gen);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const Bars bars{smem + kOffBar};
  volatile int* aborted = reinterpret_cast<volatile int*>(smem_gen + kOffMisc);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem_gen + kOffMisc + 16);
  const Wait wait{w.status, aborted};
  if (threadIdx.x == 0) {
    *aborted = 0;
    for (int s = 0; s < kStages; ++s) {
      mbar_init(bars.q_full(s), 1);
      mbar_init(bars.q_empty(s), kEpiWarps + 2);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(bars.d_full(s), 1);
      mbar_init(bars.d_empty(s), kEpiWarps);
    }
    mbar_init(bars.k_full(), kEpiWarps);
    mbar_init_fence();
  }
  if (warp == kEpiWarps) tmem_alloc(smem_u32(tmem_slot), kTmemCols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  const long long first = u.total * blockIdx.x / u.ctas;
  int count;
  const Piece begin = first_piece(u, first, u.total * (blockIdx.x + 1) / u.ctas, count);

  if (warp >= kEpiWarps) {
    if (lane == 0) {
      Piece x = begin;
      if (warp == kEpiWarps + 2) {
        // ---- row tiles, one bulk copy each
        asm volatile("griddepcontrol.wait;" ::: "memory");        // they are packed by the launch before
        int issued = 0;
        for (int it = 0; it < count; ++it) {
          const int s = it % kStages;
          if (it >= kStages && (!wait(bars.q_empty(s), (it / kStages - 1) & 1) || *aborted)) break;
          mbar_expect_tx(bars.q_full(s), kTileBytes);
          bulk_g2s(smem + s * kTileBytes, w.images + (static_cast<long long>(x.j) * u.tiles + x.r) * kTileBytes, kTileBytes, bars.q_full(s));
          issued = it + 1;
          if (++x.r == x.r_end && issued < count) x = next_piece(u, x, count - issued);
        }
        // no copy may outlive the CTA: they land (or the limit passes) before this thread ends
        for (int it = issued > kStages ? issued - kStages : 0; it < issued; ++it) {
          const long long t0 = clock64();
          while (!mbar_try_wait(bars.q_full(it % kStages), (it / kStages) & 1) && clock64() - t0 < kWaitCycles) {}
        }
      } else {
        // ---- products of one set of 128 positions: 16 of K = 16 per row tile.  Two threads issue, for an
        // issue takes its thread longer than the product takes the tensor pipe.
        const int sub = warp - kEpiWarps;
        const uint32_t d = tmem + kColD + sub * 128, a = tmem + kColK + sub * 128;
        int piece = 0;
        bool fresh = true;
        for (int it = 0; it < count; ++it) {
          const int s = it % kStages;
          if (fresh && !wait(bars.k_full(), piece & 1)) break;
          if (!wait(bars.q_full(s), (it / kStages) & 1)) break;
          if (it > 0 && !wait(bars.d_empty(sub), (it - 1) & 1)) break;
          tc_fence_after();
#pragma unroll
          for (int k = 0; k < 16; ++k)
            mma_16_ts(d, a + k * 8, smem_desc_k128(smem + s * kTileBytes + (k >> 2) * kPlaneBytes + (k & 3) * 32),
                      idesc_16<KV>(128, kRows), k > 0 ? 1u : 0u);
          tc_commit(bars.d_full(sub));
          tc_commit(bars.q_empty(s));
          fresh = ++x.r == x.r_end;
          if (fresh && it + 1 < count) {
            x = next_piece(u, x, count - it - 1);
            ++piece;
          }
        }
      }
    }
  } else {
    // ---- positions: lane set `warp & 3` of both halves of the tile, columns 32 (warp / 4) ..  Four warps
    // a scheduler: with two the exponential unit idled a third of the time behind their latencies.
    const int quarter = warp & 3, side = warp >> 2;
    const int at = quarter * 32 + lane;
    const uint32_t lanes = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
    const float factor = c.sm_scale * (kLog2e * kGiveBack);
    float* red = reinterpret_cast<float*>(smem_gen + kOffRed);
    Piece x = begin;
    int it = 0, piece = 0, slot_tile = -1, stage = 0;
    uint32_t q_phase = 0;
    long long slot = -1;             // of this lane's position in the tile
    auto slot_of = [&](int p, int sub) {
      const long long n = static_cast<long long>(p) * kPos + sub * 128 + at;
      long long v = -1;
      if (n < c.N) v = load_index(c.idx, c.idx_dtype, n);
      return v < c.pool_rows ? v : -1ll;
    };
    bool ok = true;
    while (it < count) {
      // K of 32 positions, channels 128 (side & 1) .., into TMEM.  Every product of the piece before has been
      // waited for.  Four lanes share a row, so that a load of the warp reads 64 bytes of eight rows (a row
      // per lane would be 32 lines a load); 16-lane stores put two words of a lane side by side, so the
      // channels of a row lie in TMEM as pack_rows_kernel lays those of Q (a product does not mind their order).
      {
        const int sub = side >> 1, part = side & 1;
        if (x.p != slot_tile) {
          slot_tile = x.p;
          slot = slot_of(x.p, sub);
        }
        tc_fence_after();
#pragma unroll
        for (int b = 0; b < 2; ++b) {                  // positions 16 b .. of the warp's
          uint32_t v[2][16];                           // [channels 64 ..][pairs of words: row, row + 8, ..]
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const long long row = __shfl_sync(0xffffffffu, slot, b * 16 + e * 8 + (lane >> 2));
            const uint4* src = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(c.k_pool) + (row < 0 ? 0 : row) * c.k_stride + x.j * 256) +
                               part * 16 + (lane & 3);
#pragma unroll
            for (int i = 0; i < 4; ++i) {              // 64 bytes: two groups of eight columns
              uint4 raw = make_uint4(0u, 0u, 0u, 0u);
              if (row >= 0) raw = __ldg(src + i * 4);
              uint32_t* dst = &v[i >> 1][(i & 1) * 8 + e * 2];
              dst[0] = raw.x;
              dst[1] = raw.y;
              dst[4] = raw.z;
              dst[5] = raw.w;
            }
          }
#pragma unroll
          for (int i = 0; i < 2; ++i)
            tmem_st_16x256b_x4(tmem + (static_cast<uint32_t>(quarter * 32 + b * 16) << 16) + kColK + sub * 128 + part * 64 + i * 32, v[i]);
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bars.k_full());
        // the next piece's rows (a lane's own, two lines of this warp's channels) on their way to L2
        const int left = count - it - (x.r_end - x.r);
        if (left > 0) {
          const Piece y = next_piece(u, x, left);
          if (y.p != slot_tile) {
            slot_tile = y.p;
            slot = slot_of(y.p, sub);
          }
          if (slot >= 0) {
            const uint16_t* row = static_cast<const uint16_t*>(c.k_pool) + slot * c.k_stride + y.j * 256 + part * 128;
            asm volatile("prefetch.global.L2 [%0];" ::"l"(row));
            asm volatile("prefetch.global.L2 [%0];" ::"l"(row + 64));
          }
        }
      }
      // Packed rows from (n - prefix) group on see position n, and the last tile may be short.  Of 32
      // columns against the warp's 32 positions nearly always all count or none.
      float sum[2] = {0.f, 0.f};
      int low[2], clear[2];            // first packed row that the warp's first position sees; first that all of them see
#pragma unroll
      for (int sub = 0; sub < 2; ++sub) {
        const long long n0 = static_cast<long long>(x.p) * kPos + sub * 128 + quarter * 32 - c.prefix;
        low[sub] = static_cast<int>(max(-(1ll << 29), min(1ll << 30, n0 * u.group)));
        clear[sub] = low[sub] + 31 * u.group;
      }
      const int packed = c.T * u.group;
      int col0 = x.r * kRows + side * 32;
      const uint32_t d_lanes = lanes + kColD + side * 32;
#pragma unroll 1
      for (; x.r < x.r_end; ++x.r, ++it, col0 += kRows) {
        if (ok) ok = wait(bars.q_full(stage), q_phase);
        const float* rows = reinterpret_cast<const float*>(smem_gen + stage * kTileBytes + kImage) + side * 32;
#pragma unroll
        for (int sub = 0; sub < 2; ++sub) {
          if (ok) ok = wait(bars.d_full(sub), it & 1);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) continue;
          tc_fence_after();
          uint32_t v[32];
          tmem_ld32(d_lanes + sub * 128, v);
          tmem_wait_ld();
          pin32(v);
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(bars.d_empty(sub));
          if (col0 + 32 <= packed && clear[sub] <= col0) sum[sub] += add_columns<KV, false>(v, rows, factor, 0, 32);
          else if (low[sub] < col0 + 32) sum[sub] += add_columns<KV, true>(v, rows, factor, low[sub] + lane * u.group - col0, packed - col0);
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(bars.q_empty(stage));
        if (++stage == kStages) { stage = 0; q_phase ^= 1; }
      }
      // the four quarters of the columns meet; a piece's buffer is used again two pieces, so one barrier, later
      if (!ok) sum[0] = sum[1] = __int_as_float(0x7FC00000);
      float* meet = red + (piece & 1) * 3 * kPos;
      if (side > 0) {
        meet[(side - 1) * kPos + at] = sum[0];
        meet[(side - 1) * kPos + 128 + at] = sum[1];
      }
      asm volatile("bar.sync 1, %0;" ::"n"(kEpiWarps * 32) : "memory");
      if (side == 0) {
        float* dst = x.begins ? w.sums + static_cast<long long>(x.j) * w.pos_cap + static_cast<long long>(x.p) * kPos
                              : w.more + static_cast<long long>(blockIdx.x) * kPos;
#pragma unroll
        for (int sub = 0; sub < 2; ++sub) {
          const float* m = meet + sub * 128 + at;
          dst[sub * 128 + at] = (sum[sub] + m[0]) + (m[kPos] + m[2 * kPos]);
        }
      }
      ++piece;
      if (it < count) x = next_piece(u, x, count - it);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kEpiWarps) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

// One CTA per position tile: heads in order, of each the piece that begins it and those that go on.
__global__ void __launch_bounds__(kPos) add_pieces_kernel(const akl_weights_t c, const Units u, const Work w) {
  __shared__ int sm_from[kMaxHeads], sm_to[kMaxHeads];
  const int p = blockIdx.x;
  const long long n = static_cast<long long>(p) * kPos + threadIdx.x;
  const int units = u.count(p);
  if (threadIdx.x < u.heads) {
    // CTAs whose share begins behind the first unit of (p, head): floor(total i / ctas) in [at + 1, at + units)
    const long long at = u.start(p) + static_cast<long long>(threadIdx.x) * (units + u.piece) + u.piece;
    sm_from[threadIdx.x] = static_cast<int>(((at + 1) * u.ctas + u.total - 1) / u.total);
    sm_to[threadIdx.x] = static_cast<int>(min(u.ctas, ((at + units) * u.ctas + u.total - 1) / u.total));
  }
  bool there = false;
  if (n < c.N) {
    const long long slot = load_index(c.idx, c.idx_dtype, n);
    there = slot >= 0 && slot < c.pool_rows;
  }
  __syncthreads();
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (n >= c.N) return;
  const float old = c.weight_decay == 0.f ? 0.f : c.weights[n];
  float part[kMaxHeads];
#pragma unroll
  for (int j = 0; j < kMaxHeads; ++j) {
    part[j] = 0.f;
    if (j < u.heads && units > 0 && there) {
      part[j] = w.sums[static_cast<long long>(j) * w.pos_cap + n];
      for (int i = sm_from[j]; i < sm_to[j]; ++i) part[j] += w.more[static_cast<long long>(i) * kPos + threadIdx.x];
    }
  }
  float total = 0.f;
#pragma unroll
  for (int j = 0; j < kMaxHeads; ++j) total += part[j];
  c.weights[n] = c.weight_decay == 0.f ? total : fmaf(c.weight_decay, old, total);
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
  const int64_t rows = c->T, heads = c->q_heads, positions = c->N;
  const Span output = {c->weights, 1, positions * 4, 1};
  const Span inputs[4] = {{c->q, rows, heads * 512, c->q_stride * 2},
                          {c->k_pool, c->pool_rows, static_cast<int64_t>(c->kv_heads) * 512, c->k_stride * 2},
                          {c->idx, 1, positions * index_bytes(c->idx_dtype), 1},
                          {c->lse, 1, rows * heads * 4, 1}};
  return outputs_meet(&output, 1, inputs, 4) ? AKL_ERR_INVALID : AKL_OK;
}

template <int KV>
int launch_weights(const akl_weights_t& c, const Units& u, const Work& w, uint8_t* images, cudaStream_t s) {
  static std::atomic<bool> configured[64];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && !(dev >= 0 && dev < 64 && configured[dev].load(std::memory_order_acquire))) {
    e = cudaFuncSetAttribute(extend_weights_kernel<KV>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
    if (e == cudaSuccess && dev >= 0 && dev < 64) configured[dev].store(true, std::memory_order_release);
  }
  if (e == cudaSuccess) {
    pack_rows_kernel<KV><<<dim3(u.tiles, c.kv_heads), 256, 0, s>>>(c, images, u.tiles);
    e = cudaGetLastError();
  }
  // the launches behind the first may be set up while the one before still runs
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(u.ctas));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kSmem;
  cfg.stream = s;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  if (e == cudaSuccess) e = cudaLaunchKernelEx(&cfg, extend_weights_kernel<KV>, c, u, w);
  cfg.gridDim = dim3(static_cast<unsigned>(u.ptiles));
  cfg.blockDim = dim3(kPos);
  cfg.dynamicSmemBytes = 0;
  if (e == cudaSuccess) e = cudaLaunchKernelEx(&cfg, add_pieces_kernel, c, u, w);
  if (e != cudaSuccess) { note_cuda_error(e, "extend_weights_kernel"); return AKL_ERR_CUDA; }
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
  int sms = 0;
  if ((rc = device_sm_count(&sms)) != AKL_OK) return rc;
  uint8_t* ws = static_cast<uint8_t*>(c->workspace);
  Units u;
  u.group = c->q_heads / c->kv_heads;
  u.heads = c->kv_heads;
  u.tiles = static_cast<int>((static_cast<int64_t>(c->T) * u.group + kRows - 1) / kRows);
  u.ptiles = static_cast<int>((static_cast<int64_t>(c->N) + kPos - 1) / kPos);
  u.prefix = c->prefix;
  u.full = std::min(u.ptiles, c->prefix / kPos + 1);
  // A K tile takes about four units' time to come in, which counts where row tiles are many: beside the
  // diagonal a share then has up to ten pieces, elsewhere two.  (2048 rows, 8192 before them: 180 us at
  // 2, 172 at 4, 170 at 6; with few units a share would be a K tile and no row to go with it.)
  u.piece = 0;
  u.total = u.start(u.ptiles);
  u.ctas = std::min<long long>(std::min(sms, kMaxCtas), u.total);
  if (u.total >= 16 * u.ctas) {
    u.piece = 4;
    u.total = u.start(u.ptiles);
  }
  Work w;
  w.images = ws + L.off_q;
  w.pos_cap = static_cast<int>((static_cast<int64_t>(c->plan.max_kv_len) + kPos - 1) / kPos * kPos);
  w.sums = reinterpret_cast<float*>(ws + L.off_parts);
  w.more = reinterpret_cast<float*>(ws + L.off_parts + align1k(static_cast<uint64_t>(w.pos_cap) * c->kv_heads * 4));
  w.status = reinterpret_cast<int*>(ws + L.off_status);
  return c->kv_dtype == AKL_KV_BF16 ? launch_weights<AKL_KV_BF16>(*c, u, w, ws + L.off_q, static_cast<cudaStream_t>(stream))
                                    : launch_weights<AKL_KV_FP16>(*c, u, w, ws + L.off_q, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
