// Eviction by accumulated weight: the first and last positions of a request and the heaviest of the
// others move to the front of its page-table row in position order.
//
// The weights are compared as 32-bit keys in the order of the floats (NaN as -inf, -0 as 0).  The key of
// the lightest position that stays is found digit by digit -- 11, 11 and 10 bits -- from histograms of the
// keys that share the digits found so far; of the positions with exactly that key the lowest stay.  The
// new place of a position then follows from two counts, of the positions before it that stay for
// certain and of those with that key.
//
// A CTA, or a cluster of them while the requests leave SMs idle, takes a request and keeps the keys of up to
// 32768 positions a CTA in shared memory, so a row that fits is read once and written once, whatever the
// passes.  (In registers, 32 a thread, they were measured first: the unrolled loops spilled, 47 us instead
// of 41 then.)  The histograms and counts of a cluster meet through its shared memory.  Longer rows go through in
// rounds, their weights read again for each digit (from L2).  Rows may be shortened in place: positions only
// move forward, and what a group of 8192 positions a CTA overwrites has been read by all when its barrier opens.
//
// Few bytes and two or three dependent passes.  One request of 139264 positions (16 CTAs) takes 21 to 24 us, of which
// memory would be 0.5: two or three passes with two cluster barriers each, about a microsecond apiece, and the trips to
// L2.  256 requests of up to 32768 take 37 to 38 us, memory 10: about 6 us a request whatever its length and 0.6 ns a
// position, at 60 % of the issue slots.  In place, which needs a barrier a group and leaves the requests in the order
// given, 26 and 41 us.
#include <cooperative_groups.h>

#include <atomic>
#include <mutex>

#include "akl_common.cuh"

namespace akl {

namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 1024, kWarps = kThreads / 32;
constexpr int kStep = 8, kGroups = 4;           // positions of a thread: groups of up to eight steps
constexpr int kCap = kThreads * kStep * kGroups;
constexpr int kBins = 2048;
constexpr int kSorted = kThreads;              // requests that are put in order of their lengths, at most

constexpr uint32_t kStays = 0xFFFFFFFFu;      // key of a position that stays whatever its weight; above every weight's
constexpr uint32_t kNothing = 0u;              // key where there is no position; below every weight's

__device__ __forceinline__ uint32_t weight_key(float w) {
  const uint32_t u = __float_as_uint((w != w ? -INFINITY : w) + 0.f);
  return u ^ (static_cast<uint32_t>(static_cast<int>(u) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float key_weight(uint32_t key) {
  return __uint_as_float((key & 0x80000000u) ? key ^ 0x80000000u : ~key);
}

struct Shared {
  int hist[3][kBins];
  int4 found[3];                   // of each pass, in the cluster's first CTA: digit, how many of it stay, whether all
  uint32_t counts[kGroups][kWarps];  // certain | equal << 16
  uint32_t totals[2][kGroups];     // of this CTA, by parity of the round; read by the cluster
  int warp_sums[kWarps];
  int request;
};

template <typename Slot>
__global__ void __launch_bounds__(kThreads, 1) evict_kernel(const akl_evict_t c, bool longest_first) {
  __shared__ __align__(16) Shared sm;
  cg::cluster_group cluster = cg::this_cluster();
  const int ctas = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int b = blockIdx.x / ctas;
  if (longest_first) {                                  // as the b-th longest, of up to kSorted requests
    // lengths and, where they are equal, the lower index first, as one number; rank by counting the larger ones
    int* order = &sm.hist[0][0];
    int* rank_of = &sm.hist[1][0];
    const int padded = (c.batch + 15) & ~15;
    for (int i = tid; i < padded; i += kThreads) {
      order[i] = i < c.batch ? static_cast<int>(max(0ll, min(static_cast<long long>(c.table_width), load_index(c.kv_lens, c.lens_dtype, i)))) * kSorted + (kSorted - 1 - i) : -1;
      rank_of[i] = 0;
    }
    __syncthreads();
    int wide = kSorted;                                 // threads share a request's comparisons where there are enough
    while (wide >= 2 * c.batch) wide >>= 1;
    const int i = tid & (wide - 1), part = tid / wide, parts = kThreads / wide;
    if (i < c.batch) {
      const int mine = order[i];
      int larger = 0;
#pragma unroll 4
      for (int k = part * 4; k < padded; k += parts * 4) {
        const int4 v = *reinterpret_cast<const int4*>(order + k);
        larger += (v.x > mine ? 1 : 0) + (v.y > mine ? 1 : 0) + (v.z > mine ? 1 : 0) + (v.w > mine ? 1 : 0);
      }
      if (parts > 1) atomicAdd(&rank_of[i], larger);
      else rank_of[i] = larger;
    }
    __syncthreads();
    if (tid < c.batch && rank_of[tid] == b) sm.request = tid;
    __syncthreads();
    b = sm.request;
  }
  const unsigned before = (1u << lane) - 1u;
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
  const int low = full ? c.first : n, high = full ? n - c.last : n;   // positions [low, high) compete, the others stay
  int need = c.keep;                                    // places for them all
  const bool idle = !full && slots_out == slots && weights_out == weights;   // nothing to move
  const int per_round = ctas * kCap;
  const bool once = n <= per_round;
  auto key_of = [&](float w, int i) { return i >= n ? kNothing : (i < low || i >= high ? kStays : weight_key(w)); };

  // A group is side by side in the row, in it a CTA's share, in it a warp's: `each` steps of 32 positions.
  extern __shared__ uint32_t keys[];                    // [groups][warps][each][32]
  int each = 0, groups = 0, base = 0;
  // groups of which the warp has positions; whose keys are all one; some of whose keys are not the weight's bits
  unsigned present = 0, alike = 0, odd = 0;
  auto start_of = [&](int g) { return base + ((g * ctas + rank) * kWarps + warp) * each * 32 + lane; };
  auto keys_of = [&](int g) { return keys + (g * kWarps + warp) * (kStep * 32) + lane; };
  auto load = [&]() {
    const int left = min(per_round, n - base), wide = (left + ctas * kThreads - 1) / (ctas * kThreads);
    each = min(kStep, wide);
    groups = (wide + each - 1) / each;
    present = alike = odd = 0;
#pragma unroll 2
    for (int g = 0; g < groups; ++g) {
      const int at = start_of(g), from = at - lane, to = from + each * 32;
      if (from >= n) break;
      present |= 1u << g;
      const float* src = weights + at;
      uint32_t key[kStep];
      if (each == kStep && to <= n) {
#pragma unroll
        for (int k = 0; k < kStep; ++k) key[k] = __float_as_uint(src[k * 32]);
      } else {
#pragma unroll
        for (int k = 0; k < kStep; ++k) key[k] = k < each && at + k * 32 < n ? __float_as_uint(src[k * 32]) : 0u;
      }
      // the slots are wanted behind the passes: have them in L2 by then
      const int line = from + lane * static_cast<int>(128 / sizeof(Slot));
      if (line < min(to, n)) asm volatile("prefetch.global.L2 [%0];" ::"l"(slots + line));
      uint32_t most = key[0], least = key[0];
#pragma unroll
      for (int k = 1; k < kStep; ++k) {
        most = max(most, key[k]);
        least = min(least, key[k]);
      }
      uint32_t* dst = keys_of(g);
      // weights that are at least 0 and no NaN, in positions that compete, are their own order
      if (each == kStep && from >= low && to <= high && __all_sync(0xffffffffu, most <= 0x7F800000u)) {
#pragma unroll
        for (int k = 0; k < kStep; ++k) dst[k * 32] = key[k] | 0x80000000u;
      } else {
        bool strange = false;
        least = 0xFFFFFFFFu;
        most = 0u;
#pragma unroll
        for (int k = 0; k < kStep; ++k) {
          const uint32_t bits = key[k];
          key[k] = k < each ? key_of(__uint_as_float(bits), at + k * 32) : kNothing;
          strange |= key[k] != kNothing && __float_as_uint(key_weight(key[k])) != bits;
          dst[k * 32] = key[k];
          if (k < each) { most = max(most, key[k]); least = min(least, key[k]); }
        }
        if (__any_sync(0xffffffffu, strange)) odd |= 1u << g;
      }
      const uint32_t first = __shfl_sync(0xffffffffu, least, 0);
      if (__all_sync(0xffffffffu, least == first && most == first)) alike |= 1u << g;
    }
  };
  if (!idle && n > 0 && once) load();

  uint32_t threshold = kStays;
  if (full) {
    for (int i = tid; i < 3 * kBins / 4; i += kThreads) reinterpret_cast<int4*>(sm.hist)[i] = make_int4(0, 0, 0, 0);
    __syncthreads();
    if (ctas > 1) cluster.barrier_arrive();             // waited for before anybody adds to the first CTA's counts
    uint32_t prefix = 0;
    bool exact = false;                                 // every key that begins with prefix stays
#pragma unroll
    for (int pass = 0; pass < 3; ++pass) {
      if (exact) break;
      const int shift = pass == 0 ? 21 : (pass == 1 ? 10 : 0), bits = pass == 2 ? 10 : 11;
      int* hist = sm.hist[pass];
      const uint32_t mask = (1u << bits) - 1u;
      auto add = [&](uint32_t k) {
        const uint32_t d = k >> shift;
        if (pass == 0 ? k != kNothing : (d >> bits) == prefix) atomicAdd(&hist[d & mask], 1);
      };
      if (once) {
        for (int g = 0; g < groups && ((present >> g) & 1u) != 0u; ++g) {
          const uint32_t* key = keys_of(g);
          if ((alike >> g) & 1u) {
            // one key (of weights that nobody has added to yet): one lane adds for all, or 32 would queue
            const uint32_t d = key[0] >> shift;
            if (lane == 0 && (pass == 0 ? key[0] != kNothing : (d >> bits) == prefix)) atomicAdd(&hist[d & mask], 32 * each);
          } else {
#pragma unroll
            for (int k = 0; k < kStep; ++k) add(key[k * 32]);
          }
        }
      } else {
        const int step = ctas * kThreads;
        for (int at = rank * kThreads + tid; at < n; at += kStep * step) {
          float v[kStep];
#pragma unroll
          for (int k = 0; k < kStep; ++k) v[k] = at + k * step < n ? weights[at + k * step] : 0.f;
#pragma unroll
          for (int k = 0; k < kStep; ++k) add(key_of(v[k], at + k * step));
        }
      }
      // the cluster's counts meet in its first CTA, which finds the digit for all
      __syncthreads();
      if (ctas > 1) {
        if (pass == 0) cluster.barrier_wait();
        if (rank > 0) {
          int* to = cluster.map_shared_rank(hist, 0);
          const int2 mine = reinterpret_cast<const int2*>(hist)[tid];
          if (mine.x != 0) atomicAdd(to + 2 * tid, mine.x);
          if (mine.y != 0) atomicAdd(to + 2 * tid + 1, mine.y);
        }
        cluster.sync();
      }
      if (rank == 0) {
        // bins from the top down, two a thread: the one in which the need-th heaviest lies
        const int top = kBins - 2 - 2 * tid;            // its bins are top + 1, top
        const int2 mine = *reinterpret_cast<const int2*>(hist + top);
        const int sum = mine.x + mine.y;
        int upto = sum;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
          const int v = __shfl_up_sync(0xffffffffu, upto, d);
          if (lane >= d) upto += v;
        }
        if (lane == 31) sm.warp_sums[warp] = upto;
        __syncthreads();
        upto += __reduce_add_sync(0xffffffffu, lane < warp ? sm.warp_sums[lane] : 0);
        if (upto >= need && upto - sum < need) {        // one thread
          const int left = need - (upto - sum);
          sm.found[pass] = left > mine.y ? make_int4(top, left - mine.y, left - mine.y == mine.x, 0) : make_int4(top + 1, left, left == mine.y, 0);
        }
      }
      if (ctas > 1) cluster.sync();
      else __syncthreads();
      const int4 found = *cluster.map_shared_rank(&sm.found[pass], 0);
      prefix = (prefix << bits) | static_cast<uint32_t>(found.x);
      need = max(0, found.y);
      exact = found.z != 0;
      threshold = prefix << shift;
    }
    if (exact) need = 0x7fffffff;                       // a whole bin stays: above its lower end, or equal to it
  } else {
    need = 0x7fffffff;
  }
  // (some weights are read again next to their slots, so either one in place needs the barrier)
  const bool in_place = slots_out == slots || weights_out == weights;

  int certain0 = 0, equal0 = 0;                         // in the groups before
  for (int round = 0; base < n && !idle; base += per_round, ++round) {
    if (!once) load();
    for (int g = 0; g < groups; ++g) {
      uint32_t count = 0;
      if ((present >> g) & 1u) {
        const uint32_t* key = keys_of(g);
#pragma unroll
        for (int k = 0; k < kStep; ++k) {
          const uint32_t v = key[k * 32];
          count += (v > threshold ? 1u : 0u) + (v == threshold ? 0x10000u : 0u);
        }
        count = __reduce_add_sync(0xffffffffu, count);
      }
      if (lane == 0) sm.counts[g][warp] = count;
    }
    __syncthreads();
    if (ctas > 1) {
      if (warp < groups) {
        const uint32_t total = __reduce_add_sync(0xffffffffu, sm.counts[warp][lane]);
        if (lane == 0) sm.totals[round & 1][warp] = total;
      }
      cluster.sync();                                   // the totals are there; the round's keys are in shared memory
    }
    for (int g = 0; g < groups; ++g) {
        const int at = start_of(g);
        const bool some = ((present >> g) & 1u) != 0u, again = ((odd >> g) & 1u) != 0u;
        Slot slot[kStep];
        float w[kStep];
        uint32_t key[kStep];
        if (some) {
          const Slot* from = slots + at;
          const uint32_t* src = keys_of(g);
#pragma unroll
          for (int k = 0; k < kStep; ++k) {
            key[k] = src[k * 32];
            if (key[k] != kNothing) slot[k] = from[k * 32];
          }
#pragma unroll
          for (int k = 0; k < kStep; ++k) {
            w[k] = key_weight(key[k]);
            if (again && key[k] != kNothing) w[k] = weights[at + k * 32];
          }
        }
        const uint32_t count = sm.counts[g][lane];
        const uint32_t ahead = __reduce_add_sync(0xffffffffu, lane < warp ? count : 0u);
        int certain = certain0 + static_cast<int>(ahead & 0xFFFFu), equal = equal0 + static_cast<int>(ahead >> 16);
        if (ctas > 1) {
          // sums over a cluster pass 16 bits: certain and equal apart
          const uint32_t theirs = lane < ctas ? *cluster.map_shared_rank(&sm.totals[round & 1][g], lane < ctas ? lane : 0) : 0u;
          const int theirs_c = static_cast<int>(theirs & 0xFFFFu), theirs_e = static_cast<int>(theirs >> 16);
          certain += __reduce_add_sync(0xffffffffu, lane < rank ? theirs_c : 0);
          equal += __reduce_add_sync(0xffffffffu, lane < rank ? theirs_e : 0);
          certain0 += __reduce_add_sync(0xffffffffu, theirs_c);
          equal0 += __reduce_add_sync(0xffffffffu, theirs_e);
          if (in_place) cluster.sync();                 // every slot and weight of the group has been read
        } else {
          const uint32_t total = __reduce_add_sync(0xffffffffu, count);
          certain0 += static_cast<int>(total & 0xFFFFu);
          equal0 += static_cast<int>(total >> 16);
          if (in_place) __syncthreads();
        }
        if (!some) continue;
        // Weights that were read again for each digit agree with what is moved only while nobody else writes them, which
        // a row that two requests name breaks: what is listed as freed must still end inside the request's own entries.
        if (!once && full) {
          const uint32_t mine = sm.counts[g][warp];
          const int upto = min(n, at - lane + each * 32);
          if (upto - certain - static_cast<int>(mine & 0xFFFFu) - min(equal + static_cast<int>(mine >> 16), need) > n - c.keep) continue;
        }
        if ((sm.counts[g][warp] >> 16) == 0u) {         // no key of the warp equals the threshold
          const int equals = min(equal, need);
#pragma unroll
          for (int k = 0; k < kStep; ++k) {
            const bool stay = key[k] > threshold;
            const unsigned stays = __ballot_sync(0xffffffffu, stay);
            const int to = certain + equals + __popc(stays & before);
            certain += __popc(stays);
            if (stay) slots_out[to] = slot[k];
            if (stay) weights_out[to] = w[k];
            if (!stay && key[k] != kNothing) freed[at + k * 32 - to] = slot[k];
          }
        } else {
#pragma unroll
          for (int k = 0; k < kStep; ++k) {
            const bool sure = key[k] > threshold, same = key[k] == threshold;
            const unsigned sures = __ballot_sync(0xffffffffu, sure), sames = __ballot_sync(0xffffffffu, same);
            const int rank_same = equal + __popc(sames & before);
            const int to = certain + __popc(sures & before) + min(rank_same, need);
            const bool stay = sure || (same && rank_same < need);
            certain += __popc(sures);
            equal += __popc(sames);
            if (stay) slots_out[to] = slot[k];
            if (stay) weights_out[to] = w[k];
            if (!stay && key[k] != kNothing) freed[at + k * 32 - to] = slot[k];
          }
        }
      }
    if (!once) __syncthreads();                         // counts are used again
  }
  const int stays = idle ? n : certain0 + min(equal0, need);
  for (int i = stays + rank * kThreads + tid; i < n; i += ctas * kThreads) weights_out[i] = 0.f;
  if (ctas > 1) cluster.sync();                         // nobody reads this CTA's shared memory, or the length, any more
  else __syncthreads();
  if (rank == 0 && tid == 0) {
    if (c.lens_dtype == AKL_IDX_I64) static_cast<long long*>(c.kv_lens_out)[b] = stays;
    else static_cast<int*>(c.kv_lens_out)[b] = stays;
    c.freed_lens[b] = n - stays;
  }
}

// Clusters of 2, 4, 8 and 16 CTAs that the current device holds at once (a cluster lies within one of its
// groups of SMs, so that is less than their number over the cluster's); 0 where it takes none of that size.
struct Held {
  int clusters[4];
};

cudaLaunchConfig_t launch_config(int requests, int ctas, cudaStream_t s, cudaLaunchAttribute* attr) {
  attr->id = cudaLaunchAttributeClusterDimension;
  attr->val.clusterDim.x = static_cast<unsigned>(ctas);
  attr->val.clusterDim.y = attr->val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(requests) * ctas);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kCap * 4;
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cfg;
}

// Once a device: the kernel's attributes, and what the device holds of it.
template <typename Slot>
cudaError_t configure(Held* out) {
  static std::atomic<bool> configured[64];
  static Held held[64];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const bool known = dev >= 0 && dev < 64;
  if (known && configured[dev].load(std::memory_order_acquire)) { *out = held[dev]; return e; }
  e = cudaFuncSetAttribute(evict_kernel<Slot>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (e == cudaSuccess) e = cudaFuncSetAttribute(evict_kernel<Slot>, cudaFuncAttributeMaxDynamicSharedMemorySize, kCap * 4);
  if (e != cudaSuccess) return e;
  for (int i = 0; i < 4; ++i) {
    cudaLaunchAttribute attr;
    const cudaLaunchConfig_t cfg = launch_config(1, 2 << i, nullptr, &attr);
    out->clusters[i] = 0;
    if (cudaOccupancyMaxActiveClusters(&out->clusters[i], evict_kernel<Slot>, &cfg) != cudaSuccess) {
      out->clusters[i] = 0;
      cudaGetLastError();                               // a size that the device does not take is no error of this call
    }
  }
  if (known) {
    static std::mutex mutex;
    std::lock_guard<std::mutex> lock(mutex);
    held[dev] = *out;
    configured[dev].store(true, std::memory_order_release);
  }
  return e;
}

template <typename Slot>
int launch_evict(const akl_evict_t& c, int sms, cudaStream_t s) {
  Held held;
  cudaError_t e = configure<Slot>(&held);
  if (e != cudaSuccess) { note_cuda_error(e, "evict_kernel"); return AKL_ERR_CUDA; }
  // Clusters while the device holds one for every request at once, but at least two steps for every thread of the widest row.
  // (256 requests of up to 32768: 55 us with a CTA each, 71 with two, 108 with four; one of 139264: 177, 102, 58,
  // 30 and 24 us with 1, 2, 4, 8 and 16.  Counted by SMs alone, 8 or 9 requests of 40000 got clusters of 16 of which
  // one had to wait for another to end: 27.6 us, and 13.9 now; 16 requests 25.7 and 17.6, 36 requests 31.9 and 22.7.)
  int ctas = 1;
  for (int i = 0; i < 4 && c.batch <= held.clusters[i] && c.table_width > 2 * kThreads * ctas; ++i) ctas *= 2;
  if (static_cast<int64_t>(c.batch) * ctas >= (1ll << 31)) return AKL_ERR_UNSUPPORTED;
  // More requests than SMs: the long ones first, or the last to start could be the longest (47 us became 41, and 38 with
  // the comparisons that order them shared out among the threads).
  // Every CTA then reads all lengths, so not where the first ones to finish overwrite them.
  const int64_t lens_bytes = static_cast<int64_t>(c.batch) * (c.lens_dtype == AKL_IDX_I64 ? 8 : 4);
  const int64_t apart = static_cast<const char*>(c.kv_lens_out) - static_cast<const char*>(c.kv_lens);
  const bool longest_first = ctas == 1 && c.batch > sms && c.batch <= kSorted && c.table_width < (1 << 21) && (apart >= lens_bytes || -apart >= lens_bytes);
  cudaLaunchAttribute attr;
  const cudaLaunchConfig_t cfg = launch_config(c.batch, ctas, s, &attr);
  e = cudaLaunchKernelEx(&cfg, evict_kernel<Slot>, c, longest_first);
  if (e != cudaSuccess) { note_cuda_error(e, "evict_kernel"); return AKL_ERR_CUDA; }
  return AKL_OK;
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
  if (c->table_width >= (1 << 30)) return AKL_ERR_UNSUPPORTED;      // positions are 32-bit, and rounds run past the end
  if (c->freed_width < c->table_width - c->keep) return AKL_ERR_CAPACITY;
  {
    const int64_t rows = c->table_rows, width = c->table_width, batch = c->batch, item = index_bytes(c->idx_dtype);
    const int64_t lens_bytes = batch * index_bytes(c->lens_dtype);
    const Span table = {c->page_table, rows, width * item, c->table_stride * item}, weights = {c->weights, rows, width * 4, c->weights_stride * 4};
    const Span lens = {c->kv_lens, 1, lens_bytes, 1}, which = {c->rows, 1, batch * index_bytes(c->rows_dtype), 1};
    const Span outputs[5] = {{c->page_table_out, rows, width * item, c->table_out_stride * item},
                             {c->weights_out, rows, width * 4, c->weights_out_stride * 4},
                             {c->kv_lens_out, 1, lens_bytes, 1},
                             {c->freed, batch, static_cast<int64_t>(c->freed_width) * item, c->freed_stride * item},
                             {c->freed_lens, 1, batch * 4, 1}};
    // what is changed in place is read by its own output alone
    const bool same_table = c->page_table_out == c->page_table && c->table_out_stride == c->table_stride;
    const bool same_weights = c->weights_out == c->weights && c->weights_out_stride == c->weights_stride;
    const Span none = {nullptr, 1, 0, 1};
    const Span inputs[4] = {same_table ? none : table, same_weights ? none : weights, c->kv_lens_out == c->kv_lens ? none : lens, which};
    if (outputs_meet(outputs, 5, inputs, 4)) return AKL_ERR_INVALID;
  }
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  int sms = 0;
  const int rc = device_sm_count(&sms);
  if (rc != AKL_OK) return rc;
  return c->idx_dtype == AKL_IDX_I64 ? launch_evict<long long>(*c, sms, s) : launch_evict<int>(*c, sms, s);
}
