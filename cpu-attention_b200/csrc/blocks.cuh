// Moving blocks of a paged cache: copies of many tensors in one launch, and the
// plan that packs the blocks in use at the front of the pool.
//
// copy_blocks_kernel: pair (src, dst) of every tensor [num_blocks, ...]; a CTA
// copies one block of one tensor, or (blocks up to 1 KiB: scales) 64 pairs of it.
// Bound by HBM: each byte read and written once; 8 words a thread in flight. 65
// blocks of 48 tensors (204 MB both ways) in 33 us, 6.1 TB/s.
//
// compact_plan_kernel (one CTA): with U the blocks that the page table's rows
// use and n = |U|, the k-th smallest member of U that is >= n goes to the k-th
// smallest id < n that is not in U; everything else stays. The sources and
// the destinations are disjoint, so the copies need no order. A block
// several rows share moves once. U is a bitmap in shared memory; ranks are
// prefix sums of its population counts. A pool of 2111 blocks is planned in 9.5
// us; with its moves (24 8-bit caches and their scales, 387 MB) 69 us.
#pragma once

#include "common.cuh"

namespace ca {

constexpr int kCopyTensors = 128;  // tensors per launch
constexpr int kCopyThreads = 256;
constexpr int kPlanThreads = 1024;
constexpr int kPlanMaxBlocks = 1 << 20;  // a 128 KiB bitmap

constexpr int kCopySmall = 1024;  // bytes up to which a CTA takes kCopyGroup pairs of a tensor at a time
constexpr int kCopyGroup = 64;

struct CopyParams {
  char* base[kCopyTensors];       // those with large blocks first
  long long bytes[kCopyTensors];  // per block
  int tensors, large;
  long long num_blocks;
  const long long* pairs;  // [n][2] (src, dst), or NULL: moves
  const int* moves;        // [n][2]
  const int* count;        // moves: n, on the device
  long long n;             // pairs: n
  int* status;
};

// 8 words a thread in flight.
template <typename W>
__device__ __forceinline__ void copy_words(char* dst, const char* src, long long bytes) {
  const W* s = reinterpret_cast<const W*>(src);
  W* d = reinterpret_cast<W*>(dst);
  const long long n = bytes / (long long)sizeof(W);
  constexpr int U = 8;
  for (long long x0 = 0; x0 < n; x0 += U * kCopyThreads) {
    const int left = (int)min((long long)U * kCopyThreads, n - x0);
    W r[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int x = threadIdx.x + u * kCopyThreads;
      if (x < left) r[u] = s[x0 + x];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int x = threadIdx.x + u * kCopyThreads;
      if (x < left) d[x0 + x] = r[u];
    }
  }
}

// (src, dst) of a pair; false when it is left out.
__device__ __forceinline__ bool copy_pair(const CopyParams& p, long long pair, long long* src, long long* dst) {
  if (p.pairs) {
    *src = __ldg(p.pairs + 2 * pair);
    *dst = __ldg(p.pairs + 2 * pair + 1);
    if (*src < 0 || *dst < 0) return false;  // padding
    if (*src >= p.num_blocks || *dst >= p.num_blocks) {
      if (p.status) atomicOr(p.status, CA_STATUS_SLOT);
      return false;
    }
  } else {
    *src = __ldcg(p.moves + 2 * pair);  // (the plan may still write them as the launch begins)
    *dst = __ldcg(p.moves + 2 * pair + 1);
  }
  return *src != *dst;
}

template <typename W>
__device__ __forceinline__ void copy_group(const CopyParams& p, char* base, int bytes, long long first, int pairs) {
  const int per = bytes / (int)sizeof(W);
  for (int x = threadIdx.x; x < pairs * per; x += kCopyThreads) {
    const int k = x / per, w = x - k * per;
    long long src, dst;
    if (!copy_pair(p, first + k, &src, &dst)) continue;
    reinterpret_cast<W*>(base + dst * bytes)[w] = reinterpret_cast<const W*>(base + src * bytes)[w];
  }
}

__global__ void __launch_bounds__(kCopyThreads) copy_blocks_kernel(const __grid_constant__ CopyParams p) {
  asm volatile("griddepcontrol.wait;" ::: "memory");  // behind a plan: its moves are written
  const long long n = p.pairs ? p.n : __ldcg(p.count);
  const int small = p.tensors - p.large;
  const long long groups = (n + kCopyGroup - 1) / kCopyGroup;
  // units: a pair of a tensor with large blocks, then a group of pairs of one with small blocks
  for (long long u = blockIdx.x; u < n * p.large + groups * small; u += gridDim.x) {
    if (u < n * p.large) {
      const unsigned long long pair = u <= 0xffffffffLL ? (unsigned)u / (unsigned)p.large : u / p.large;
      const int t = (int)(u - pair * p.large);
      long long src, dst;
      if (!copy_pair(p, pair, &src, &dst)) continue;
      const long long bytes = p.bytes[t];
      const char* s = p.base[t] + src * bytes;
      char* d = p.base[t] + dst * bytes;
      const unsigned long long at = (unsigned long long)p.base[t] | (unsigned long long)bytes;
      if ((at & 15) == 0)
        copy_words<uint4>(d, s, bytes);
      else if ((at & 3) == 0)
        copy_words<uint32_t>(d, s, bytes);
      else
        copy_words<uint8_t>(d, s, bytes);
    } else {
      const long long v = u - n * p.large;
      const long long group = v / small;
      const int t = p.large + (int)(v - group * small);
      const int bytes = (int)p.bytes[t];
      const long long first = group * kCopyGroup;
      const int pairs = (int)min((long long)kCopyGroup, n - first);
      const unsigned long long at = (unsigned long long)p.base[t] | (unsigned long long)bytes;
      if ((at & 15) == 0)
        copy_group<uint4>(p, p.base[t], bytes, first, pairs);
      else if ((at & 3) == 0)
        copy_group<uint32_t>(p, p.base[t], bytes, first, pairs);
      else
        copy_group<uint8_t>(p, p.base[t], bytes, first, pairs);
    }
  }
}

struct CompactParams {
  const int* page_table;  // [B, width]
  const int* lens;
  int* new_table;  // [B, width]
  int* used;       // [1]
  int* moves;      // [num_blocks][2]: the first count[0] are set
  int* count;      // [1]
  int* place;      // [num_blocks]: where a moved block goes
  long long num_blocks;
  int B, width, page;
  int left, sinks;
  int* status;
};

// The block of entry (i, pg) when its page holds a token that counts, else -1.
__device__ __forceinline__ int compact_live(const CompactParams& p, int i, int pg, bool flag, bool* live) {
  long long L = __ldg(p.lens + i);
  const long long cap = (long long)p.width * p.page;
  if (L > cap) {
    if (flag && p.status) atomicOr(p.status, CA_STATUS_LENS);
    L = cap;
  }
  const long long at = (long long)pg * p.page;
  *live = at < L && (p.left < 0 || at + p.page > L - 1 - p.left || at < p.sinks);
  if (!*live) return -1;
  const int b = __ldg(p.page_table + (long long)i * p.width + pg);
  if (b < 0 || b >= p.num_blocks) {
    if (flag && p.status) atomicOr(p.status, CA_STATUS_TABLE);
    return -1;
  }
  return b;
}

// Sum over the CTA before this thread, and the CTA's total.
__device__ __forceinline__ int plan_scan(int x, int* wsum, int* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int incl = warp_scan_i(x, lane);
  __syncthreads();  // wsum of an earlier scan has been read
  if (lane == 31) wsum[warp] = incl;
  __syncthreads();
  if (warp == 0) {
    const int s = warp_scan_i(wsum[lane], lane);
    __syncwarp();
    wsum[lane] = s;
  }
  __syncthreads();
  *total = wsum[31];
  return incl - x + (warp ? wsum[warp - 1] : 0);
}

__global__ void __launch_bounds__(kPlanThreads) compact_plan_kernel(const __grid_constant__ CompactParams p) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  extern __shared__ uint32_t plan_bits[];  // one bit per block
  __shared__ int wsum[32];
  const int words = (int)((p.num_blocks + 31) / 32);
  for (int x = threadIdx.x; x < words; x += kPlanThreads) plan_bits[x] = 0u;
  __syncthreads();
  const long long entries = (long long)p.B * p.width;
  for (long long e = threadIdx.x; e < entries; e += kPlanThreads) {
    const int i = (int)(e / p.width);
    bool live;
    const int b = compact_live(p, i, (int)(e - (long long)i * p.width), true, &live);
    if (b >= 0) atomicOr(plan_bits + (b >> 5), 1u << (b & 31));
  }
  __syncthreads();
  // words [x0, x1) of this thread, in order of the thread
  const int per = (words + kPlanThreads - 1) / kPlanThreads;
  const int x0 = min(words, (int)threadIdx.x * per), x1 = min(words, x0 + per);
  int mine = 0, n, dummy;
  for (int x = x0; x < x1; ++x) mine += __popc(plan_bits[x]);
  plan_scan(mine, wsum, &n);
  // ids below n that are free, ids from n on that are used
  auto below = [&](int x) -> uint32_t {  // the bits of word x whose id is < n
    const int k = n - 32 * x;
    return k >= 32 ? 0xffffffffu : (k <= 0 ? 0u : (1u << k) - 1u);
  };
  int holes = 0, movers = 0;
  for (int x = x0; x < x1; ++x) {
    holes += __popc(~plan_bits[x] & below(x));
    movers += __popc(plan_bits[x] & ~below(x));
  }
  int hole = plan_scan(holes, wsum, &dummy);
  int mover = plan_scan(movers, wsum, &dummy);
  for (int x = x0; x < x1; ++x) {
    for (uint32_t w = ~plan_bits[x] & below(x); w; w &= w - 1) p.moves[2 * hole++ + 1] = 32 * x + __ffs(w) - 1;
    for (uint32_t w = plan_bits[x] & ~below(x); w; w &= w - 1) p.moves[2 * mover++] = 32 * x + __ffs(w) - 1;
  }
  const int count = dummy;  // as many holes as movers
  if (threadIdx.x == 0) {
    *p.used = n;
    *p.count = count;
  }
  __syncthreads();  // (the CTA's writes of moves are visible to it)
  for (int k = threadIdx.x; k < count; k += kPlanThreads) p.place[p.moves[2 * k]] = p.moves[2 * k + 1];
  __syncthreads();
  for (long long e = threadIdx.x; e < entries; e += kPlanThreads) {
    const int i = (int)(e / p.width);
    bool live;
    const int b = compact_live(p, i, (int)(e - (long long)i * p.width), false, &live);
    // an entry no row can use becomes -1, and so does a bad one (flagged above)
    p.new_table[e] = b < 0 ? -1 : (b >= n ? p.place[b] : b);
  }
}

}  // namespace ca
