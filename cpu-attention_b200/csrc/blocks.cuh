// Moving blocks of a paged cache: copies of many tensors in one launch, and the
// plan that packs the blocks in use at the front of the pool.
//
// copy_blocks_kernel: pair (src, dst) of every tensor [num_blocks, ...]; a CTA
// copies one block of one tensor, or (blocks up to 1 KiB: scales) 64 pairs of it.
// Bound by HBM: each byte read and written once; 8 words a thread in flight
// (4 at twice the warps: 44 us; 512 threads: 48 us; 128: 34 us). 65 blocks of 48
// tensors (204 MB both ways) in 34 us, 6.0 TB/s. Few large blocks leave most SMs
// without work: one pair of 1 MiB blocks in 30 tensors takes 33 us.
//
// compact_plan_kernel (one CTA): with U the blocks that the page table's rows
// use and n = |U|, the k-th smallest member of U that is >= n goes to the k-th
// smallest id < n that is not in U; everything else stays. The sources and
// the destinations are disjoint, so the copies need no order. A block
// several rows share moves once. U is a bitmap in shared memory; ranks are
// prefix sums of its population counts. A pool of 2111 blocks is planned in 9.5
// us; with its moves (24 8-bit caches and their scales, 387 MB) 70 us (a move's ids
// loaded only once the last one's bytes are written: 77 us). What does not fit the
// CTA's registers of a table (4096 entries) is read twice by this one CTA: 256 x
// 2048 entries take 587 us in all, their moves' bytes 16 of them.
#pragma once

#include "common.cuh"

namespace ca {

constexpr int kCopyTensors = 128;  // tensors per launch
constexpr int kCopyThreads = 256;
constexpr int kPlanThreads = 1024;
constexpr int kPlanHeld = 4;  // table entries a thread reads once; those behind are read twice
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

struct CopyPair {
  long long src, dst;
};
__device__ __forceinline__ CopyPair copy_pair(const CopyParams& p, long long pair) {
  CopyPair c;
  if (p.pairs) {
    c.src = __ldg(p.pairs + 2 * pair);
    c.dst = __ldg(p.pairs + 2 * pair + 1);
  } else {  // (the plan may still write them as the launch begins: not by the read-only path)
    c.src = p.moves[2 * pair];
    c.dst = p.moves[2 * pair + 1];
  }
  return c;
}
// Whether it is copied: negative ids are padding, one beyond the pool is flagged.
__device__ __forceinline__ bool copy_counts(const CopyParams& p, const CopyPair& c) {
  if (c.src < 0 || c.dst < 0) return false;
  if (c.src >= p.num_blocks || c.dst >= p.num_blocks) {
    if (p.status) atomicOr(p.status, CA_STATUS_SLOT);
    return false;
  }
  return c.src != c.dst;
}

template <typename W>
__device__ __forceinline__ void copy_group(const CopyParams& p, char* base, int bytes, long long first, int pairs) {
  const int per = bytes / (int)sizeof(W);
  for (int x = threadIdx.x; x < pairs * per; x += kCopyThreads) {
    const int k = x / per, w = x - k * per;
    const CopyPair c = copy_pair(p, first + k);
    if (!copy_counts(p, c)) continue;
    reinterpret_cast<W*>(base + c.dst * bytes)[w] = reinterpret_cast<const W*>(base + c.src * bytes)[w];
  }
}

__global__ void __launch_bounds__(kCopyThreads) copy_blocks_kernel(const __grid_constant__ CopyParams p) {
  asm volatile("griddepcontrol.wait;" ::: "memory");  // behind a plan: its moves are written
  const long long n = p.pairs ? p.n : __ldcg(p.count);
  const int small = p.tensors - p.large;
  const long long groups = (n + kCopyGroup - 1) / kCopyGroup;
  // units: a pair of a tensor with large blocks, then a group of pairs of one with
  // small blocks. The next unit's pair is loaded while this one's bytes move.
  const long long many = n * p.large;
  auto pair_of = [&](long long u) -> long long { return u <= 0xffffffffLL ? (unsigned)u / (unsigned)p.large : u / p.large; };
  long long u = blockIdx.x;
  CopyPair next{-1, -1};
  if (u < many) next = copy_pair(p, pair_of(u));
  for (; u < many; u += gridDim.x) {
    const CopyPair c = next;
    const int t = (int)(u - pair_of(u) * p.large);
    if (u + gridDim.x < many) next = copy_pair(p, pair_of(u + gridDim.x));
    if (!copy_counts(p, c)) continue;
    const long long bytes = p.bytes[t];
    const char* s = p.base[t] + c.src * bytes;
    char* d = p.base[t] + c.dst * bytes;
    const unsigned long long at = (unsigned long long)p.base[t] | (unsigned long long)bytes;
    if ((at & 15) == 0)
      copy_words<uint4>(d, s, bytes);
    else if ((at & 3) == 0)
      copy_words<uint32_t>(d, s, bytes);
    else
      copy_words<uint8_t>(d, s, bytes);
  }
  for (; u < many + groups * small; u += gridDim.x) {
    const long long group = (u - many) / small;
    const int t = p.large + (int)(u - many - group * small);
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

struct CompactParams {
  const int* page_table;  // [B, width]
  const int* lens;
  const int* reserved;  // [B] lengths up to which pages are kept (at least lens), or NULL
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

// The block of entry e of the table when its page holds a token that counts or
// is reserved for one to come, else -1. The window ends at the tokens that are
// there, whatever is reserved. (The length and the entry are loaded side by side.)
__device__ __forceinline__ int compact_live(const CompactParams& p, long long e, bool flag) {
  const int b = __ldg(p.page_table + e);
  const int i = (int)(e <= 0xffffffffLL ? (unsigned)e / (unsigned)p.width : e / p.width);
  const long long at = (e - (long long)i * p.width) * p.page;
  long long L = __ldg(p.lens + i);
  const long long cap = (long long)p.width * p.page;
  long long end = p.reserved && L >= 0 ? max(L, (long long)__ldg(p.reserved + i)) : L;
  if (end > cap) {
    if (flag && p.status) atomicOr(p.status, CA_STATUS_LENS);
    end = cap;
    L = min(L, cap);
  }
  if (at >= end || !(p.left < 0 || at + p.page > L - 1 - p.left || at < p.sinks)) return -1;
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
  int held[kPlanHeld];
#pragma unroll
  for (int k = 0; k < kPlanHeld; ++k) {
    const long long e = threadIdx.x + k * kPlanThreads;
    held[k] = e < entries ? compact_live(p, e, true) : -1;
    if (held[k] >= 0) atomicOr(plan_bits + (held[k] >> 5), 1u << (held[k] & 31));
  }
  for (long long e = threadIdx.x + kPlanHeld * kPlanThreads; e < entries; e += kPlanThreads) {
    const int b = compact_live(p, e, true);
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
  // an entry no row can use becomes -1, and so does a bad one (flagged above)
  auto placed = [&](int b) { return b < 0 ? -1 : (b >= n ? p.place[b] : b); };
#pragma unroll
  for (int k = 0; k < kPlanHeld; ++k) {
    const long long e = threadIdx.x + k * kPlanThreads;
    if (e < entries) p.new_table[e] = placed(held[k]);
  }
  for (long long e = threadIdx.x + kPlanHeld * kPlanThreads; e < entries; e += kPlanThreads)
    p.new_table[e] = placed(compact_live(p, e, false));
}

}  // namespace ca
