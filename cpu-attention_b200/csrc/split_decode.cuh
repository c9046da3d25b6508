// Paged one-token decode over the tokens a row sees, for caches held in 8 bits
// and for sliding windows with a few first tokens that stay visible.
//
// For sequence i of length L (cache_seqlens[i], plus the tokens the call
// appended) and query head h, with x_t = (q . k_t) * scale * log2(e):
//     seen t : t < L and (t >= L - 1 - left or t < sinks)     (left < 0: t < L)
//     out = sum_seen 2^(x_t - m) v_t / l,  l = sum_seen 2^(x_t - m),  m = max_seen x_t
//     lse = (m + log2 l) ln 2;  a row that sees no key gives 0 and -inf.
// An 8-bit cache holds e4m3 codes and one fp32 scale per (block, KV head) for K
// and one for V: k_t = s_k(block) * code_t. Its layout is [block][head][token]
// [dim] for both (codes are read as matrix fragments, no transpose is needed);
// float caches keep the layout of store.cuh.
//
// What bounds it: HBM. 16 tokens of one KV head are 4 KiB of codes at head_dim
// 128 (8 KiB bf16, 16 KiB fp32), read once for up to 8 query rows. Measured
// (one B200, device time, inputs larger than L2): bf16 behind a window of 4096,
// 64 sequences, 32 / 8 heads: 155 us for 1.00 GB (6.5 TB/s, 98% of the measured
// copy rate); 8-bit, 64 sequences to 8191 tokens, 64 / 8 heads: 94 us for 0.54
// GB (5.7 TB/s); 32 sequences of 16 heads to 2047 tokens: 33 us for 136 MB, of
// which about 6 us pass before the first tile is in (lengths, block ids and
// scales, tiles: round trips that wait for one another) and 5 us behind the
// last one (the join); 8-bit tiles are then bound by latency of the chain
// widen, multiply, weigh (40% of issue slots used), not by HBM. fp32 caches
// behind a window of 4096, 32 sequences, 32 / 8 heads of 128: 229 us for 0.99 GB
// (4.3 TB/s); heads of 64: 257 us, of 32: 351 us for as many bytes.
//
// Work: the visible tokens of every item (sequence, KV head, up to 8 of its
// query heads) are cut into tiles of 16 tokens (more for small head_dims); pages
// between the first tokens and the window are neither read nor looked up, so
// their page-table entries may be anything. All tiles are numbered in (sequence,
// head, token) order and every warp of the grid takes an equal, contiguous share
// of them (an item counts two tiles more than it has, for its queries, its join
// and its output), so lengths need not be known on the host and ragged batches
// stay balanced. An item cut by a warp boundary leaves its (m, l, O) in shared
// memory, where its CTA joins the pieces in tile order; one cut by a CTA
// boundary goes through a small global buffer and split_merge_kernel, also in
// order. The result does not depend on timing, and nothing is kept between calls.
//
// A tile in a warp (lane = 4 * g + t), MMA kinds (8-bit and bf16 caches):
//   S^T = K Q^T   m16n8k16: rows = keys, columns = query rows. The lane's K
//                 bytes come straight from global memory as 16-byte vectors
//                 (8-bit) or 8-byte pairs of keys (bf16, K transposed in its
//                 page); the order of the dims is free as long as Q has the same.
//   O^T = V^T P^T m16n8k16: rows = dims. Two V rows of the lane are interleaved
//                 byte by byte (8-bit) or half by half (bf16) so that a register
//                 holds one dim of two keys; P^T is S^T through movmatrix.
//   8-bit codes widen exactly to f16; q is scaled by a power of two per row so
//   that f16 holds it. P enters as one f16 value for bf16 outputs (2^-12 of the
//   weight, against 2^-9 of the output's rounding) and as a value plus its rest
//   for fp32 ones and for bf16 caches; s_v enters with it, its exponent with the
//   weight's, so any scales a user stores are followed.
// fp32 caches run the same tiles on FMAs, through a ring in shared memory.
//
// 8-bit and bf16 caches: loads of tile n+1 are issued as soon as the registers of
// tile n are free: 12 warps an SM with a tile each in flight are 48 KiB, about
// twice what HBM's latency asks for; 8-bit tiles are called into L2 one tile
// earlier still (-8%; four tiles earlier: +4%, eight: +17%). Measured against this (8-bit grouped,
// 96 us then): cp.async into shared memory with four tiles ahead 132 us, TMA
// tiles swizzled for conflict-free fragment loads 96 us, two tiles ahead in
// registers 98 us, the next tile's scores before this one's weights 117 us, 8
// warps an SM 112 us, 16 warps 99 us (spills). mma.sync with e4m3 operands
// widens inside on sm_100a: 134 us. mma.sync and not tcgen05: a tcgen05 tile has
// at least 64 rows, of which at most 8 (16) query rows would be used.
#pragma once

#include <cuda_fp16.h>

#include "common.cuh"

namespace ca {

enum SplitKind { kSplitF32 = 0, kSplitBf16 = 1, kSplitE4m3 = 2 };

constexpr int kSplitWarps = 6;        // warps per CTA
// CTAs per SM of the grid. Two of the 8-bit and bf16 kinds fit; one of the fp32
// kind (130 to 185 KB of shared memory: rings, query rows, pieces), whose grid
// runs as two rounds.
constexpr int kSplitCtasPerSm = 2;
constexpr int kSplitTile = 16;        // tokens per tile
constexpr int kSplitMaxBatch = 1024;  // sequences per launch (their tile counts sit in shared memory)
constexpr int kSplitRing = 16384;     // fp32 caches: bytes of tiles a warp has in flight
constexpr int kSplitMeta = 64;        // tiles whose places a warp keeps
constexpr int kSplitAhead = 2;        // tiles ahead whose lines are brought to L2 (at most 16)
// Weights are kept as 2^(x - m + kUp), m a reference that a column's largest x
// may pass by kSlack before it moves (a vote per tile, no reduction): up to 2^14
// for f16, whose smallest step is then 2^-30 of the reference's weight.
constexpr float kUp = 6.f, kSlack = 8.f;
// Shares of an item's pieces that a join takes side by side: this many when items
// are few and cut into many pieces (one long sequence, 37 pieces: 57 -> 56 us),
// else half (blocks of 512 threads, all resident at once: two or three pieces an
// item, 32 x 16 heads, 35 -> 33 us).
constexpr int kSplitMergeShares = 4;  // at most

struct SplitParams {
  const void* q;
  long long q_stride;  // elements between sequences
  const void* kc;
  const void* vc;
  const float* ks;  // [num_blocks, Hk] scales of 8-bit caches
  const float* vs;
  long long num_blocks;
  const int* lens;
  int extra;  // tokens the call appended at lens[i] before this launch
  const int* page_table;
  long long pt_stride;  // table width
  void* out;            // [B, H, E]
  float* lse;           // [B, H] or NULL
  int B, H, Hk, G;      // G = H / Hk
  int NRG, IH;          // groups of 8 query rows per KV head, items per sequence (Hk * NRG)
  int page;
  int left, sinks;  // left < 0: no window
  float c;          // softmax_scale * log2(e)
  int q_vec;        // q's rows are 16-byte aligned
  float* partial;   // pieces [CTAs][2] of items cut by a CTA boundary
  int* meta;        // [CTAs][4]: the item CTA c leaves unfinished {sequence, item, last CTA, 1}, or {.., 0}
  int* status;
};

// The tokens of one sequence that its row sees, in tiles.
struct SplitSeq {
  int L;         // attended length
  int low;       // first token of the window (<= 0: everything)
  int ts, skip;  // tiles [0, ts), then `skip` tiles that are not read
  int nt;        // tiles read
};

__device__ __forceinline__ SplitSeq split_seq(const SplitParams& p, int i) {
  SplitSeq s;
  const int before = __ldg(p.lens + i);
  // a negative length is a sequence that is skipped
  long long L = before < 0 ? 0LL : (long long)before + p.extra;
  const long long cap = p.pt_stride * (long long)p.page;
  if (L > cap) {
    if (p.status) atomicOr(p.status, CA_STATUS_LENS);
    L = cap;
  }
  s.L = (int)L;
  const int all = (s.L + kSplitTile - 1) / kSplitTile;
  s.low = 0;
  s.ts = 0;
  s.skip = 0;
  if (p.left >= 0) {
    const int low = s.L - 1 - p.left;
    if (low > p.sinks) {
      s.low = low;
      s.ts = (p.sinks + kSplitTile - 1) / kSplitTile;
      s.skip = max(0, low / kSplitTile - s.ts);
    }
  }
  s.nt = all - s.skip;
  return s;
}

// ---- instructions -----------------------------------------------------------
__device__ __forceinline__ uint32_t f16x2_of_e4m3x2(uint32_t two) {  // the low 16 bits
  uint32_t r;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t}" : "=r"(r) : "r"(two));
  return r;
}
__device__ __forceinline__ uint32_t f16x2_of_e4m3x2_hi(uint32_t two) {  // the high 16 bits
  uint32_t r;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, hi;\n\t}" : "=r"(r) : "r"(two));
  return r;
}
template <bool BF16>
__device__ __forceinline__ void split_mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (BF16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t split_transpose(uint32_t x) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
template <bool BF16>
__device__ __forceinline__ uint32_t split_pack(float lo, float hi) {
  uint32_t r;
  if constexpr (BF16)
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
template <bool BF16>
__device__ __forceinline__ void split_unpack(uint32_t w, float* lo, float* hi) {
  if constexpr (BF16) {
    *lo = bf16_lo(w);
    *hi = bf16_hi(w);
  } else {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
    *lo = f.x;
    *hi = f.y;
  }
}

// BYTES from global to this lane's shared memory, or zeros (FULL: never zeros).
template <int BYTES, bool FULL>
__device__ __forceinline__ void split_copy(uint32_t dst, const void* src, bool on) {
  const int n = on ? BYTES : 0;
  if constexpr (FULL && BYTES == 16)
    asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
  else if constexpr (FULL)
    asm volatile("cp.async.ca.shared.global.L2::128B [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(BYTES) : "memory");
  else if constexpr (BYTES == 16)
    asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
  else
    asm volatile("cp.async.ca.shared.global.L2::128B [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(BYTES), "r"(n)
                 : "memory");
}
// The same to registers; lines are read once per item, past L1. (Not by the
// read-only path: an append may still write the cache as the launch begins.)
template <int BYTES, bool FULL>
__device__ __forceinline__ void split_load(uint32_t* r, const void* p, bool on) {
  if constexpr (!FULL) {
#pragma unroll
    for (int x = 0; x < BYTES / 4; ++x) r[x] = 0u;
    if (!on) return;
  }
  if constexpr (BYTES == 16)
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "l"(p));
  else if constexpr (BYTES == 8)
    asm volatile("ld.global.L1::no_allocate.v2.u32 {%0,%1}, [%2];" : "=r"(r[0]), "=r"(r[1]) : "l"(p));
  else
    asm volatile("ld.global.L1::no_allocate.u32 %0, [%1];" : "=r"(r[0]) : "l"(p));
}
__device__ __forceinline__ void split_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void split_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
template <int BYTES>
__device__ __forceinline__ void split_lds(uint32_t* r, const char* p) {
  if constexpr (BYTES == 16) {
    const uint4 x = *reinterpret_cast<const uint4*>(p);
    r[0] = x.x;
    r[1] = x.y;
    r[2] = x.z;
    r[3] = x.w;
  } else if constexpr (BYTES == 8) {
    const uint2 x = *reinterpret_cast<const uint2*>(p);
    r[0] = x.x;
    r[1] = x.y;
  } else {
    r[0] = *reinterpret_cast<const uint32_t*>(p);
  }
}

// ---- shapes of a kind -------------------------------------------------------
// O is held as E/16 groups of 4 registers; group j of lane (g, t) is dims
// dim(j, g), dim(j, g) + 1 of columns 2t, 2t + 1 (registers {dim, col} =
// {0,0}, {0,1}, {1,0}, {1,1}).
template <int KIND, int E>
struct SplitCfg {
  static constexpr bool kF32 = KIND == kSplitF32, kBf16 = KIND == kSplitBf16, k8 = KIND == kSplitE4m3;
  static constexpr int ES = kF32 ? 4 : (kBf16 ? 2 : 1);
  // V: a lane reads RUNS runs of RL dims of each of its keys
  static constexpr int RUNB = (E / 8) * ES < 16 ? (E / 8) * ES : 16;  // bytes per run
  static constexpr int RL = RUNB / ES;
  static constexpr int RUNS = E / (8 * RL);
  static constexpr int NM = E / 16;  // m-tiles of O^T, k-steps of S^T
  static __device__ __forceinline__ int dim(int j, int g) {
    const int d = 2 * j;
    return (d / RL) * (8 * RL) + g * RL + d % RL;
  }
  // K, 8-bit: a lane reads KC vectors of KB bytes of each of its two keys
  static constexpr int KB = E / 4 < 16 ? E / 4 : 16;
  static constexpr int KC = E / (4 * KB);
  // keys of the S^T rows g and g + 8, and of the four P^T columns 2t, 2t+1, 2t+8, 2t+9
  static __device__ __forceinline__ int skey(int half, int g) { return k8 ? g + 8 * half : 2 * g + half; }
  static __device__ __forceinline__ int vkey(int a, int t) {
    return k8 ? 2 * t + (a & 1) + 8 * (a >> 1) : 4 * t + 2 * (a & 1) + (a >> 1);
  }
  static constexpr int kRegs = 4 * NM + 4;  // a piece: O, m[2], l[2]
  static constexpr int kPieceFloats = kRegs * 32;
};

// A warp's shared memory: fp32 caches keep a ring of tiles there (8-bit and
// bf16 ones are loaded to registers, which took 20% less time than copying them
// to shared memory first); the tiles' places and scales; fp32 query rows.
// Groups of 16 tokens a tile has: small heads take several, so that a warp has 4
// KiB (bf16: 4 KiB or more) in flight whatever the head_dim.
template <int KIND, int E>
__host__ __device__ constexpr int split_sub() {
  return KIND == kSplitE4m3 ? 128 / E : (KIND == kSplitBf16 && E == 32 ? 2 : 1);
}

template <int KIND, int E>
struct SplitRing {
  static constexpr bool kRing = KIND == kSplitF32;
  static constexpr int kSide = kSplitTile * E * SplitCfg<KIND, E>::ES;  // bytes of a tile's K (V)
  static constexpr int kStages =
      !kRing ? 1 : (2 * kSide * 8 <= kSplitRing ? 8 : (2 * kSide <= kSplitRing ? kSplitRing / (2 * kSide) : 1));
  static constexpr int kMetaAt = kRing ? kStages * 2 * kSide : 0;
  static constexpr int kScaleAt = kMetaAt + kSplitMeta * 16;
  static constexpr int kQueryAt = kScaleAt + (KIND == kSplitE4m3 ? kSplitMeta * 16 : 0);
  static constexpr int kWarpBytes = kQueryAt + (KIND == kSplitF32 ? 8 * E * 4 : 0);
};

// (m, l, O) of up to 8 query rows over some tiles; columns 2t and 2t + 1 in lane (g, t).
template <int NM>
struct SplitState {
  float o[NM][4];
  float m[2], l[2];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int j = 0; j < NM; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      m[x] = -INFINITY;
      l[x] = 0.f;
    }
  }
  __device__ __forceinline__ void put(float* piece, int lane) const {
#pragma unroll
    for (int j = 0; j < NM; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) piece[(4 * j + r) * 32 + lane] = o[j][r];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      piece[(4 * NM + x) * 32 + lane] = m[x];
      piece[(4 * NM + 2 + x) * 32 + lane] = l[x];
    }
  }
  // joins the tiles of `piece` (which follow this state's)
  __device__ __forceinline__ void join(const float* piece, int lane) {
    float a[2], b[2];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const float mo = piece[(4 * NM + x) * 32 + lane], lo = piece[(4 * NM + 2 + x) * 32 + lane];
      const float mn = fmaxf(m[x], mo);
      const float mu = mn == -INFINITY ? 0.f : mn;
      a[x] = exp2_approx(m[x] - mu);
      b[x] = exp2_approx(mo - mu);
      l[x] = l[x] * a[x] + lo * b[x];
      m[x] = mn;
    }
#pragma unroll
    for (int j = 0; j < NM; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        o[j][r] = o[j][r] * a[r & 1] + piece[(4 * j + r) * 32 + lane] * b[r & 1];
  }
};

// Writes the output rows (and log-sum-exps) of item ih of sequence i.
template <int KIND, typename QT, int E>
__device__ __forceinline__ void split_write(const SplitParams& p, const SplitState<E / 16>& st, int i, int ih,
                                            int lane) {
  using C = SplitCfg<KIND, E>;
  const int g = lane >> 2, t = lane & 3;
  const int kvh = ih / p.NRG, r0 = (ih - kvh * p.NRG) * 8;
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    const int row = r0 + 2 * t + x;
    if (row >= p.G) continue;
    const long long h = (long long)i * p.H + (long long)kvh * p.G + row;
    const float l = st.l[x];
    const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);  // NaN stays
    QT* out = static_cast<QT*>(p.out) + h * E;
#pragma unroll
    for (int j = 0; j < C::NM; ++j) {
      const int d = C::dim(j, g);
      const float a = l == 0.f ? 0.f : st.o[j][x] * inv, b = l == 0.f ? 0.f : st.o[j][2 + x] * inv;
      if constexpr (sizeof(QT) == 2)
        *reinterpret_cast<uint32_t*>(out + d) = split_pack<true>(a, b);
      else
        *reinterpret_cast<float2*>(out + d) = make_float2(a, b);
    }
    if (p.lse && g == 0) p.lse[h] = l == 0.f ? -INFINITY : (st.m[x] + (log2f(l) - kUp)) * 0.69314718055994531f;
  }
}

// ---- a warp's tiles ---------------------------------------------------------
// What a tile's place says: the byte offset of its (block, head) page, the
// tile's first token in the page, and which keys count.
struct SplitPlace {
  long long page;
  int off;
  uint32_t mask;  // bit j: key j is seen (none: the tile is skipped); bit 16: the item's last tile
};

// What every kind of warp shares: the places of its tiles and the walk over them.
template <int KIND, typename QT, int E>
struct SplitWalk {
  using C = SplitCfg<KIND, E>;
  using R = SplitRing<KIND, E>;
  static constexpr int S = R::kStages;
  static constexpr int SUB = split_sub<KIND, E>();
  SplitState<E / 16> st;
  char* sm;  // this warp's shared memory
  int lane;

  // ---- places, 32 at a time: lane l has the 16 tokens l % SUB of tile l / SUB
  // of the next 32 / SUB tiles, which start at tile v0 of item ih0 of sequence i0.
  int i0, ih0, v0;
  int left;  // tiles from there on
  int m_id, m_kvh, m_off;
  uint32_t m_mask;

  // the lane's tile, and its block id
  __device__ __forceinline__ void place_begin(const SplitParams& p, const int* prefix) {
    m_id = -1;
    m_mask = 0u;
    int i = i0, ih = ih0, v = v0;
    if (lane / SUB < left) {
      int rem = lane / SUB;
      int nt = prefix[i + 1] - prefix[i];
      for (;;) {
        const long long here = (long long)(p.IH - ih) * nt - v;  // tiles the sequence still has
        if (rem < here) break;
        rem -= (int)here;
        ++i;
        ih = v = 0;
        nt = prefix[i + 1] - prefix[i];
      }
      v += rem;
      if (v >= nt) {
        const int d = v / nt;
        ih += d;
        v -= d * nt;
      }
      const SplitSeq sq = split_seq(p, i);
      const int u = v * SUB + lane % SUB;  // of the sequence's groups of 16 tokens
      m_kvh = ih / p.NRG;
      if (u < sq.nt) {
        const int r = u < sq.ts ? u : u + sq.skip;
        const int tpp = p.page / kSplitTile, pg = r / tpp;
        const int t0 = r * kSplitTile;
        m_off = (r - pg * tpp) * kSplitTile;
        m_id = __ldg(p.page_table + (long long)i * p.pt_stride + pg);
        // keys [0, L - t0) that are first tokens or in the window
        const int top = min(kSplitTile, sq.L - t0);
        m_mask = (1u << top) - 1u;
        if (sq.low > t0) {
          const int lo = min(kSplitTile, sq.low - t0), first = max(0, min(kSplitTile, p.sinks - t0));
          m_mask &= ~((1u << lo) - 1u) | ((1u << first) - 1u);
        }
      }
      if (v == nt - 1) m_mask |= 1u << 16;
      if (v == 0 && lane % SUB == 0) {  // an item starts here: its query rows will be wanted
        const char* row = reinterpret_cast<const char*>(static_cast<const QT*>(p.q) + (long long)i * p.q_stride +
                                                        ((long long)m_kvh * p.G + (ih - m_kvh * p.NRG) * 8) * E);
        const int bytes = min(8, p.G - (ih - m_kvh * p.NRG) * 8) * E * (int)sizeof(QT);
        for (int x = 0; x < bytes; x += 128) asm volatile("prefetch.global.L1 [%0];" ::"l"(row + x));
      }
      ++v;
      if (v == nt) {
        v = 0;
        ++ih;
      }
    }
    // the next ones start behind lane 31's tile
    i0 = __shfl_sync(0xffffffffu, i, 31);
    ih0 = __shfl_sync(0xffffffffu, ih, 31);
    v0 = __shfl_sync(0xffffffffu, v, 31);
    left -= 32 / SUB;
  }
  // its scales
  float m_sk, m_sv;
  __device__ __forceinline__ void place_scales(const SplitParams& p) {
    m_sk = m_sv = 0.f;
    if (m_mask & 0xffffu) {
      if (m_id < 0 || m_id >= p.num_blocks) {
        if (p.status) atomicOr(p.status, CA_STATUS_TABLE);
        m_mask &= ~0xffffu;
      } else if constexpr (C::k8) {
        m_sk = __ldcg(p.ks + (long long)m_id * p.Hk + m_kvh);
        m_sv = __ldcg(p.vs + (long long)m_id * p.Hk + m_kvh);
      }
    }
  }
  // all of it to shared memory, as the tiles from `base` on
  __device__ __forceinline__ void place_store(const SplitParams& p, int base) {
    const int slot = (base * SUB + lane) & (kSplitMeta - 1);
    SplitPlace a;
    a.page = ((long long)max(m_id, 0) * p.Hk + m_kvh) * (long long)p.page * E * C::ES;
    a.off = m_off;
    a.mask = m_mask;
    if (!(m_mask & 0xffffu)) a.page = a.off = 0;
    if constexpr (C::k8) {
      // s_v as 2^e * g, 1 <= |g| < 2
      const int e = m_sv == 0.f ? -1000 : ilogbf(m_sv);
      const float g = m_sv == 0.f ? 0.f : scalbnf(m_sv, -e);
      *reinterpret_cast<float4*>(sm + R::kScaleAt + slot * 16) = make_float4(m_sk, (float)e, g, 0.f);
    }
    *reinterpret_cast<int4*>(sm + R::kMetaAt + slot * 16) = *reinterpret_cast<const int4*>(&a);
    __syncwarp();
  }
  __device__ __forceinline__ SplitPlace place(int n) const {  // of the 16 tokens n of the stream
    const int4 x = *reinterpret_cast<const int4*>(sm + R::kMetaAt + (n & (kSplitMeta - 1)) * 16);
    return *reinterpret_cast<const SplitPlace*>(&x);
  }
  __device__ __forceinline__ char* slot(int n) const { return sm + (n % S) * 2 * R::kSide; }

  // The warp's n tiles, from tile v of item ih of sequence i on, on W (this).
  // `done` is called with each item's state: done(i, ih, starts, ends).
  template <typename W, typename F>
  __device__ __forceinline__ void run(W& w, const SplitParams& p, const int* prefix, int i, int ih, int v, int n,
                                      F done) {
    constexpr int kBatch = 32 / SUB;
    i0 = i;
    ih0 = ih;
    v0 = v;
    left = n;
    m_kvh = m_off = 0;
    place_begin(p, prefix);
    place_scales(p);
    place_store(p, 0);
    bool starts = v == 0;
#pragma unroll
    for (int x = 0; x < S; ++x) {
      if (x < n) w.copy_k(p, x);
      split_commit();
      if (x < n) w.copy_v(p, x);
      split_commit();
    }
    for (int x = S; x < min(n, kSplitAhead); ++x) w.ahead(p, x);
    w.load_q(p, i, ih);
    w.clear();
    for (int j = 0; j < n; ++j) {
      // the next places, in three steps so that no load is waited for (the
      // ring runs S <= 8 tiles ahead)
      const int phase = j & (kBatch - 1);
      if (__builtin_expect(j - phase + kBatch < n, 0)) {
        if (phase == 0) place_begin(p, prefix);
        if (phase == kBatch / 4) place_scales(p);
        if (phase == kBatch / 2) place_store(p, j + kBatch / 2);
      }
      const bool ends = w.step(p, j, n);
      if (__builtin_expect(ends || j == n - 1, 0)) {
        w.finish();
        done(i, ih, starts, ends);
        if (j < n - 1) {
          if (++ih == p.IH) {
            ih = 0;
            do ++i;
            while (prefix[i + 1] == prefix[i]);
          }
          starts = true;
          w.load_q(p, i, ih);
          w.clear();
        }
      }
    }
  }
};

template <int KIND, typename QT, int E>
struct SplitWarp : SplitWalk<KIND, QT, E> {
  using C = SplitCfg<KIND, E>;
  using Walk = SplitWalk<KIND, QT, E>;
  using R = typename Walk::R;
  using Walk::lane;
  using Walk::place;
  using Walk::slot;
  using Walk::sm;
  using Walk::st;
  static constexpr bool kPBf16 = KIND == kSplitBf16;                       // operand type of the MMAs
  static constexpr int NQ = KIND == kSplitE4m3 && sizeof(QT) == 4 ? 2 : 1;  // values q is split into
  static constexpr int NP = KIND == kSplitE4m3 && sizeof(QT) == 2 ? 1 : 2;  // values P is split into
  static constexpr int S = Walk::S, SUB = Walk::SUB;
  // bf16 outputs: the tensor core adds the tiles up (fp32 outputs add them with FMAs, which round)
  static constexpr bool kDirect = sizeof(QT) == 2;
  uint32_t q[KIND == kSplitF32 ? 1 : NQ][KIND == kSplitF32 ? 1 : C::NM][2];
  float qc[2];  // per column: what turns S into log2 units (but for the block's scale)
  float up[2];  // kUp - m per column; +inf before there is an m
  // 8-bit caches: O is in units of 2^unit, the largest V scale's exponent so far.
  // A weight times its scale is 2^(x + e - m + kUp) * g, e the scale's exponent
  // less unit: m follows x + e, so the weights that count most for the values
  // are near f16's largest whatever the scales. (lift: see follow().)
  float unit, lift;
  uint32_t kr[SUB][R::kRing ? 1 : (C::k8 ? 2 : 4) * C::NM];                    // the next tile's K
  uint32_t vr[SUB][R::kRing ? 1 : 4][R::kRing ? 1 : C::RUNS * (C::RUNB / 4)];  // and V

  __device__ __forceinline__ void clear() {
    st.clear();
    up[0] = up[1] = INFINITY;
    unit = -1000.f;
    lift = 0.f;
  }

  // The B fragments of Q^T: column g is query row r0 + g of the item.
  __device__ __forceinline__ void load_q(const SplitParams& p, int i, int ih) {
    const int g = lane >> 2, t = lane & 3;
    const int kvh = ih / p.NRG, r0 = (ih - kvh * p.NRG) * 8;
    const bool have = r0 + g < p.G;
    const QT* src = static_cast<const QT*>(p.q) + (long long)i * p.q_stride + ((long long)kvh * p.G + r0 + g) * E;
    if constexpr (KIND == kSplitBf16) {
#pragma unroll
      for (int kk = 0; kk < C::NM; ++kk)
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          const int d = 16 * kk + 8 * b + 2 * t;
          if (p.q_vec) {
            q[0][kk][b] = have ? __ldg(reinterpret_cast<const uint32_t*>(src + d)) : 0u;
          } else {
            const float lo = have ? to_f32(src[d]) : 0.f, hi = have ? to_f32(src[d + 1]) : 0.f;
            q[0][kk][b] = split_pack<true>(lo, hi);
          }
        }
      qc[0] = qc[1] = p.c;
    } else if constexpr (KIND == kSplitE4m3) {
      float x[4 * C::NM];
      // the lane's dims: KC runs of KB contiguous ones
#pragma unroll
      for (int c = 0; c < C::KC; ++c) {
        const QT* run = src + c * 4 * C::KB + t * C::KB;
        if (p.q_vec && have) {
#pragma unroll
          for (int w = 0; w < C::KB * (int)sizeof(QT) / 16; ++w) {
            const uint4 u = __ldg(reinterpret_cast<const uint4*>(run) + w);
            const uint32_t r[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int y = 0; y < 4; ++y) {
              if constexpr (sizeof(QT) == 2) {
                x[c * C::KB + 8 * w + 2 * y] = bf16_lo(r[y]);
                x[c * C::KB + 8 * w + 2 * y + 1] = bf16_hi(r[y]);
              } else {
                x[c * C::KB + 4 * w + y] = __uint_as_float(r[y]);
              }
            }
          }
        } else {
#pragma unroll
          for (int e = 0; e < C::KB; ++e) x[c * C::KB + e] = have ? to_f32(run[e]) : 0.f;
        }
      }
      float top = 0.f;
#pragma unroll
      for (int e = 0; e < 4 * C::NM; ++e) top = fmaxf(top, fabsf(x[e]));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      // the row's largest value to [2^13, 2^14): f16 then holds a bf16 row to
      // 2^-38 of it, and an fp32 row in two values to 2^-23 of each element.
      // (An infinity keeps its size: f16 has one.)
      int ex = 0;
      if (top > 0.f && top < INFINITY) ex = max(-120, min(120, 13 - ilogbf(top)));
      const float up = exp2f((float)ex);
#pragma unroll
      for (int kk = 0; kk < C::NM; ++kk)
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          const float lo = x[4 * kk + 2 * b] * up, hi = x[4 * kk + 2 * b + 1] * up;
          q[0][kk][b] = split_pack<false>(lo, hi);
          if constexpr (NQ == 2) {
            float l0, h0;
            split_unpack<false>(q[0][kk][b], &l0, &h0);
            q[1][kk][b] = split_pack<false>(lo - l0, hi - h0);
          }
        }
      // the columns of this lane's S values are rows 2t and 2t + 1
      const float down = exp2f((float)-ex) * p.c;
      qc[0] = __shfl_sync(0xffffffffu, down, 8 * t);
      qc[1] = __shfl_sync(0xffffffffu, down, 8 * t + 4);
    } else {
      // fp32 caches: the rows go to shared memory, [dim][8]
      float* sq = reinterpret_cast<float*>(sm + R::kQueryAt);
      __syncwarp();
      for (int x = lane; x < 8 * E; x += 32) {
        const int r = x / E, d = x - r * E;
        sq[d * 8 + r] = r0 + r < p.G
                            ? static_cast<const float*>(p.q)[(long long)i * p.q_stride +
                                                             ((long long)kvh * p.G + r0 + r) * E + d]
                            : 0.f;
      }
      __syncwarp();
      qc[0] = qc[1] = p.c;
    }
  }

  // ---- a tile's K and V: to registers, or (fp32) into the ring. Keys that do
  // not count are zeros there, never NaN times 0.
  __device__ __forceinline__ void copy_k(const SplitParams& p, int n) {
#pragma unroll
    for (int u = 0; u < SUB; ++u) {
      const SplitPlace a = place(n * SUB + u);
      if ((a.mask & 0xffffu) == 0xffffu)
        copy_k_of<true>(p, a, slot(n), kr[u]);
      else
        copy_k_of<false>(p, a, slot(n), kr[u]);
    }
  }
  __device__ __forceinline__ void copy_v(const SplitParams& p, int n) {
#pragma unroll
    for (int u = 0; u < SUB; ++u) {
      const SplitPlace a = place(n * SUB + u);
      if ((a.mask & 0xffffu) == 0xffffu)
        copy_v_of<true>(p, a, slot(n) + R::kSide, vr[u]);
      else
        copy_v_of<false>(p, a, slot(n) + R::kSide, vr[u]);
    }
  }
  template <bool FULL, int N>
  __device__ __forceinline__ void copy_k_of(const SplitParams& p, const SplitPlace& a, char* ring, uint32_t (&kr)[N]) {
    const int g = lane >> 2, t = lane & 3;
    const char* src = static_cast<const char*>(p.kc) + a.page;
    if constexpr (C::k8) {
      src += a.off * E + C::skey(0, g) * E + t * C::KB;
#pragma unroll
      for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int c = 0; c < C::KC; ++c)
          split_load<C::KB, FULL>(kr + (half * C::KC + c) * (C::KB / 4), src + half * 8 * E + c * 4 * C::KB,
                                  (a.mask >> C::skey(half, g)) & 1);
    } else {
      // a pair of keys of dim pair (bf16) or dim (fp32) d
      src += (a.off + 2 * g) * 4 + (long long)t * p.page * 4;
      const bool on = (a.mask >> (2 * g)) & 3;
      const long long step = 16LL * p.page;
      if constexpr (C::kBf16) {
#pragma unroll
        for (int x = 0; x < 2 * C::NM; ++x) {
          split_load<8, FULL>(kr + 2 * x, src + x * step, on);
          if constexpr (!FULL) {  // one of the pair may not count
            if (!((a.mask >> (2 * g)) & 1)) kr[2 * x] = 0u;
            if (!((a.mask >> (2 * g + 1)) & 1)) kr[2 * x + 1] = 0u;
          }
        }
      } else {
        const uint32_t dst = smem_u32(ring) + lane * 8;
#pragma unroll
        for (int x = 0; x < E / 4; ++x) split_copy<8, FULL>(dst + x * 256, src + x * step, on);
      }
    }
  }
  template <bool FULL, int N4, int N>
  __device__ __forceinline__ void copy_v_of(const SplitParams& p, const SplitPlace& a, char* ring,
                                            uint32_t (&vr)[N4][N]) {
    const int g = lane >> 2, t = lane & 3;
    const char* src = static_cast<const char*>(p.vc) + a.page + (long long)a.off * E * C::ES;
    if constexpr (C::kF32) {
      // every lane reads all of V there: the slot has been read by now
      __syncwarp();
      const uint32_t dst = smem_u32(ring);
#pragma unroll
      for (int x = 0; x < R::kSide / 512; ++x) {
        const int at = x * 512 + lane * 16;
        split_copy<16, FULL>(dst + at, src + at, (a.mask >> (at / (E * 4))) & 1);
      }
    } else {
      src += (C::vkey(0, t) * E + g * C::RL) * C::ES;
#pragma unroll
      for (int x = 0; x < 4; ++x)
#pragma unroll
        for (int r = 0; r < C::RUNS; ++r)
          split_load<C::RUNB, FULL>(vr[x] + r * (C::RUNB / 4), src + (C::vkey(x, 0) * E + r * 8 * C::RL) * C::ES,
                                    (a.mask >> C::vkey(x, t)) & 1);
    }
  }

  // S^T of the tile: s[0], s[1] = key row g of columns 2t, 2t+1; s[2], s[3] = row g + 8.
  template <int N>
  __device__ __forceinline__ void scores(float (&s)[4], const char* ks, uint32_t mask, const uint32_t (&kr)[N]) {
    if constexpr (KIND == kSplitF32) {
      // lane (g, t): keys 2g, 2g+1, every 4th dim, all 8 columns; then the t
      // lanes' sums are added so that each keeps its two columns
      const int g = lane >> 2, t = lane & 3;
      const float* sq = reinterpret_cast<const float*>(sm + R::kQueryAt);
      float acc[2][8];
#pragma unroll
      for (int c = 0; c < 8; ++c) acc[0][c] = acc[1][c] = 0.f;
      const bool on0 = (mask >> (2 * g)) & 1, on1 = (mask >> (2 * g + 1)) & 1;
#pragma unroll 8
      for (int x = 0; x < E / 4; ++x) {
        uint32_t r[2];
        split_lds<8>(r, ks + (x * 32 + lane) * 8);
        const float k0 = on0 ? __uint_as_float(r[0]) : 0.f, k1 = on1 ? __uint_as_float(r[1]) : 0.f;
        const float4 qa = *reinterpret_cast<const float4*>(sq + (4 * x + t) * 8);
        const float4 qb = *reinterpret_cast<const float4*>(sq + (4 * x + t) * 8 + 4);
        const float qq[8] = {qa.x, qa.y, qa.z, qa.w, qb.x, qb.y, qb.z, qb.w};
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          acc[0][c] = fmaf(k0, qq[c], acc[0][c]);
          acc[1][c] = fmaf(k1, qq[c], acc[1][c]);
        }
      }
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        // t's bit 1 chooses columns 0-3 or 4-7, bit 0 the pair among them
        float four[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const float mine = (t & 2) ? acc[half][4 + c] : acc[half][c];
          const float give = (t & 2) ? acc[half][c] : acc[half][4 + c];
          four[c] = mine + __shfl_xor_sync(0xffffffffu, give, 2);
        }
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const float mine = (t & 1) ? four[2 + c] : four[c];
          const float give = (t & 1) ? four[c] : four[2 + c];
          s[2 * half + c] = mine + __shfl_xor_sync(0xffffffffu, give, 1);
        }
      }
    } else {
#pragma unroll
      for (int r = 0; r < 4; ++r) s[r] = 0.f;
#pragma unroll
      for (int kk = 0; kk < C::NM; ++kk) {
        uint32_t f[4];
        if constexpr (C::k8) {
          const uint32_t w0 = kr[kk], w1 = kr[C::NM + kk];
          f[0] = f16x2_of_e4m3x2(w0);
          f[1] = f16x2_of_e4m3x2(w1);
          f[2] = f16x2_of_e4m3x2_hi(w0);
          f[3] = f16x2_of_e4m3x2_hi(w1);
        } else {
          f[0] = kr[4 * kk];
          f[1] = kr[4 * kk + 1];
          f[2] = kr[4 * kk + 2];
          f[3] = kr[4 * kk + 3];
        }
#pragma unroll
        for (int x = 0; x < NQ; ++x) split_mma<kPBf16>(s, f, q[x][kk][0], q[x][kk][1]);
      }
    }
  }

  // A larger V scale than any before: O in its units. Its tokens' weights would
  // be small against m, which was made with smaller scales: m goes down with
  // them (l and O up), by 2^90 in all at most, so that l stays finite.
  __device__ __forceinline__ void follow(float e) {
    const float d = unit - e;  // < 0
    const float rise = unit < -500.f ? 0.f : fminf(-d, 90.f - lift);
    const float fo = unit < -500.f ? 0.f : exp2f(fmaxf(d + rise, -140.f)), fl = exp2f(rise);
#pragma unroll
    for (int j = 0; j < C::NM; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) st.o[j][r] *= fo;
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      st.l[y] *= fl;
      st.m[y] -= rise;
      up[y] += rise;
    }
    lift += rise;
    unit = e;
  }

  // The tile's weights 2^(x + e - m + kUp) (s), m the column's reference, and
  // what they are multiplied by for the values (g).
  __device__ __forceinline__ void softmax(float (&s)[SUB][4], const uint32_t (&mask)[SUB], const float4 (&sc)[SUB],
                                          float (&gv)[SUB]) {
    const int g = lane >> 2;
    float x[SUB][4], e[SUB], back[SUB];  // back: 2^-e, from these weights to those of l
    bool fits = true;
#pragma unroll
    for (int u = 0; u < SUB; ++u) {
      e[u] = 0.f;
      back[u] = gv[u] = 1.f;
      if constexpr (C::k8)
        if (__builtin_expect(sc[u].y > unit, 0)) follow(sc[u].y);  // (uniform)
    }
#pragma unroll
    for (int u = 0; u < SUB; ++u) {
      if constexpr (C::k8) {
        const float d = sc[u].y - unit;
        e[u] = fmaxf(d, -90.f);
        back[u] = exp2_approx(-e[u]);
        gv[u] = d >= -90.f ? sc[u].z : sc[u].z * exp2_approx(fmaxf(d, -200.f) + 90.f);
      }
#pragma unroll
      for (int r = 0; r < 4; ++r)
        x[u][r] = fmaf(s[u][r], C::k8 ? qc[r & 1] * sc[u].x : qc[r & 1], C::k8 ? up[r & 1] + e[u] : up[r & 1]);
      if ((mask[u] & 0xffffu) != 0xffffu) {
        const bool on0 = (mask[u] >> C::skey(0, g)) & 1, on1 = (mask[u] >> C::skey(1, g)) & 1;
        x[u][0] = on0 ? x[u][0] : -INFINITY;
        x[u][1] = on0 ? x[u][1] : -INFINITY;
        x[u][2] = on1 ? x[u][2] : -INFINITY;
        x[u][3] = on1 ? x[u][3] : -INFINITY;
      }
      fits = fits && fmaxf(x[u][0], x[u][2]) <= kUp + kSlack && fmaxf(x[u][1], x[u][3]) <= kUp + kSlack;
    }
    // a weight past 2^(kUp + kSlack) (or one that is no number, as all are
    // before a column has a reference) moves the references
    if (__builtin_expect(__any_sync(0xffffffffu, !fits), 0)) {
      float mt[2] = {-INFINITY, -INFINITY}, alpha[2];
#pragma unroll
      for (int u = 0; u < SUB; ++u) {
        const bool on0 = (mask[u] >> C::skey(0, g)) & 1, on1 = (mask[u] >> C::skey(1, g)) & 1;
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const float c = C::k8 ? qc[y] * sc[u].x : qc[y];
          x[u][y] = on0 ? fmaf(s[u][y], c, e[u]) : -INFINITY;
          x[u][2 + y] = on1 ? fmaf(s[u][2 + y], c, e[u]) : -INFINITY;
          mt[y] = fmaxf(mt[y], fmaxf(x[u][y], x[u][2 + y]));
        }
      }
#pragma unroll
      for (int y = 0; y < 2; ++y) {
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) mt[y] = fmaxf(mt[y], __shfl_xor_sync(0xffffffffu, mt[y], o));
        const float mn = fmaxf(st.m[y], mt[y]);
        const float mu = mn == -INFINITY ? 0.f : mn;
        alpha[y] = exp2_approx(st.m[y] - mu);
        st.l[y] *= alpha[y];
        st.m[y] = mn;
        up[y] = kUp - mn;  // (still no reference: +inf)
#pragma unroll
        for (int u = 0; u < SUB; ++u) {
          x[u][y] = x[u][y] - mu + kUp;
          x[u][2 + y] = x[u][2 + y] - mu + kUp;
        }
      }
#pragma unroll
      for (int j = 0; j < C::NM; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) st.o[j][r] *= alpha[r & 1];
    }
#pragma unroll
    for (int u = 0; u < SUB; ++u) {
#pragma unroll
      for (int r = 0; r < 4; ++r) s[u][r] = exp2_approx(x[u][r]);
      st.l[0] = fmaf(s[u][0] + s[u][2], back[u], st.l[0]);
      st.l[1] = fmaf(s[u][1] + s[u][3], back[u], st.l[1]);
    }
  }

  // O += P V, P = s * f
  template <int N4, int N>
  __device__ __forceinline__ void values(float (&s)[4], float f, const char* vs, const uint32_t (&vr)[N4][N]) {
    if constexpr (KIND == kSplitF32) {
      const int g = lane >> 2, t = lane & 3;
#pragma unroll 4
      for (int key = 0; key < 16; ++key) {
        const int from = (key >> 1) * 4 + t;
        const float w0 = __shfl_sync(0xffffffffu, (key & 1) ? s[2] : s[0], from);
        const float w1 = __shfl_sync(0xffffffffu, (key & 1) ? s[3] : s[1], from);
#pragma unroll
        for (int r = 0; r < C::RUNS; ++r) {
          uint32_t w[4];
          split_lds<16>(w, vs + (key * E + r * 32 + g * 4) * 4);
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            float* o = st.o[2 * r + (y >> 1)];
            o[2 * (y & 1)] = fmaf(w0, __uint_as_float(w[y]), o[2 * (y & 1)]);
            o[2 * (y & 1) + 1] = fmaf(w1, __uint_as_float(w[y]), o[2 * (y & 1) + 1]);
          }
        }
      }
    } else {
      if constexpr (C::k8) {
#pragma unroll
        for (int r = 0; r < 4; ++r) s[r] *= f;
      }
      uint32_t b[NP][2];
      b[0][0] = split_pack<kPBf16>(s[0], s[1]);
      b[0][1] = split_pack<kPBf16>(s[2], s[3]);
      if constexpr (NP == 2) {
        float r[4];
        split_unpack<kPBf16>(b[0][0], &r[0], &r[1]);
        split_unpack<kPBf16>(b[0][1], &r[2], &r[3]);
        b[1][0] = split_pack<kPBf16>(s[0] - r[0], s[1] - r[1]);
        b[1][1] = split_pack<kPBf16>(s[2] - r[2], s[3] - r[3]);
      }
#pragma unroll
      for (int x = 0; x < NP; ++x) {
        b[x][0] = split_transpose(b[x][0]);
        b[x][1] = split_transpose(b[x][1]);
      }
#pragma unroll
      for (int j = 0; j < C::NM; ++j) {
        uint32_t m[4];
        if constexpr (C::k8) {
          const int w = j >> 1;
          const uint32_t sel = (j & 1) ? 0x7362u : 0x5140u;
          const uint32_t ab = __byte_perm(vr[0][w], vr[1][w], sel), cd = __byte_perm(vr[2][w], vr[3][w], sel);
          m[0] = f16x2_of_e4m3x2(ab);
          m[1] = f16x2_of_e4m3x2_hi(ab);
          m[2] = f16x2_of_e4m3x2(cd);
          m[3] = f16x2_of_e4m3x2_hi(cd);
        } else {
          m[0] = __byte_perm(vr[0][j], vr[1][j], 0x5410u);
          m[1] = __byte_perm(vr[0][j], vr[1][j], 0x7632u);
          m[2] = __byte_perm(vr[2][j], vr[3][j], 0x5410u);
          m[3] = __byte_perm(vr[2][j], vr[3][j], 0x7632u);
        }
        if constexpr (kDirect) {
#pragma unroll
          for (int x = 0; x < NP; ++x) split_mma<kPBf16>(st.o[j], m, b[x][0], b[x][1]);
        } else {
          float d[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int x = 0; x < NP; ++x) split_mma<kPBf16>(d, m, b[x][0], b[x][1]);
#pragma unroll
          for (int r = 0; r < 4; ++r) st.o[j][r] += d[r];
        }
      }
    }
  }

  // Tile j's lines to L2, ahead of the loads (8-bit caches: 16 rows of K and of V
  // are one run of bytes each).
  __device__ __forceinline__ void ahead(const SplitParams& p, int j) const {
    if constexpr (C::k8 && kSplitAhead > S) {
      if (lane < 2 * SUB) {
        const SplitPlace a = place(j * SUB + (lane >> 1));
        if (a.mask & 0xffffu)
          bulk_prefetch_l2(static_cast<const char*>(lane & 1 ? p.vc : p.kc) + a.page + (long long)a.off * E, 16 * E);
      }
    }
  }

  // Tile j: true when its item ends.
  __device__ __forceinline__ bool step(const SplitParams& p, int j, int n) {
    if (j + kSplitAhead < n) ahead(p, j + kSplitAhead);
    uint32_t mask[SUB];
    float4 sc[SUB];
    float gv[SUB];
#pragma unroll
    for (int u = 0; u < SUB; ++u) {
      mask[u] = place(j * SUB + u).mask;
      if constexpr (C::k8)
        sc[u] = *reinterpret_cast<const float4*>(sm + R::kScaleAt + ((j * SUB + u) & (kSplitMeta - 1)) * 16);
    }
    char* at = slot(j);
    float s[SUB][4];
    if constexpr (R::kRing) split_wait<2 * S - 1>();
#pragma unroll
    for (int u = 0; u < SUB; ++u) scores(s[u], at, mask[u], kr[u]);
    if (j + S < n) copy_k(p, j + S);
    if constexpr (R::kRing) split_commit();
    softmax(s, mask, sc, gv);
    if constexpr (R::kRing) split_wait<2 * S - 1>();
    if constexpr (C::kF32) __syncwarp();
#pragma unroll
    for (int u = 0; u < SUB; ++u) values(s[u], gv[u], at + R::kSide, vr[u]);
    if (j + S < n) copy_v(p, j + S);
    if constexpr (R::kRing) split_commit();
    return (mask[0] >> 16) & 1;
  }
  __device__ __forceinline__ void finish() {
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) st.l[x] += __shfl_xor_sync(0xffffffffu, st.l[x], o);
    if constexpr (C::k8) {
      const float scale = exp2f(unit);
#pragma unroll
      for (int x = 0; x < C::NM; ++x)
#pragma unroll
        for (int r = 0; r < 4; ++r) st.o[x][r] *= scale;
    }
  }
};

// A piece of an item that a warp could not finish alone.
struct SplitPiece {
  int i, ih;
  int last;  // the item's last tile lies in this piece
  int have;
};

template <int KIND, int E>
__host__ __device__ constexpr int split_smem_fixed() {
  return kSplitWarps * (SplitRing<KIND, E>::kWarpBytes + 2 * SplitCfg<KIND, E>::kPieceFloats * 4) + kSplitWarps * 2 * (int)sizeof(SplitPiece) + 128;
}

// Work is shared out in units: an item is kSplitItemUnits (2 and 3: the same; 1:
// +7% on 32 x 16 heads) and one for each of its tiles. Where unit u of the launch lies: the tile at or after it.
constexpr int kSplitItemUnits = 2;

struct SplitSpot {
  int i, ih, v;
  long long tile;  // its number among the launch's tiles
};
__device__ __forceinline__ long long split_units(const int* prefix, int i, int IH) {
  return ((long long)prefix[i] + (long long)kSplitItemUnits * i) * IH;
}
__device__ __forceinline__ SplitSpot split_spot(const int* prefix, int B, int IH, long long u) {
  int lo = 0, hi = B;  // the last i that starts at or before u
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (split_units(prefix, mid, IH) <= u)
      lo = mid;
    else
      hi = mid;
  }
  SplitSpot s;
  s.i = lo;
  const int nt = prefix[lo + 1] - prefix[lo];
  const long long r = u - split_units(prefix, lo, IH);
  const long long ih = min((long long)IH, r / (nt + kSplitItemUnits));
  s.ih = (int)ih;
  s.v = (int)max(0LL, r - ih * (nt + kSplitItemUnits) - kSplitItemUnits);
  if (s.ih == IH) s.v = 0;  // (u is the end)
  s.tile = (long long)prefix[lo] * IH + ih * nt + min(s.v, nt);
  return s;
}

template <int KIND, typename QT, int E>
__global__ void __launch_bounds__(32 * kSplitWarps, kSplitCtasPerSm)
    split_decode_kernel(const __grid_constant__ SplitParams p) {
  using C = SplitCfg<KIND, E>;
  constexpr int kWarpBytes = SplitRing<KIND, E>::kWarpBytes;
  extern __shared__ __align__(16) char split_smem[];
  float* pieces = reinterpret_cast<float*>(split_smem + kSplitWarps * kWarpBytes);  // [warp][head, tail]
  SplitPiece* info = reinterpret_cast<SplitPiece*>(pieces + kSplitWarps * 2 * C::kPieceFloats);
  int* wsum = reinterpret_cast<int*>(info + kSplitWarps * 2);
  int* prefix = wsum + 32;  // [B + 1]: tiles of one item before sequence i
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int kThreads = 32 * kSplitWarps;

  // ---- tiles before each sequence
  {
    const int per = (p.B + kThreads - 1) / kThreads;
    const int i0 = min(p.B, (int)threadIdx.x * per), i1 = min(p.B, i0 + per);
    int sum = 0;
    for (int i = i0; i < i1; ++i) {
      prefix[i] = sum;  // (before the threads ahead are known)
      sum += (split_seq(p, i).nt + split_sub<KIND, E>() - 1) / split_sub<KIND, E>();
    }
    const int incl = warp_scan_i(sum, lane);
    if (lane == 31) wsum[warp] = incl;
    __syncthreads();
    int base = incl - sum;
    for (int w = 0; w < warp; ++w) base += wsum[w];
    for (int i = i0; i < i1; ++i) prefix[i] += base;
    if (threadIdx.x == kThreads - 1) prefix[p.B] = base + sum;
    if (threadIdx.x < 2 * kSplitWarps) info[threadIdx.x].have = 0;
    __syncthreads();
  }
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const long long total = split_units(prefix, p.B, p.IH);
  const long long warps = (long long)gridDim.x * kSplitWarps;
  const long long chunk = max(1LL, (total + warps - 1) / warps);
  const long long w0 = min(total, ((long long)blockIdx.x * kSplitWarps + warp) * chunk);
  const long long w1 = min(total, w0 + chunk);

  // ---- this warp's tiles
  // (lane 1 looks up the end while the others look up the start)
  SplitSpot a = split_spot(prefix, p.B, p.IH, lane == 1 ? w1 : w0);
  const int n = w0 < w1 ? (int)(__shfl_sync(0xffffffffu, a.tile, 1) - __shfl_sync(0xffffffffu, a.tile, 0)) : 0;
  a.i = __shfl_sync(0xffffffffu, a.i, 0);
  a.ih = __shfl_sync(0xffffffffu, a.ih, 0);
  a.v = __shfl_sync(0xffffffffu, a.v, 0);
  if (n > 0)
    while (prefix[a.i + 1] == prefix[a.i]) {  // sequences that see nothing have no tiles
      ++a.i;
      a.ih = a.v = 0;
    }
  // What an append just before this launch writes is read from here on. (Every
  // warp waits: what follows in the stream waits for this launch only.)
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (n > 0) {
      SplitWarp<KIND, QT, E> w;
      w.sm = split_smem + warp * kWarpBytes;
      w.lane = lane;
      w.run(w, p, prefix, a.i, a.ih, a.v, n, [&](int i, int ih, bool starts, bool ends) {
        if (starts && ends) {
          split_write<KIND, QT, E>(p, w.st, i, ih, lane);
        } else {
          w.st.put(pieces + (warp * 2 + (starts ? 1 : 0)) * C::kPieceFloats, lane);
          if (lane == 0) info[warp * 2 + (starts ? 1 : 0)] = SplitPiece{i, ih, ends ? 1 : 0, 1};
        }
      });
  }
  // ---- sequences that see nothing: zeros
  for (int i = blockIdx.x; i < p.B; i += gridDim.x)
    if (prefix[i + 1] == prefix[i]) {
      for (int x = threadIdx.x; x < p.H * E; x += kThreads)
        static_cast<QT*>(p.out)[(long long)i * p.H * E + x] = from_f32<QT>(0.f);
      if (p.lse)
        for (int x = threadIdx.x; x < p.H; x += kThreads) p.lse[(long long)i * p.H + x] = -INFINITY;
    }
  if (threadIdx.x == 0) p.meta[4 * blockIdx.x + 3] = 0;
  __syncthreads();

  // ---- join the pieces of one item inside this CTA, in order. A group starts
  // with a warp's tail piece (the item's first tile), or with the head piece of
  // the first warp that has tiles (the item began in an earlier CTA), and goes
  // on through the next warps' head pieces until the item's last tile or the
  // CTA's end. (A range that starts inside an item has tiles of it.)
  for (int kind = 0; kind < 2; ++kind) {  // 0: warp 0's head, 1: this warp's tail
    if (kind == 0 && warp != 0) continue;
    const int first = warp * 2 + kind;
    const SplitPiece me = info[first];
    if (!me.have) continue;
    SplitState<C::NM> st;
    st.clear();
    st.join(pieces + first * C::kPieceFloats, lane);
    bool done = me.last != 0;
    for (int k = warp + 1; !done && k < kSplitWarps && info[2 * k].have; ++k) {
      st.join(pieces + 2 * k * C::kPieceFloats, lane);
      done = info[2 * k].last != 0;
    }
    if (kind == 1 && done) {
      split_write<KIND, QT, E>(p, st, me.i, me.ih, lane);
    } else {
      st.put(p.partial + (2LL * blockIdx.x + kind) * C::kPieceFloats, lane);
      if (kind == 1 && lane == 0) {
        // the CTA that holds the item's last unit (its last tile)
        const long long end = split_units(prefix, me.i, p.IH) +
                              (long long)(me.ih + 1) * (prefix[me.i + 1] - prefix[me.i] + kSplitItemUnits) - 1;
        int* m = p.meta + 4 * blockIdx.x;
        m[0] = me.i;
        m[1] = me.ih;
        m[2] = (int)(end / (chunk * kSplitWarps));
        m[3] = 1;
      }
    }
  }
}

// Joins the items that cross CTA boundaries: block c takes the one that CTA c
// began and did not end, if there is one. Warp (r, j) joins a contiguous share r
// of the item's pieces for the four registers j of O (loads of several pieces in
// flight); then the shares are joined in order.
template <int KIND, typename QT, int E>
__global__ void __launch_bounds__(32 * kSplitMergeShares * (E / 16))
    split_merge_kernel(const __grid_constant__ SplitParams p) {
  using C = SplitCfg<KIND, E>;
  __shared__ float shares[kSplitMergeShares * C::kPieceFloats];
  const int lane = threadIdx.x & 31;
  const int j = (threadIdx.x >> 5) % C::NM, share = (threadIdx.x >> 5) / C::NM;
  const int count = (int)blockDim.x / (32 * C::NM);  // shares
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int c = blockIdx.x;
  const int* m = p.meta + 4 * c;
  if (m[3] != 1) return;
  const int n = m[2] - c + 1;
  const int per = (n + count - 1) / count;
  const int k0 = share * per, k1 = min(n, k0 + per);
  // one group of four registers, and (m, l) with it
  SplitState<1> st;
  st.clear();
#pragma unroll 4
  for (int k = k0; k < k1; ++k) {
    const float* piece = p.partial + (2LL * (c + k) + (k == 0 ? 1 : 0)) * C::kPieceFloats + lane;
    float o[4], mo[2], lo[2];
#pragma unroll
    for (int r = 0; r < 4; ++r) o[r] = piece[(4 * j + r) * 32];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      mo[x] = piece[(4 * C::NM + x) * 32];
      lo[x] = piece[(4 * C::NM + 2 + x) * 32];
    }
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const float mn = fmaxf(st.m[x], mo[x]);
      const float mu = mn == -INFINITY ? 0.f : mn;
      const float a = exp2_approx(st.m[x] - mu), b = exp2_approx(mo[x] - mu);
      st.l[x] = st.l[x] * a + lo[x] * b;
      st.m[x] = mn;
      st.o[0][x] = st.o[0][x] * a + o[x] * b;
      st.o[0][2 + x] = st.o[0][2 + x] * a + o[2 + x] * b;
    }
  }
  float* mine = shares + share * C::kPieceFloats + lane;
#pragma unroll
  for (int r = 0; r < 4; ++r) mine[(4 * j + r) * 32] = st.o[0][r];
  if (j == 0) {
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      mine[(4 * C::NM + x) * 32] = st.m[x];
      mine[(4 * C::NM + 2 + x) * 32] = st.l[x];
    }
  }
  __syncthreads();
  if (threadIdx.x < 32) {
    SplitState<C::NM> all;
    all.clear();
#pragma unroll 1
    for (int r = 0; r < count; ++r) all.join(shares + r * C::kPieceFloats, lane);
    split_write<KIND, QT, E>(p, all, m[0], m[1], lane);
  }
}

}  // namespace ca
