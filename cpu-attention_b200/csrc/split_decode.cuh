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
// What bounds it: HBM. A 16-token tile of one KV head is 4 KiB of codes at
// head_dim 128 (8 KiB bf16, 16 KiB fp32), read once for up to 8 query rows.
//
// Work: the visible tokens of every item (sequence, KV head, up to 8 of its
// query heads) are cut into tiles of 16 tokens; pages between the first tokens
// and the window are neither read nor looked up, so their page-table entries
// may be anything. All tiles are numbered in (sequence, head, token) order and
// every warp of the grid takes an equal, contiguous run of them, so lengths
// need not be known on the host and ragged batches stay balanced. An item cut
// by a warp boundary leaves its (m, l, O) in shared memory, where its CTA joins
// the pieces in tile order; one cut by a CTA boundary goes through a small
// global buffer and split_merge_kernel, also in order. The result does not
// depend on timing, and nothing is kept between calls.
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
//   that f16 holds it. P is taken against the tile's own maximum, so a tile's
//   largest weight is 1 whatever came before, and enters as one f16 value for
//   bf16 outputs (2^-12 of the weight, against 2^-9 of the output's rounding)
//   and as a value plus its rest for fp32 ones and for bf16 caches.
//   The tile's product is scaled by s_v * 2^(m_tile - m) when it is added, so
//   any scale a user stores is followed.
// fp32 caches run the same tiles on FMAs.
//
// Loads of tile n+1 are issued as soon as the registers of tile n are free: 12
// warps an SM with a tile each in flight are 48 KiB, about twice what HBM's
// latency asks for. mma.sync and not tcgen05: a tcgen05 tile has at least 64
// rows, of which at most 8 (16) query rows would be used.
#pragma once

#include <cuda_fp16.h>

#include "common.cuh"

namespace ca {

enum SplitKind { kSplitF32 = 0, kSplitBf16 = 1, kSplitE4m3 = 2 };

constexpr int kSplitWarps = 6;        // warps per CTA
constexpr int kSplitCtasPerSm = 2;    // CTAs per SM
constexpr int kSplitTile = 16;        // tokens per tile
constexpr int kSplitMaxBatch = 8192;  // sequences per launch (their tile counts sit in shared memory)
constexpr int kSplitMergeWarps = 4;

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
  int min_chunk;    // tiles a warp takes at least
  float* partial;   // [2 * CTAs] pieces of items cut by a CTA boundary
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
  long long L = (long long)__ldg(p.lens + i) + p.extra;
  const long long cap = p.pt_stride * (long long)p.page;
  if (L > cap) {
    if (p.status) atomicOr(p.status, CA_STATUS_LENS);
    L = cap;
  }
  // a negative length is a sequence that is skipped
  if (__ldg(p.lens + i) < 0) L = 0;
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

// Cache lines are read once per item: past L1.
template <int BYTES>
__device__ __forceinline__ void split_load(uint32_t* r, const void* p) {
  if constexpr (BYTES == 16)
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "l"(p));
  else if constexpr (BYTES == 8)
    asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0,%1}, [%2];" : "=r"(r[0]), "=r"(r[1]) : "l"(p));
  else
    asm volatile("ld.global.nc.L1::no_allocate.u32 %0, [%1];" : "=r"(r[0]) : "l"(p));
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

// (m, l, O) of up to 8 query rows over some tiles; columns 2t and 2t + 1 in lane (g, t).
template <int NM>
struct SplitState {
  float o[NM][4];
  float m[2], l[2];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int j = 0; j < NM; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
    m[0] = m[1] = -INFINITY;
    l[0] = l[1] = 0.f;
  }
  __device__ __forceinline__ void put(float* piece, int lane) const {
#pragma unroll
    for (int j = 0; j < NM; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) piece[(4 * j + r) * 32 + lane] = o[j][r];
    piece[(4 * NM + 0) * 32 + lane] = m[0];
    piece[(4 * NM + 1) * 32 + lane] = m[1];
    piece[(4 * NM + 2) * 32 + lane] = l[0];
    piece[(4 * NM + 3) * 32 + lane] = l[1];
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
    if (p.lse && g == 0) p.lse[h] = l == 0.f ? -INFINITY : (st.m[x] + log2f(l)) * 0.69314718055994531f;
  }
}

// ---- a warp's tiles ---------------------------------------------------------
// One tile's place: its block, rows inside the page, and which keys count.
struct SplitTile {
  const char* k;
  const char* v;
  uint32_t mask;  // bit j: key j of the tile is seen (0: the tile is skipped)
  float sk, sv;
};

template <int KIND, typename QT, int E>
struct SplitWarp {
  using C = SplitCfg<KIND, E>;
  static constexpr bool kPBf16 = KIND == kSplitBf16;                       // operand type of the MMAs
  static constexpr int NQ = KIND == kSplitE4m3 && sizeof(QT) == 4 ? 2 : 1;  // values q is split into
  static constexpr int NP = KIND == kSplitE4m3 && sizeof(QT) == 2 ? 1 : 2;  // values P is split into
  SplitState<C::NM> st;
  uint32_t q[NQ][C::NM][2];
  float qc[2];  // per column: what turns S into log2 units (but for the block's scale)
  uint32_t kr[KIND == kSplitF32 ? 1 : (C::k8 ? 2 * C::KC * (C::KB / 4) : 4 * C::NM)];
  uint32_t vr[KIND == kSplitF32 ? 1 : 4][KIND == kSplitF32 ? 1 : C::RUNS * (C::RUNB / 4)];

  // The B fragments of Q^T: column g is query row r0 + g of the item.
  __device__ __forceinline__ void load_q(const SplitParams& p, int i, int kvh, int r0, int lane, float* sq) {
    const int g = lane >> 2, t = lane & 3;
    const bool have = r0 + g < p.G;
    const QT* src = static_cast<const QT*>(p.q) + (long long)i * p.q_stride + ((long long)kvh * p.G + r0 + g) * E;
    if constexpr (KIND == kSplitBf16) {
#pragma unroll
      for (int kk = 0; kk < C::NM; ++kk)
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          const int d = 16 * kk + 8 * b + 2 * t;
          const float lo = have ? to_f32(src[d]) : 0.f, hi = have ? to_f32(src[d + 1]) : 0.f;
          q[0][kk][b] = split_pack<true>(lo, hi);
        }
      qc[0] = qc[1] = p.c;
    } else if constexpr (KIND == kSplitE4m3) {
      float x[4 * C::NM];
      float top = 0.f;
#pragma unroll
      for (int kk = 0; kk < C::NM; ++kk)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int d = (kk / (C::KB / 4)) * 4 * C::KB + t * C::KB + 4 * (kk % (C::KB / 4)) + e;
          x[4 * kk + e] = have ? to_f32(src[d]) : 0.f;
          top = fmaxf(top, fabsf(x[4 * kk + e]));
        }
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

  // Keys that do not count are not read: zero there (never NaN times 0).
  __device__ __forceinline__ void load_k(const SplitTile& a, int page, int lane) {
    const int g = lane >> 2, t = lane & 3;
    if constexpr (C::k8) {
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int key = C::skey(half, g);
        const bool on = (a.mask >> key) & 1;
#pragma unroll
        for (int c = 0; c < C::KC; ++c) {
          uint32_t* r = kr + (half * C::KC + c) * (C::KB / 4);
#pragma unroll
          for (int w = 0; w < C::KB / 4; ++w) r[w] = 0u;
          if (on) split_load<C::KB>(r, a.k + key * E + c * 4 * C::KB + t * C::KB);
        }
      }
    } else if constexpr (KIND == kSplitBf16) {
      const bool on0 = (a.mask >> (2 * g)) & 1, on1 = (a.mask >> (2 * g + 1)) & 1;
#pragma unroll
      for (int kk = 0; kk < C::NM; ++kk)
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          uint32_t* r = kr + (2 * kk + b) * 2;
          r[0] = r[1] = 0u;
          if (on0 || on1) split_load<8>(r, a.k + ((long long)(8 * kk + 4 * b + t) * page + 2 * g) * 4);
          if (!on0) r[0] = 0u;
          if (!on1) r[1] = 0u;
        }
    }
  }
  __device__ __forceinline__ void load_v(const SplitTile& a, int lane) {
    if constexpr (KIND != kSplitF32) {
      const int g = lane >> 2, t = lane & 3;
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int key = C::vkey(x, t);
        const bool on = (a.mask >> key) & 1;
#pragma unroll
        for (int r = 0; r < C::RUNS; ++r) {
          uint32_t* w = vr[x] + r * (C::RUNB / 4);
#pragma unroll
          for (int y = 0; y < C::RUNB / 4; ++y) w[y] = 0u;
          if (on) split_load<C::RUNB>(w, a.v + ((long long)key * E + r * 8 * C::RL + g * C::RL) * C::ES);
        }
      }
    }
  }

  // S^T of the tile: s[0], s[1] = key row g of columns 2t, 2t+1; s[2], s[3] = row g + 8.
  __device__ __forceinline__ void scores(float (&s)[4], const SplitTile& a, int page, int lane, const float* sq) {
    if constexpr (KIND == kSplitF32) {
      // lane (g, t): keys 2g, 2g+1, every 4th dim, all 8 columns; then the t
      // lanes' sums are added so that each keeps its two columns
      const int g = lane >> 2, t = lane & 3;
      float acc[2][8];
#pragma unroll
      for (int c = 0; c < 8; ++c) acc[0][c] = acc[1][c] = 0.f;
      const bool on0 = (a.mask >> (2 * g)) & 1, on1 = (a.mask >> (2 * g + 1)) & 1;
#pragma unroll 8
      for (int d = t; d < E; d += 4) {
        uint32_t r[2] = {0u, 0u};
        if (on0 || on1) split_load<8>(r, a.k + ((long long)d * page + 2 * g) * 4);
        const float k0 = on0 ? __uint_as_float(r[0]) : 0.f, k1 = on1 ? __uint_as_float(r[1]) : 0.f;
        const float4 qa = *reinterpret_cast<const float4*>(sq + d * 8);
        const float4 qb = *reinterpret_cast<const float4*>(sq + d * 8 + 4);
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
      float s2[2][4];  // two chains
#pragma unroll
      for (int r = 0; r < 4; ++r) s2[0][r] = s2[1][r] = 0.f;
#pragma unroll
      for (int kk = 0; kk < C::NM; ++kk) {
        uint32_t f[4];
        if constexpr (C::k8) {
          const uint32_t w0 = kr[kk], w1 = kr[C::KC * (C::KB / 4) + kk];
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
        for (int x = 0; x < NQ; ++x) split_mma<kPBf16>(s2[kk & 1], f, q[x][kk][0], q[x][kk][1]);
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) s[r] = s2[0][r] + s2[1][r];
    }
  }

  // Adds the tile: s as scores() left it.
  __device__ __forceinline__ void softmax(float (&s)[4], const SplitTile& a, int lane, float (&f)[2]) {
    const int g = lane >> 2;
    const bool on0 = (a.mask >> C::skey(0, g)) & 1, on1 = (a.mask >> C::skey(1, g)) & 1;
    float mt[2], alpha[2];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const float c = C::k8 ? qc[x] * a.sk : qc[x];
      s[x] = on0 ? s[x] * c : -INFINITY;
      s[2 + x] = on1 ? s[2 + x] * c : -INFINITY;
      mt[x] = fmaxf(s[x], s[2 + x]);
    }
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) {
      mt[0] = fmaxf(mt[0], __shfl_xor_sync(0xffffffffu, mt[0], o));
      mt[1] = fmaxf(mt[1], __shfl_xor_sync(0xffffffffu, mt[1], o));
    }
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const float mn = fmaxf(st.m[x], mt[x]);
      const float mu = mn == -INFINITY ? 0.f : mn, tu = mt[x] == -INFINITY ? 0.f : mt[x];
      alpha[x] = exp2_approx(st.m[x] - mu);
      const float beta = exp2_approx(mt[x] - mu);  // the tile's weights are taken against its own maximum
      s[x] = exp2_approx(s[x] - tu);
      s[2 + x] = exp2_approx(s[2 + x] - tu);
      st.l[x] = st.l[x] * alpha[x] + (s[x] + s[2 + x]) * beta;
      f[x] = C::k8 ? beta * a.sv : beta;
      if (mt[x] == -INFINITY) f[x] = 0.f;
      st.m[x] = mn;
    }
    if (__any_sync(0xffffffffu, alpha[0] != 1.f || alpha[1] != 1.f)) {
#pragma unroll
      for (int j = 0; j < C::NM; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) st.o[j][r] *= alpha[r & 1];
    }
  }

  // O += f * (P V), P = s
  __device__ __forceinline__ void values(const float (&s)[4], const float (&f)[2], const SplitTile& a, int lane) {
    if constexpr (KIND == kSplitF32) {
      const int g = lane >> 2, t = lane & 3;
      const float p0[2] = {s[0] * f[0], s[1] * f[1]}, p1[2] = {s[2] * f[0], s[3] * f[1]};
#pragma unroll 4
      for (int key = 0; key < 16; ++key) {
        const int from = (key >> 1) * 4 + t;
        const float w0 = __shfl_sync(0xffffffffu, (key & 1) ? p1[0] : p0[0], from);
        const float w1 = __shfl_sync(0xffffffffu, (key & 1) ? p1[1] : p0[1], from);
        if (!((a.mask >> key) & 1)) continue;  // (uniform)
#pragma unroll
        for (int r = 0; r < C::RUNS; ++r) {
          uint32_t w[4];
          split_load<16>(w, a.v + ((long long)key * E + r * 32 + g * 4) * 4);
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            float* o = st.o[2 * r + (y >> 1)];
            o[2 * (y & 1)] = fmaf(w0, __uint_as_float(w[y]), o[2 * (y & 1)]);
            o[2 * (y & 1) + 1] = fmaf(w1, __uint_as_float(w[y]), o[2 * (y & 1) + 1]);
          }
        }
      }
    } else {
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
        float d[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int x = 0; x < NP; ++x) split_mma<kPBf16>(d, m, b[x][0], b[x][1]);
#pragma unroll
        for (int r = 0; r < 4; ++r) st.o[j][r] = fmaf(f[r & 1], d[r], st.o[j][r]);
      }
    }
  }

  // Tiles [v, v + n) of item (i, kvh, r0).
  __device__ __forceinline__ void run(const SplitParams& p, const SplitSeq& sq, int i, int kvh, int r0, int v, int n,
                                      int lane, float* smq) {
    st.clear();
    const int tpp = p.page / kSplitTile;
    const long long rowbytes = (long long)p.page * E * C::ES;
    // the block ids (and scales) of 32 tiles at a time, one per lane
    int id = -1, off = 0, pos = 0;
    float sk = 0.f, sv = 0.f;
    auto meta = [&](int b0) {
      const int j = b0 + lane;
      id = -1;
      if (j < n) {
        const int vt = v + j;
        const int r = vt < sq.ts ? vt : vt + sq.skip;
        const int pg = r / tpp;
        off = (r - pg * tpp) * kSplitTile;
        pos = r * kSplitTile;
        id = __ldg(p.page_table + (long long)i * p.pt_stride + pg);
        if (id < 0 || id >= p.num_blocks) {
          if (p.status) atomicOr(p.status, CA_STATUS_TABLE);
          id = -1;
        } else if constexpr (C::k8) {
          sk = __ldg(p.ks + (long long)id * p.Hk + kvh);
          sv = __ldg(p.vs + (long long)id * p.Hk + kvh);
        }
      }
    };
    auto tile = [&](int j) {  // tile j of the 32
      SplitTile a;
      const int b = __shfl_sync(0xffffffffu, id, j), o = __shfl_sync(0xffffffffu, off, j),
                t0 = __shfl_sync(0xffffffffu, pos, j);
      a.sk = __shfl_sync(0xffffffffu, sk, j);
      a.sv = __shfl_sync(0xffffffffu, sv, j);
      const long long at = ((long long)max(b, 0) * p.Hk + kvh) * rowbytes;
      a.k = static_cast<const char*>(p.kc) + at + (long long)o * (C::k8 ? E : 4);
      a.v = static_cast<const char*>(p.vc) + at + (long long)o * E * C::ES;
      // keys [0, L - t0) that are first tokens or in the window
      const int top = min(kSplitTile, sq.L - t0);
      uint32_t mask = (1u << top) - 1u;
      if (sq.low > t0) {
        const int lo = min(kSplitTile, sq.low - t0), first = max(0, min(kSplitTile, p.sinks - t0));
        mask &= ~((1u << lo) - 1u) | ((1u << first) - 1u);
      }
      a.mask = b < 0 ? 0u : mask;
      return a;
    };
    meta(0);
    SplitTile cur = tile(0);
    load_q(p, i, kvh, r0, lane, smq);
    load_k(cur, p.page, lane);
    load_v(cur, lane);
    for (int j = 0; j < n; ++j) {
      SplitTile next = cur;
      const bool more = j + 1 < n;
      if (more) {
        if (((j + 1) & 31) == 0) meta(j + 1);
        next = tile((j + 1) & 31);
      }
      float s[4], f[2];
      scores(s, cur, p.page, lane, smq);
      if (more) load_k(next, p.page, lane);
      softmax(s, cur, lane, f);
      values(s, f, cur, lane);
      if (more) load_v(next, lane);
      cur = next;
    }
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) st.l[x] += __shfl_xor_sync(0xffffffffu, st.l[x], o);
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
  return kSplitWarps * 2 * SplitCfg<KIND, E>::kPieceFloats * 4 + kSplitWarps * 2 * (int)sizeof(SplitPiece) +
         (KIND == kSplitF32 ? kSplitWarps * 8 * E * 4 : 0) + 128;
}

template <int KIND, typename QT, int E>
__global__ void __launch_bounds__(32 * kSplitWarps, kSplitCtasPerSm)
    split_decode_kernel(const __grid_constant__ SplitParams p) {
  using C = SplitCfg<KIND, E>;
  extern __shared__ __align__(16) char split_smem[];
  float* pieces = reinterpret_cast<float*>(split_smem);  // [warp][head, tail]
  float* smq = pieces + kSplitWarps * 2 * C::kPieceFloats;
  SplitPiece* info = reinterpret_cast<SplitPiece*>(smq + (KIND == kSplitF32 ? kSplitWarps * 8 * E : 0));
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
      sum += split_seq(p, i).nt;
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
  const long long total = (long long)prefix[p.B] * p.IH;
  const long long warps = (long long)gridDim.x * kSplitWarps;
  const long long chunk = max((long long)p.min_chunk, (total + warps - 1) / warps);
  const long long w0 = ((long long)blockIdx.x * kSplitWarps + warp) * chunk;
  const long long w1 = min(total, w0 + chunk);

  // ---- sequences that see nothing: zeros
  for (int i = blockIdx.x; i < p.B; i += gridDim.x)
    if (prefix[i + 1] == prefix[i]) {
      for (int x = threadIdx.x; x < p.H * E; x += kThreads)
        static_cast<QT*>(p.out)[(long long)i * p.H * E + x] = from_f32<QT>(0.f);
      if (p.lse)
        for (int x = threadIdx.x; x < p.H; x += kThreads) p.lse[(long long)i * p.H + x] = -INFINITY;
    }

  // ---- this warp's tiles
  if (w0 < w1) {
    const long long u = w0 / p.IH;
    int lo = 0, hi = p.B;  // the last i with prefix[i] <= u
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (prefix[mid] <= u)
        lo = mid;
      else
        hi = mid;
    }
    int i = lo;
    const int nt0 = prefix[i + 1] - prefix[i];
    const long long rem = w0 - (long long)prefix[i] * p.IH;
    int ih = (int)(rem / nt0), v = (int)(rem - (long long)ih * nt0);
    SplitSeq sq = split_seq(p, i);
    SplitWarp<KIND, QT, E> w;
    for (long long at = w0;;) {
      const int n = (int)min((long long)(sq.nt - v), w1 - at);
      const int kvh = ih / p.NRG;
      w.run(p, sq, i, kvh, (ih - kvh * p.NRG) * 8, v, n, lane, smq + warp * 8 * E);
      const bool starts = v == 0, ends = v + n == sq.nt;
      if (starts && ends) {
        split_write<KIND, QT, E>(p, w.st, i, ih, lane);
      } else {
        const int slot = warp * 2 + (starts ? 1 : 0);
        w.st.put(pieces + slot * C::kPieceFloats, lane);
        if (lane == 0) info[slot] = SplitPiece{i, ih, ends ? 1 : 0, 1};
      }
      at += n;
      if (at >= w1) break;
      v = 0;
      if (++ih == p.IH) {
        ih = 0;
        do ++i;
        while (prefix[i + 1] == prefix[i]);
        sq = split_seq(p, i);
      }
    }
  }
  if (threadIdx.x == 0) p.meta[4 * blockIdx.x + 3] = 0;
  __syncthreads();

  // ---- join the pieces of one item inside this CTA, in order. A group starts
  // with a warp's tail piece (the item's first tile), or with warp 0's head
  // piece (the item began in an earlier CTA), and goes on through the next
  // warps' head pieces until the item's last tile or the CTA's end.
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
        // the item's last tile, and the CTA that holds it
        const long long end = (long long)prefix[me.i] * p.IH +
                              (long long)(me.ih + 1) * (prefix[me.i + 1] - prefix[me.i]) - 1;
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
// began and did not end, if there is one.
template <int KIND, typename QT, int E>
__global__ void __launch_bounds__(32 * kSplitMergeWarps) split_merge_kernel(const __grid_constant__ SplitParams p) {
  using C = SplitCfg<KIND, E>;
  __shared__ float pieces[kSplitMergeWarps * C::kPieceFloats];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int c = blockIdx.x;
  const int* m = p.meta + 4 * c;
  if (m[3] != 1) return;
  const int last = m[2], n = last - c + 1;
  // warp w joins a contiguous share of the pieces, then warp 0 the shares
  const int per = (n + kSplitMergeWarps - 1) / kSplitMergeWarps;
  SplitState<C::NM> st;
  st.clear();
  for (int k = warp * per; k < min(n, (warp + 1) * per); ++k)
    st.join(p.partial + (2LL * (c + k) + (k == 0 ? 1 : 0)) * C::kPieceFloats, lane);
  st.put(pieces + warp * C::kPieceFloats, lane);
  __syncthreads();
  if (warp == 0) {
#pragma unroll 1
    for (int w = 1; w < kSplitMergeWarps; ++w) st.join(pieces + w * C::kPieceFloats, lane);
    split_write<KIND, QT, E>(p, st, m[0], m[1], lane);
  }
}

}  // namespace ca
