// New tokens into a paged cache, at cache_seqlens[i] through the page table.
//
// append_8bit_kernel: the cache holds e4m3 codes, [block][head][token][dim],
// and one fp32 scale per (block, head) for K and one for V. For the new tokens
// x of a (block, head):
//     fit = 2^e, the smallest e >= -126 with max |x| <= 448 * 2^e (finite x)
//     s'  = fit when position 0 of the block is among them (the block starts
//           afresh), else max(s, fit);   code = rn_e4m3(x / s')
// and when s' differs from s the block's other codes become rn_e4m3(code *
// (s / s')). Powers of two: x / s' is exact, so a value is rounded once, and a
// block whose scale grows keeps its values but for codes that fall among
// e4m3's subnormals (2^-9 of the unit 2^6 * s'). An infinity is stored as the
// largest code and does not set the scale; NaN stays NaN.
//
// One warp owns a (sequence, touched page, head) of K or of V: it is the only
// writer of that block and scale, so there are no atomics and the result does
// not depend on order. Bound by HBM (2 bytes read and 1 written per value at
// bf16) for prompts: 24.6k tokens of 16 heads of 128 dims, 302 MB, in 49 us
// replayed from a graph (6.2 TB/s, 94% of the measured copy rate), 51 to 54 us
// as calls of their own whose inputs change (85 to 90%); fp32 tokens, 504 MB, in
// 101 us (5.0 TB/s: a lane holds 8 of a 16-token page's 16 vectors and loads the
// rest twice). One token per sequence is a launch and three loads that wait for
// one another (length, block id, scale): 2.6 us.
//
// append_rows_kernel: the same places in a float cache, bit-exact (the layout
// of store.cuh), any number of tokens per sequence.
#pragma once

#include <cuda_fp16.h>

#include "common.cuh"

namespace ca {

struct AppendParams {
  const void* key;
  const void* value;
  long long seq_stride;    // elements between sequences (dense)
  long long token_stride;  // elements between tokens
  void* kc;
  void* vc;
  float* ks;  // [num_blocks, H]
  float* vs;
  long long num_blocks;
  const int* lens;        // [B] lengths before
  const int* page_table;  // [B, width]
  long long pt_stride;
  const int* cu;     // packed: sequence i's new tokens are rows [cu[i], cu[i+1]), or NULL
  long long total;   // packed: rows of key/value
  int n_new;         // tokens per sequence (dense), or the most of any (packed)
  int B, H, page;
  int pages;  // pages a sequence touches at most (packed: all of them)
  long long left, sinks;  // the window of the decode behind this append (left < 0: none)
  int* status;
};

// Sequence i's new tokens: how many, and the element of the first one's row.
__device__ __forceinline__ int append_tokens(const AppendParams& p, int i, long long* row) {
  if (!p.cu) {
    *row = (long long)i * p.seq_stride;
    return p.n_new;
  }
  const long long a = min(max((long long)__ldg(p.cu + i), 0LL), p.total);
  const long long z = min(max((long long)__ldg(p.cu + i + 1), a), p.total);
  *row = a * p.token_stride;
  if (z - a > p.n_new) {
    if (p.status) atomicOr(p.status, CA_STATUS_LENS);
    return p.n_new;
  }
  return (int)(z - a);
}

// Entry b of page pg, or -1: flagged, but where the page lies wholly between the
// first tokens and the window that sees `len` tokens (it may be freed already).
__device__ __forceinline__ int append_block(const AppendParams& p, long long pg, int b, long long len) {
  if (pg >= p.pt_stride) {
    if (p.status) atomicOr(p.status, CA_STATUS_LENS);
    return -1;
  }
  if (b < 0 || b >= p.num_blocks) {
    const bool freed = p.left >= 0 && pg * p.page >= p.sinks && (pg + 1) * p.page <= len - 1 - p.left;
    if (p.status && !freed) atomicOr(p.status, CA_STATUS_TABLE);
    return -1;
  }
  return b;
}

// two fp32 -> two e4m3 (round to nearest even; beyond 448 to 448, NaN stays)
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float2 e4m3x2_to_f32(uint32_t two) {
  uint32_t h;
  const uint16_t x = (uint16_t)two;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(x));
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

// 2^e, the smallest e >= -126 with top <= 448 * 2^e (top finite, >= 0)
__device__ __forceinline__ float e4m3_scale(float top) {
  const uint32_t bits = __float_as_uint(top);
  // exponent of top / 448, rounded up: 448 = 1.75 * 2^8
  int e = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  e = max(e, -126);
  return __uint_as_float((uint32_t)(e + 127) << 23);
}

// A 16-byte vector's values.
template <typename T, int VEC>
__device__ __forceinline__ void append_widen(float (&x)[VEC], const uint4& w) {
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    if constexpr (sizeof(T) == 2) {
      x[2 * c] = bf16_lo(u[c]);
      x[2 * c + 1] = bf16_hi(u[c]);
    } else {
      x[c] = __uint_as_float(u[c]);
    }
  }
}
// VEC values from p (one 16-byte load, or one value)
template <typename T, int VEC>
__device__ __forceinline__ void append_load(float (&x)[VEC], const T* p) {
  if constexpr (VEC == 1)
    x[0] = to_f32(*p);
  else
    append_widen<T>(x, __ldg(reinterpret_cast<const uint4*>(p)));
}

constexpr int kAppendWarps = 4;
// 8 CTAs an SM (64 registers, nothing of bf16 spilled) keep enough loads in flight:
// prompts 49.1 us (graph replay, as all of these); 6 CTAs 55.1, as many as the registers would leave (5) 58.4,
// 10 (held vectors spill) 55.2. One token a sequence does not fill an SM and loses
// 0.1 us to the tighter schedule.
constexpr int kAppendCtas = 8;
constexpr int kAppendHeld = 8;  // vectors a lane keeps between the maximum and the codes

// The largest magnitude of a vector's values and `top`, as bits (two bf16 at a
// time: magnitudes order like whole numbers; infinities and NaN are the largest).
template <typename T>
__device__ __forceinline__ uint32_t append_top(const uint4& w, uint32_t top) {
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    if constexpr (sizeof(T) == 2)
      asm("max.u16x2 %0, %0, %1;" : "+r"(top) : "r"(u[c] & 0x7fff7fffu));
    else
      top = max(top, u[c] & 0x7fffffffu);
  }
  return top;
}
template <int VEC>
__device__ __forceinline__ void append_codes(const float (&v)[VEC], uint8_t* dst) {
  if constexpr (VEC == 8) {
    const uint32_t w0 = e4m3x2(v[0], v[1]) | e4m3x2(v[2], v[3]) << 16;
    const uint32_t w1 = e4m3x2(v[4], v[5]) | e4m3x2(v[6], v[7]) << 16;
    *reinterpret_cast<uint2*>(dst) = make_uint2(w0, w1);
  } else if constexpr (VEC == 4) {
    *reinterpret_cast<uint32_t*>(dst) = e4m3x2(v[0], v[1]) | e4m3x2(v[2], v[3]) << 16;
  } else {
    *dst = (uint8_t)e4m3x2(v[0], 0.f);
  }
}
// The other codes of a block whose scale moved from `old` to `now`.
__device__ __noinline__ void append_rescale(uint8_t* block, int bytes, int lo, int hi, float old, float now, int lane) {
  const float ratio = __fdiv_rn(old, now);
  uint32_t* w = reinterpret_cast<uint32_t*>(block);
  for (int x = lane; x < bytes / 4; x += 32) {
    if (4 * x >= lo && 4 * x < hi) continue;
    const uint32_t c = w[x];
    const float2 f0 = e4m3x2_to_f32(c), f1 = e4m3x2_to_f32(c >> 16);
    w[x] = e4m3x2(f0.x * ratio, f0.y * ratio) | e4m3x2(f1.x * ratio, f1.y * ratio) << 16;
  }
}

// A vector's values times inv, a power of two (bf16: two at a time, exact but
// for results below bf16's normal range, whose codes are 0).
template <typename T, int VEC>
__device__ __forceinline__ void append_scaled(float (&v)[VEC], uint4 w, float inv) {
  if constexpr (sizeof(T) == 2) {
    const __nv_bfloat162 by = __float2bfloat162_rn(inv);
    __nv_bfloat162* u = reinterpret_cast<__nv_bfloat162*>(&w);
#pragma unroll
    for (int c = 0; c < 4; ++c) u[c] = __hmul2(u[c], by);
    append_widen<T>(v, w);
  } else {
    append_widen<T>(v, w);
#pragma unroll
    for (int c = 0; c < VEC; ++c) v[c] *= inv;
  }
}

// Where packed sequence i's pages start among the launch's (their number grows
// by at least what the sequence's tokens can touch).
__device__ __forceinline__ long long append_start(const AppendParams& p, int i) {
  return __ldg(p.cu + i) / p.page + 2LL * i;
}
// The last sequence that starts at or before page u (32 probes at a time).
__device__ __forceinline__ int append_sequence(const AppendParams& p, long long u, int lane) {
  int lo = 0, n = p.B;  // it is in [lo, lo + n)
  while (n > 1) {
    const int step = (n + 31) / 32;
    const int at = lo + lane * step;
    const bool before = lane * step < n && append_start(p, at) <= u;
    const int k = max(0, __popc(__ballot_sync(0xffffffffu, before)) - 1);
    n = min(step, n - k * step);
    lo += k * step;
  }
  return lo;
}

// Grid: x = group of 4 (head, side) units of a page, y = sequence; packed: x =
// all pages of all sequences, so short sequences beside long ones cost nothing.
// The rows are loaded before the block id is known; a 16-token page of head_dim
// 128 (bf16) stays in registers, so new tokens are read once.
template <typename T, int E, bool VEC16>
__global__ void __launch_bounds__(32 * kAppendWarps, kAppendCtas) append_8bit_kernel(const __grid_constant__ AppendParams p) {
  constexpr int VEC = VEC16 ? 16 / (int)sizeof(T) : 1;
  constexpr int PER_ROW = E / VEC;                            // vectors of a row
  constexpr int LANES = PER_ROW < 32 ? PER_ROW : 32;          // lanes that share a row
  constexpr int ROWS = 32 / LANES, STEPS = PER_ROW / LANES;   // rows a warp takes at a time, steps they take
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // (a decode waits before it reads the cache)
  const int lane = threadIdx.x & 31;
  const unsigned groups = (2u * p.H + kAppendWarps - 1) / kAppendWarps;
  const int pi = (int)(blockIdx.x / groups);
  const int unit = (int)(blockIdx.x - pi * groups) * kAppendWarps + (threadIdx.x >> 5);
  if (unit >= 2 * p.H) return;
  const int h = unit >> 1, side = unit & 1;
  const int r0 = lane / LANES, c0 = (lane % LANES) * VEC;
  const int first = p.cu ? append_sequence(p, pi, lane) : (int)blockIdx.y;
  for (int i = first; i < p.B; i += p.cu ? p.B : (int)gridDim.y) {
    const int before = __ldg(p.lens + i);
    if (before < 0) continue;
    long long row;
    const int n = append_tokens(p, i, &row);
    const int mine = p.cu ? (int)(pi - append_start(p, i)) : pi;  // of the pages the sequence touches
    if (mine < 0) continue;
    const int pg = before / p.page + mine;
    const long long p0 = (long long)pg * p.page;
    const long long a = max((long long)before, p0), z = min((long long)before + n, p0 + p.page);
    if (a >= z) continue;
    const int id = pg < p.pt_stride ? __ldg(p.page_table + i * p.pt_stride + pg) : -1;
    const T* src = static_cast<const T*>(side ? p.value : p.key) + row + (a - before) * p.token_stride +
                   (long long)h * E + r0 * p.token_stride + c0;
    const long long down = ROWS * p.token_stride;
    const int rows = (int)(z - a) - r0;  // of this lane: r0, r0 + ROWS, ...
    uint4 held[kAppendHeld];
    if constexpr (VEC16) {
      const T* at = src;
#pragma unroll
      for (int k = 0; k < kAppendHeld; ++k, at += down) {
        held[k] = make_uint4(0u, 0u, 0u, 0u);
        if (k * ROWS < rows) held[k] = __ldg(reinterpret_cast<const uint4*>(at));
      }
    }
    const int b = append_block(p, pg, id, (long long)before + n);
    if (b < 0) continue;
    float* scale = (side ? p.vs : p.ks) + (long long)b * p.H + h;
    uint8_t* block = static_cast<uint8_t*>(side ? p.vc : p.kc) + ((long long)b * p.H + h) * p.page * E;
    const bool fresh = a == p0;
    const float old = fresh ? 0.f : *scale;

    // the largest magnitude; once more without what is not finite if there is any
    uint32_t bits = 0u;
    constexpr int kFirst = VEC16 ? kAppendHeld : 0;
    if constexpr (VEC16) {
#pragma unroll
      for (int k = 0; k < kAppendHeld; ++k) bits = append_top<T>(held[k], bits);
      const T* at = src + kFirst * down;
      for (int k = kFirst; k * ROWS < rows; ++k, at += down)
        bits = append_top<T>(__ldg(reinterpret_cast<const uint4*>(at)), bits);
      if constexpr (sizeof(T) == 2) bits = max(bits & 0xffffu, bits >> 16) << 16;
    } else {
      const T* at = src;
      for (int k = 0; k * ROWS < rows; ++k, at += down)
#pragma unroll
        for (int c = 0; c < STEPS; ++c) bits = max(bits, __float_as_uint(to_f32(at[c * LANES])) & 0x7fffffffu);
    }
    bits = __reduce_max_sync(0xffffffffu, bits);
    if (bits >= 0x7f800000u) {
      bits = 0u;
      const T* at = src;
      for (int k = 0; k * ROWS < rows; ++k, at += down)
        for (int c = 0; c < STEPS; ++c)
          for (int e = 0; e < VEC; ++e) {
            const uint32_t m = __float_as_uint(to_f32(at[c * LANES * VEC + e])) & 0x7fffffffu;
            if (m < 0x7f800000u) bits = max(bits, m);
          }
      bits = __reduce_max_sync(0xffffffffu, bits);
    }
    const float now = fmaxf(old, e4m3_scale(__uint_as_float(bits)));
    if (!fresh && now != old)
      append_rescale(block, p.page * E, (int)(a - p0) * E, (int)(z - p0) * E, old, now, lane);
    uint8_t* dst = block + ((int)(a - p0) + r0) * E + c0;
    if ((__float_as_uint(now) & 0x7fffffu) == 0u) {
      const float inv = 1.f / now;  // exact: now is a power of two
      if constexpr (VEC16) {
#pragma unroll
        for (int k = 0; k < kAppendHeld; ++k)
          if (k * ROWS < rows) {
            float v[VEC];
            append_scaled<T>(v, held[k], inv);
            append_codes(v, dst + k * ROWS * E);
          }
      }
      const T* at = src + kFirst * down;
      for (int k = kFirst; k * ROWS < rows; ++k, at += down)
#pragma unroll
        for (int c = 0; c < STEPS; ++c) {
          float v[VEC];
          if constexpr (VEC16) {
            append_scaled<T>(v, __ldg(reinterpret_cast<const uint4*>(at + c * LANES * VEC)), inv);
          } else {
            append_load<T, VEC>(v, at + c * LANES * VEC);
            v[0] *= inv;
          }
          append_codes(v, dst + k * ROWS * E + c * LANES * VEC);
        }
    } else {
      // the caller's own scale was larger: the quotient is rounded once before the code is
      const T* at = src;
      for (int k = 0; k * ROWS < rows; ++k, at += down)
        for (int c = 0; c < STEPS; ++c) {
          float v[VEC];
          append_load<T, VEC>(v, at + c * LANES * VEC);
#pragma unroll
          for (int e = 0; e < VEC; ++e) v[e] = __fdiv_rn(v[e], now);
          append_codes(v, dst + k * ROWS * E + c * LANES * VEC);
        }
    }
    if (lane == 0 && now != old) *scale = now;
  }
}

// Float caches: one thread moves one element or 16-byte vector of a (sequence,
// token, head) row of K and of V (dense rows only).
template <typename T, int E, bool VEC16>
__global__ void __launch_bounds__(256) append_rows_kernel(const __grid_constant__ AppendParams p) {
  constexpr int VEC = VEC16 ? 16 / (int)sizeof(T) : 1;
  constexpr int PER_ROW = E / VEC;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // (a decode waits before it reads the cache)
  const long long idx = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  const int v = (int)(idx % PER_ROW);
  long long r = idx / PER_ROW;
  const int h = (int)(r % p.H);
  r /= p.H;
  const int j = (int)(r % p.n_new);
  const long long i = r / p.n_new;
  if (i >= p.B) return;
  const int before = __ldg(p.lens + i);
  if (before < 0) return;
  const long long pos = (long long)before + j;
  const long long pg = pos / p.page;
  const int b = append_block(p, pg, pg < p.pt_stride ? __ldg(p.page_table + i * p.pt_stride + pg) : -1,
                             (long long)before + p.n_new);
  if (b < 0) return;
  const int off = (int)(pos - pg * p.page);
  const long long src = i * p.seq_stride + j * p.token_stride + (long long)h * E + v * VEC;
  const long long base = ((long long)b * p.H + h) * p.page * E;
  const T* ks = static_cast<const T*>(p.key) + src;
  const T* vs = static_cast<const T*>(p.value) + src;
  T* kd = static_cast<T*>(p.kc) + base;
  T* vd = static_cast<T*>(p.vc) + base + (long long)off * E + v * VEC;
  if constexpr (VEC16) {
    const uint4 kw = *reinterpret_cast<const uint4*>(ks);
    *reinterpret_cast<uint4*>(vd) = *reinterpret_cast<const uint4*>(vs);
    const uint32_t w[4] = {kw.x, kw.y, kw.z, kw.w};
    uint32_t* kdw = reinterpret_cast<uint32_t*>(kd);  // bf16: words of dim pairs, fp32: dims
#pragma unroll
    for (int c = 0; c < 4; ++c) kdw[(long long)(v * 4 + c) * p.page + off] = w[c];
  } else {
    *vd = *vs;
    if constexpr (sizeof(T) == 2)
      kd[((long long)(v >> 1) * p.page + off) * 2 + (v & 1)] = *ks;
    else
      kd[(long long)v * p.page + off] = *ks;
  }
}

}  // namespace ca
