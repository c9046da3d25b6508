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
// bf16) for prompts, by three dependent loads (length, block id, rows) for
// one token per sequence.
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
  int pages;  // pages a sequence touches at most
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

// The block of page pg of sequence i, or -1 (flagged).
__device__ __forceinline__ int append_block(const AppendParams& p, int i, long long pg) {
  if (pg >= p.pt_stride) {
    if (p.status) atomicOr(p.status, CA_STATUS_LENS);
    return -1;
  }
  const int b = __ldg(p.page_table + i * p.pt_stride + pg);
  if (b < 0 || b >= p.num_blocks) {
    if (p.status) atomicOr(p.status, CA_STATUS_TABLE);
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

// VEC values from p (VEC16: one 16-byte load, else one value)
template <typename T, int VEC>
__device__ __forceinline__ void append_load(float (&x)[VEC], const T* p) {
  if constexpr (VEC == 1) {
    x[0] = to_f32(*p);
  } else {
    const uint4 w = *reinterpret_cast<const uint4*>(p);
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
}

constexpr int kAppendWarps = 4;

template <typename T, int E, bool VEC16>
__global__ void __launch_bounds__(32 * kAppendWarps) append_8bit_kernel(const __grid_constant__ AppendParams p) {
  constexpr int VEC = VEC16 ? 16 / (int)sizeof(T) : 1;
  constexpr int PER_ROW = E / VEC;
  const int lane = threadIdx.x & 31;
  // unit = ((sequence * pages + page) * H + head) * 2 + side
  long long u = (long long)blockIdx.x * kAppendWarps + (threadIdx.x >> 5);
  const int side = (int)(u & 1);
  u >>= 1;
  const int h = (int)(u % p.H);
  u /= p.H;
  const int pi = (int)(u % p.pages);
  const long long i = u / p.pages;
  if (i >= p.B) return;
  const int before = __ldg(p.lens + i);
  if (before < 0) return;
  long long row;
  const int n = append_tokens(p, (int)i, &row);
  const long long pg = before / p.page + pi;
  const long long p0 = pg * p.page;
  const long long a = max((long long)before, p0), z = min((long long)before + n, p0 + p.page);
  if (a >= z) return;
  const int b = append_block(p, (int)i, pg);
  if (b < 0) return;
  const T* src = static_cast<const T*>(side ? p.value : p.key) + row + (a - before) * p.token_stride + (long long)h * E;
  float* scale = (side ? p.vs : p.ks) + (long long)b * p.H + h;
  uint8_t* dst = static_cast<uint8_t*>(side ? p.vc : p.kc) + ((long long)b * p.H + h) * p.page * E;
  const int vecs = (int)(z - a) * PER_ROW;
  const bool fresh = a == p0;
  const float old = fresh ? 0.f : *scale;

  float top = 0.f;
#pragma unroll 4
  for (int x = lane; x < vecs; x += 32) {
    float v[VEC];
    append_load<T, VEC>(v, src + (long long)(x / PER_ROW) * p.token_stride + (x % PER_ROW) * VEC);
#pragma unroll
    for (int c = 0; c < VEC; ++c) {
      const float m = fabsf(v[c]);
      if (m < INFINITY) top = fmaxf(top, m);
    }
  }
  top = warp_max(top);
  const float now = fmaxf(old, e4m3_scale(top));
  // the block's other tokens, when the scale moved
  if (!fresh && now != old) {
    const float ratio = __fdiv_rn(old, now);
    const int lo = (int)(a - p0) * E, hi = (int)(z - p0) * E;
    uint32_t* w = reinterpret_cast<uint32_t*>(dst);
    for (int x = lane; x < p.page * E / 4; x += 32) {
      if (4 * x >= lo && 4 * x < hi) continue;
      const uint32_t c = w[x];
      const float2 f0 = e4m3x2_to_f32(c), f1 = e4m3x2_to_f32(c >> 16);
      w[x] = e4m3x2(f0.x * ratio, f0.y * ratio) | e4m3x2(f1.x * ratio, f1.y * ratio) << 16;
    }
  }
  // now is a power of two unless the caller's own scale was larger: then the
  // quotient is rounded once before the code is
  dst += (a - p0) * E;
#pragma unroll 4
  for (int x = lane; x < vecs; x += 32) {
    float v[VEC];
    append_load<T, VEC>(v, src + (long long)(x / PER_ROW) * p.token_stride + (x % PER_ROW) * VEC);
#pragma unroll
    for (int c = 0; c < VEC; ++c) v[c] = __fdiv_rn(v[c], now);
    if constexpr (VEC == 8) {
      const uint32_t w0 = e4m3x2(v[0], v[1]) | e4m3x2(v[2], v[3]) << 16;
      const uint32_t w1 = e4m3x2(v[4], v[5]) | e4m3x2(v[6], v[7]) << 16;
      *reinterpret_cast<uint2*>(dst + (long long)x * 8) = make_uint2(w0, w1);
    } else if constexpr (VEC == 4) {
      *reinterpret_cast<uint32_t*>(dst + (long long)x * 4) = e4m3x2(v[0], v[1]) | e4m3x2(v[2], v[3]) << 16;
    } else {
      dst[x] = (uint8_t)e4m3x2(v[0], 0.f);
    }
  }
  if (lane == 0 && now != old) *scale = now;
}

// Float caches: one thread moves one element or 16-byte vector of a (sequence,
// token, head) row of K and of V (dense rows only).
template <typename T, int E, bool VEC16>
__global__ void __launch_bounds__(256) append_rows_kernel(const __grid_constant__ AppendParams p) {
  constexpr int VEC = VEC16 ? 16 / (int)sizeof(T) : 1;
  constexpr int PER_ROW = E / VEC;
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
  const int b = append_block(p, (int)i, pg);
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
