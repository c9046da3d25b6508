// The split decode kernel's instantiations and launch.
#include "split_launch.cuh"

#include "split_decode.cuh"

namespace ca {
namespace {

template <int KIND, typename QT, int E>
cudaError_t launch(SplitParams prm, int ctas, bool after_append, int device, cudaStream_t stream) {
  const int smem = split_smem_fixed<KIND, E>() + 4 * (prm.B + 1);
  auto kern = split_decode_kernel<KIND, QT, E>;
  static unsigned char configured[64] = {};
  if (device < 0 || device >= 64) return cudaErrorInvalidDevice;
  if (!configured[device]) {
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         split_smem_fixed<KIND, E>() + 4 * (kSplitMaxBatch + 1));
    if (e != cudaSuccess) return e;
    configured[device] = 1;  // (a race sets the same value twice)
  }
  // Each launch may start while the one before drains: the decode behind an
  // append of this call (up to its first look at the cache), the join of items
  // cut by a CTA boundary behind the decode.
  cudaLaunchAttribute early = {};
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)ctas);
  cfg.blockDim = dim3(32 * kSplitWarps);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = &early;
  cfg.numAttrs = after_append ? 1 : 0;
  cudaError_t e = cudaLaunchKernelEx(&cfg, kern, prm);
  if (e != cudaSuccess) return e;
  // few items: each is cut into many pieces, which more warps join side by side
  const int shares = 8LL * prm.B * prm.IH <= ctas ? kSplitMergeShares : kSplitMergeShares / 2;
  cfg.blockDim = dim3(32 * shares * (E / 16));
  cfg.dynamicSmemBytes = 0;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, split_merge_kernel<KIND, QT, E>, prm);
}

template <int KIND, typename QT>
cudaError_t by_dim(const SplitParams& prm, int head_dim, int ctas, bool after, int device, cudaStream_t s) {
  switch (head_dim) {
    case 32: return launch<KIND, QT, 32>(prm, ctas, after, device, s);
    case 64: return launch<KIND, QT, 64>(prm, ctas, after, device, s);
    default: return launch<KIND, QT, 128>(prm, ctas, after, device, s);
  }
}

size_t piece_bytes(int head_dim) { return (size_t)(head_dim / 4 + 4) * 32 * 4; }

}  // namespace

size_t split_workspace_bytes(int head_dim, int sms) {
  return (size_t)sms * kSplitCtasPerSm * (2 * piece_bytes(head_dim) + 16);
}

cudaError_t split_launch(const SplitCall& c, int sms, int device, cudaStream_t stream) {
  const int ctas = sms * kSplitCtasPerSm;
  const size_t es = c.q_dtype == CA_DTYPE_BF16 ? 2 : 4;
  // sequences per launch: their tile counts fit shared memory and 32 bits
  const long long row_tiles = std::max(1LL, c.table_width * (c.page / kSplitTile));
  const long long most = std::max(1LL, std::min<long long>(kSplitMaxBatch, 0x7fffffffLL / row_tiles));
  for (long long b0 = 0; b0 < c.batch; b0 += most) {
    SplitParams prm{};
    prm.q = static_cast<const char*>(c.q) + b0 * c.q_stride * (long long)es;
    prm.q_stride = c.q_stride;
    prm.kc = c.kc;
    prm.vc = c.vc;
    prm.ks = c.ks;
    prm.vs = c.vs;
    prm.num_blocks = c.num_blocks;
    prm.lens = c.lens + b0;
    prm.extra = (int)c.n_new;
    prm.page_table = c.page_table + b0 * c.table_width;
    prm.pt_stride = c.table_width;
    prm.out = static_cast<char*>(c.out) + b0 * c.heads * c.head_dim * (long long)es;
    prm.lse = c.lse ? c.lse + b0 * c.heads : nullptr;
    prm.B = (int)std::min(most, c.batch - b0);
    prm.H = (int)c.heads;
    prm.Hk = (int)c.kv_heads;
    prm.G = (int)(c.heads / c.kv_heads);
    prm.NRG = (prm.G + 7) / 8;
    prm.IH = prm.Hk * prm.NRG;
    prm.page = (int)c.page;
    prm.left = c.left < 0 ? -1 : (int)std::min<long long>(c.left, 0x7fffffff);
    prm.sinks = (int)std::min<long long>(c.sinks, 0x7fffff00);
    prm.c = c.c;
    prm.q_vec = (reinterpret_cast<uintptr_t>(prm.q) % 16 == 0) && (c.q_stride * es) % 16 == 0;
    prm.partial = static_cast<float*>(c.workspace);
    prm.meta = reinterpret_cast<int*>(prm.partial + (size_t)ctas * 2 * piece_bytes(c.head_dim) / 4);
    prm.status = c.status;
    const bool after = c.n_new > 0 && b0 == 0;  // the launch before this one is the append
    cudaError_t e;
    if (c.cache_dtype == CA_DTYPE_E4M3)
      e = c.q_dtype == CA_DTYPE_BF16 ? by_dim<kSplitE4m3, __nv_bfloat16>(prm, c.head_dim, ctas, after, device, stream)
                                     : by_dim<kSplitE4m3, float>(prm, c.head_dim, ctas, after, device, stream);
    else if (c.cache_dtype == CA_DTYPE_BF16)
      e = by_dim<kSplitBf16, __nv_bfloat16>(prm, c.head_dim, ctas, after, device, stream);
    else
      e = by_dim<kSplitF32, float>(prm, c.head_dim, ctas, after, device, stream);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

}  // namespace ca
