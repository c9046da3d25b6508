// The C ABI's serving entries beside the reference's three: caches held in 8
// bits, decode over them and behind a sliding window, and block moves.
// Declarations and the contract live in include/cpu_attention_b200.h.
#include <cmath>

#include "append.cuh"
#include "blocks.cuh"
#include "split_launch.cuh"

namespace {

bool head_dim_ok(long long e) { return e == 32 || e == 64 || e == 128; }
bool page_ok(long long page) { return page > 0 && page % 16 == 0 && page <= (1 << 20); }
size_t elem_size(int dtype) { return dtype == CA_DTYPE_BF16 ? 2 : 4; }
bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }

template <typename T, int E>
int launch_append(const ca::AppendParams& prm, bool eight, bool vec16, cudaStream_t stream) {
  if (eight) {
    const long long ctas = (long long)prm.pages * ((2 * prm.H + ca::kAppendWarps - 1) / ca::kAppendWarps);
    if (ctas > 0x7fffffffLL) return CA_EUNSUPPORTED;
    auto kern = vec16 ? ca::append_8bit_kernel<T, E, true> : ca::append_8bit_kernel<T, E, false>;
    const dim3 grid((unsigned)ctas, prm.cu ? 1u : (unsigned)std::min(prm.B, 65535));
    kern<<<grid, 32 * ca::kAppendWarps, 0, stream>>>(prm);
  } else {
    const long long per_row = vec16 ? E / (16 / (int)sizeof(T)) : E;
    const long long ctas = ((long long)prm.B * prm.n_new * prm.H * per_row + 255) / 256;
    if (ctas > 0x7fffffffLL) return CA_EUNSUPPORTED;
    auto kern = vec16 ? ca::append_rows_kernel<T, E, true> : ca::append_rows_kernel<T, E, false>;
    kern<<<(unsigned)ctas, 256, 0, stream>>>(prm);
  }
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? CA_OK : ca::host_cuda_fail(e, "append launch");
}

int append(const ca::AppendParams& prm, long long head_dim, int dtype, bool eight, bool vec16, cudaStream_t s) {
  if (dtype == CA_DTYPE_BF16) {
    switch (head_dim) {
      case 32: return launch_append<__nv_bfloat16, 32>(prm, eight, vec16, s);
      case 64: return launch_append<__nv_bfloat16, 64>(prm, eight, vec16, s);
      default: return launch_append<__nv_bfloat16, 128>(prm, eight, vec16, s);
    }
  }
  switch (head_dim) {
    case 32: return launch_append<float, 32>(prm, eight, vec16, s);
    case 64: return launch_append<float, 64>(prm, eight, vec16, s);
    default: return launch_append<float, 128>(prm, eight, vec16, s);
  }
}

// The checks and parameters both appends share.
int append_plan(ca::AppendParams* prm, const void* key, const void* value, int64_t seq_stride, int64_t token_stride,
                int64_t n_new, const int32_t* cu, int64_t total, void* kc, void* vc, float* ks, float* vs,
                int64_t num_blocks, const int32_t* lens, const int32_t* page_table, int64_t table_width,
                int64_t batch, int64_t heads, int64_t head_dim, int64_t page, int dtype, int32_t* status,
                bool* vec16) {
  // (an empty pool or table has no address, and is not read)
  if (!key || !value || !lens || (num_blocks && (!kc || !vc)) || (table_width && !page_table)) return CA_ENULL;
  const size_t es = elem_size(dtype);
  if (token_stride < heads * head_dim && (cu ? total > 1 : n_new > 1)) return CA_ELAYOUT;
  if (!cu && seq_stride < (n_new > 1 ? n_new * token_stride : heads * head_dim) && batch > 1) return CA_ELAYOUT;
  if (!aligned(key, es) || !aligned(value, es) || !aligned(kc, 16) || !aligned(vc, 16)) return CA_ELAYOUT;
  *vec16 = aligned(key, 16) && aligned(value, 16) && (cu || (seq_stride * es) % 16 == 0) &&
           ((n_new == 1 && !cu) || (token_stride * es) % 16 == 0);
  prm->key = key;
  prm->value = value;
  prm->seq_stride = seq_stride;
  prm->token_stride = token_stride;
  prm->kc = kc;
  prm->vc = vc;
  prm->ks = ks;
  prm->vs = vs;
  prm->num_blocks = num_blocks;
  prm->lens = lens;
  prm->page_table = page_table;
  prm->pt_stride = table_width;
  prm->cu = cu;
  prm->total = total;
  prm->n_new = (int)n_new;
  prm->B = (int)batch;
  prm->H = (int)heads;
  prm->page = (int)page;
  const int64_t pages = cu ? total / page + 2 * batch : (n_new + page - 2) / page + 1;
  if (pages > 0x7fffffffLL) return CA_EUNSUPPORTED;
  prm->pages = (int)pages;
  prm->left = -1;
  prm->status = status;
  return CA_OK;
}

bool sizes_ok(int64_t batch, int64_t heads, int64_t num_blocks, int64_t table_width, int64_t n_new) {
  return batch >= 0 && batch <= (1 << 24) && heads > 0 && heads <= (1 << 16) && num_blocks >= 0 &&
         num_blocks <= 0x7fffffffLL && table_width >= 0 && table_width <= 0x7fffffffLL && n_new >= 0 &&
         n_new <= (1 << 28);
}

int copy_params(ca::CopyParams* prm, void* const* base, const int64_t* bytes, int64_t first, int64_t tensors,
                int64_t num_blocks, int32_t* status) {
  prm->tensors = (int)std::min<int64_t>(ca::kCopyTensors, tensors - first);
  int at = 0;
  for (int small = 0; small < 2; ++small) {
    for (int t = 0; t < prm->tensors; ++t)
      if ((bytes[first + t] <= ca::kCopySmall) == (small != 0)) {
        prm->base[at] = static_cast<char*>(base[first + t]);
        prm->bytes[at++] = bytes[first + t];
      }
    if (!small) prm->large = at;
  }
  prm->num_blocks = num_blocks;
  prm->status = status;
  return CA_OK;
}

int copy_checks(void* const* base, const int64_t* bytes, int64_t tensors, int64_t num_blocks) {
  if (tensors < 0 || num_blocks < 0 || num_blocks > 0x7fffffffLL) return CA_ESHAPE;
  if (tensors && (!base || !bytes)) return CA_ENULL;
  for (int64_t t = 0; t < tensors; ++t) {
    if (!base[t]) return CA_ENULL;
    if (bytes[t] < 1) return CA_ESHAPE;
  }
  return CA_OK;
}

}  // namespace

extern "C" {

int ca_append_8bit(const void* key, const void* value, int64_t seq_stride, int64_t token_stride, int64_t n_new,
                   const int32_t* cu_new, int64_t total_new, void* k_cache, void* v_cache, float* k_scale,
                   float* v_scale, int64_t num_blocks, const int32_t* lens, const int32_t* page_table,
                   int64_t table_width, int64_t batch, int64_t heads, int64_t head_dim, int64_t page, int dtype,
                   int32_t* status, void* stream) {
  if (dtype != CA_DTYPE_F32 && dtype != CA_DTYPE_BF16) return CA_EDTYPE;
  if (!head_dim_ok(head_dim)) return CA_EHEADDIM;
  if (!page_ok(page)) return CA_EPAGE;
  if (!sizes_ok(batch, heads, num_blocks, table_width, n_new) || total_new < 0) return CA_ESHAPE;
  // (packed tokens with n_new = 0 go on: a sequence that has some is flagged)
  if (batch == 0 || (cu_new ? total_new == 0 : n_new == 0)) return CA_OK;
  if (num_blocks && (!k_scale || !v_scale)) return CA_ENULL;
  if (!aligned(k_scale, 4) || !aligned(v_scale, 4)) return CA_ELAYOUT;
  ca::AppendParams prm{};
  bool vec16;
  const int rc = append_plan(&prm, key, value, seq_stride, token_stride, n_new, cu_new, total_new, k_cache, v_cache,
                             k_scale, v_scale, num_blocks, lens, page_table, table_width, batch, heads, head_dim,
                             page, dtype, status, &vec16);
  if (rc) return rc;
  return append(prm, head_dim, dtype, true, vec16, static_cast<cudaStream_t>(stream));
}

size_t ca_decode_split_workspace_bytes(int64_t head_dim, int device) {
  if (!head_dim_ok(head_dim)) return 0;
  int sms = 0;
  if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device) != cudaSuccess) return 0;
  return ca::split_workspace_bytes((int)head_dim, sms);
}

int ca_decode_split(const void* q, int64_t q_stride, void* k_cache, void* v_cache, float* k_scale, float* v_scale,
                    int64_t num_blocks, const void* k_new, const void* v_new, int64_t kv_stride,
                    int64_t kv_token_stride, int64_t n_new, const int32_t* lens, const int32_t* page_table,
                    int64_t table_width, void* out, float* lse, int64_t batch, int64_t heads, int64_t kv_heads,
                    int64_t head_dim, int64_t page, int q_dtype, int cache_dtype, int64_t window_left,
                    int64_t sink_tokens, float softmax_scale, void* workspace, size_t workspace_bytes,
                    int32_t* status, void* stream) {
  if (q_dtype != CA_DTYPE_F32 && q_dtype != CA_DTYPE_BF16) return CA_EDTYPE;
  const bool eight = cache_dtype == CA_DTYPE_E4M3;
  if (!eight && cache_dtype != q_dtype) return CA_EDTYPE;
  if (!head_dim_ok(head_dim)) return CA_EHEADDIM;
  if (!page_ok(page)) return CA_EPAGE;
  if (!sizes_ok(batch, heads, num_blocks, table_width, n_new) || kv_heads <= 0 || heads % kv_heads) return CA_ESHAPE;
  if (batch * heads > (1LL << 30) || window_left < -1 || sink_tokens < 0) return CA_ESHAPE;
  if (table_width * page > 0x7fffffffLL) return CA_ESHAPE;
  if ((k_new == nullptr) != (v_new == nullptr) || (k_new == nullptr) != (n_new == 0)) return CA_ESHAPE;
  if (batch == 0) return CA_OK;
  if (!q || !lens || !out || !workspace || (table_width && !page_table)) return CA_ENULL;
  if (num_blocks && (!k_cache || !v_cache || (eight && (!k_scale || !v_scale)))) return CA_ENULL;
  if (q_stride < heads * head_dim && batch > 1) return CA_ELAYOUT;
  const size_t es = elem_size(q_dtype);
  if (!aligned(q, es) || !aligned(out, 2 * es) || !aligned(lse, 4) || !aligned(k_cache, 16) ||
      !aligned(v_cache, 16) || !aligned(k_scale, 4) || !aligned(v_scale, 4) || !aligned(workspace, 16))
    return CA_ELAYOUT;
  int sms;
  int rc = ca::host_sms(&sms);
  if (rc) return rc;
  if (workspace_bytes < ca::split_workspace_bytes((int)head_dim, sms)) return CA_EWORKSPACE;
  int device;
  cudaError_t e = cudaGetDevice(&device);
  if (e != cudaSuccess) return ca::host_cuda_fail(e, "cudaGetDevice");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (n_new) {
    ca::AppendParams prm{};
    bool vec16;
    rc = append_plan(&prm, k_new, v_new, kv_stride, kv_token_stride, n_new, nullptr, 0, k_cache, v_cache, k_scale,
                     v_scale, num_blocks, lens, page_table, table_width, batch, kv_heads, head_dim, page, q_dtype,
                     status, &vec16);
    if (rc) return rc;
    prm.left = window_left;
    prm.sinks = sink_tokens;
    if ((rc = append(prm, head_dim, q_dtype, eight, vec16, s))) return rc;
  }
  ca::SplitCall c{};
  c.q = q;
  c.q_stride = q_stride;
  c.kc = k_cache;
  c.vc = v_cache;
  c.ks = k_scale;
  c.vs = v_scale;
  c.num_blocks = num_blocks;
  c.lens = lens;
  c.n_new = n_new;
  c.page_table = page_table;
  c.table_width = table_width;
  c.out = out;
  c.lse = lse;
  c.batch = batch;
  c.heads = heads;
  c.kv_heads = kv_heads;
  c.head_dim = (int)head_dim;
  c.page = page;
  c.q_dtype = q_dtype;
  c.cache_dtype = cache_dtype;
  c.left = window_left;
  c.sinks = sink_tokens;
  const double scale = std::isnan(softmax_scale) ? 1.0 / std::sqrt((double)head_dim) : (double)softmax_scale;
  c.c = (float)(scale * 1.4426950408889634);
  c.workspace = workspace;
  c.status = status;
  e = ca::split_launch(c, sms, device, s);
  return e == cudaSuccess ? CA_OK : ca::host_cuda_fail(e, "split decode launch");
}

int ca_copy_blocks(void* const* base, const int64_t* block_bytes, int64_t tensors, int64_t num_blocks,
                   const int64_t* pairs, int64_t n, int32_t* status, void* stream) {
  int rc = copy_checks(base, block_bytes, tensors, num_blocks);
  if (rc) return rc;
  if (n < 0) return CA_ESHAPE;
  if (n == 0 || tensors == 0) return CA_OK;
  if (!pairs) return CA_ENULL;
  for (int64_t first = 0; first < tensors; first += ca::kCopyTensors) {
    ca::CopyParams prm{};
    copy_params(&prm, base, block_bytes, first, tensors, num_blocks, status);
    prm.pairs = reinterpret_cast<const long long*>(pairs);
    prm.n = n;
    const int64_t units = n > (1LL << 40) / prm.tensors ? (1LL << 40) : n * prm.tensors;
    ca::copy_blocks_kernel<<<(unsigned)std::min<int64_t>(units, 1 << 16), ca::kCopyThreads, 0,
                             static_cast<cudaStream_t>(stream)>>>(prm);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return ca::host_cuda_fail(e, "copy launch");
  }
  return CA_OK;
}

// moves [num_blocks][2], place [num_blocks], count
size_t ca_compact_workspace_bytes(int64_t num_blocks) { return num_blocks < 0 ? 0 : (size_t)num_blocks * 12 + 16; }

int ca_compact_blocks(void* const* base, const int64_t* block_bytes, int64_t tensors, int64_t num_blocks,
                      const int32_t* page_table, const int32_t* lens, int64_t batch, int64_t table_width,
                      int64_t page, int64_t window_left, int64_t sink_tokens, int32_t* new_table, int32_t* used,
                      void* workspace, size_t workspace_bytes, int32_t* status, void* stream) {
  return ca_compact_blocks_ex(base, block_bytes, tensors, num_blocks, page_table, lens, nullptr, batch, table_width,
                              page, window_left, sink_tokens, new_table, used, workspace, workspace_bytes, status,
                              stream);
}

int ca_compact_blocks_ex(void* const* base, const int64_t* block_bytes, int64_t tensors, int64_t num_blocks,
                         const int32_t* page_table, const int32_t* lens, const int32_t* reserved, int64_t batch,
                         int64_t table_width, int64_t page, int64_t window_left, int64_t sink_tokens,
                         int32_t* new_table, int32_t* used, void* workspace, size_t workspace_bytes, int32_t* status,
                         void* stream) {
  int rc = copy_checks(base, block_bytes, tensors, num_blocks);
  if (rc) return rc;
  if (!page_ok(page)) return CA_EPAGE;
  if (!sizes_ok(batch, 1, num_blocks, table_width, 0) || window_left < -1 || sink_tokens < 0) return CA_ESHAPE;
  if (num_blocks > ca::kPlanMaxBlocks) return CA_EUNSUPPORTED;
  if (!used || !workspace) return CA_ENULL;
  if (batch && table_width && (!page_table || !lens || !new_table)) return CA_ENULL;
  if (!aligned(workspace, 16)) return CA_ELAYOUT;
  if (workspace_bytes < ca_compact_workspace_bytes(num_blocks)) return CA_EWORKSPACE;
  ca::CompactParams p{};
  p.page_table = page_table;
  p.lens = lens;
  p.reserved = reserved;
  p.new_table = new_table;
  p.used = used;
  p.count = static_cast<int*>(workspace);
  p.moves = p.count + 4;
  p.place = p.moves + 2 * num_blocks;
  p.num_blocks = num_blocks;
  p.B = (int)batch;
  p.width = (int)table_width;
  p.page = (int)page;
  p.left = window_left < 0 ? -1 : (int)std::min<int64_t>(window_left, 0x7fffffff);
  p.sinks = (int)std::min<int64_t>(sink_tokens, 0x7fffffff);
  p.status = status;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int bitmap = (int)((num_blocks + 31) / 32) * 4;
  cudaError_t e = cudaFuncSetAttribute(ca::compact_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       ca::kPlanMaxBlocks / 8);
  if (e != cudaSuccess) return ca::host_cuda_fail(e, "cudaFuncSetAttribute(compact)");
  ca::compact_plan_kernel<<<1, ca::kPlanThreads, bitmap, s>>>(p);
  e = cudaGetLastError();
  if (e != cudaSuccess) return ca::host_cuda_fail(e, "compact launch");
  int sms;
  if ((rc = ca::host_sms(&sms))) return rc;
  for (int64_t first = 0; first < tensors; first += ca::kCopyTensors) {
    ca::CopyParams prm{};
    copy_params(&prm, base, block_bytes, first, tensors, num_blocks, status);
    prm.moves = p.moves;
    prm.count = p.count;
    // (how many blocks move is known on the device only: 8 CTAs an SM share them.
    // The first launch may come up while the plan is made.)
    cudaLaunchAttribute early = {};
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(8 * sms));
    cfg.blockDim = dim3(ca::kCopyThreads);
    cfg.stream = s;
    cfg.attrs = &early;
    cfg.numAttrs = first == 0 ? 1 : 0;
    e = cudaLaunchKernelEx(&cfg, ca::copy_blocks_kernel, prm);
    if (e != cudaSuccess) return ca::host_cuda_fail(e, "compact copy launch");
  }
  return CA_OK;
}

}  // extern "C"
