// The decode, prefill and store entries' host path in C++: the same argument
// checks as cpu_attention/_native.py::decode, ::flash and ::store (which
// mirror `_C.mojo:87-171`, `:232-316` and `:174-213`), done on at::Tensor
// fields instead of Python attribute calls, then the C ABI call (ca_decode_ex /
// ca_flash_ex / ca_store) on the device's current stream; the entries for 8-bit caches, windows and block
// moves likewise. Varlen prefill and prefill log-sum-exp without a window take the Python path. A decode step is short enough
// (tens of µs) that the Python checks and the ctypes call were the larger part
// of an end-to-end step's host time.
//
// Every decline returns None, exactly where the Python path returns None, so
// the caller then runs the reference's checks to raise the precise error.
// The per-(device, stream) workspaces live here too (the Python workspace()
// hands out the same tensors), so status reads see what the kernels wrote.

#include <torch/extension.h>

#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <algorithm>
#include <cmath>
#include <map>
#include <mutex>
#include <utility>
#include <vector>

#include "../../include/cpu_attention_b200.h"

namespace {

std::mutex g_ws_mutex;
std::map<std::pair<int, uintptr_t>, at::Tensor> g_ws;
std::vector<at::Tensor> g_ws_outgrown;  // (sizes double: no more bytes than those in use)
constexpr int64_t kMinWorkspace = 1 << 16;

// Zeros that are there before this returns when the current stream is capturing:
// made in the graph they would be zeros only once that graph has run, and the
// next graph captured on the stream, or a call outside, may come first.
at::Tensor zeroed(int64_t device, int64_t size) {
  const auto options = at::TensorOptions().dtype(at::kByte).device(at::kCUDA, device);
  if (c10::cuda::currentStreamCaptureStatusMayInitCtx() == c10::cuda::CaptureStatus::None)
    return at::zeros({size}, options);
  const c10::cuda::CUDAStreamCaptureModeGuard relaxed(cudaStreamCaptureModeRelaxed);
  for (int tries = 0; tries < 64; ++tries) {
    const c10::cuda::CUDAStream side = c10::cuda::getStreamFromPool(false, (c10::DeviceIndex)device);
    cudaStreamCaptureStatus status;
    C10_CUDA_CHECK(cudaStreamIsCapturing(side.stream(), &status));
    if (status != cudaStreamCaptureStatusNone) continue;  // (the pool hands its streams out in turn)
    const c10::cuda::CUDAStreamGuard guard(side);
    at::Tensor ws = at::zeros({size}, options);
    C10_CUDA_CHECK(cudaStreamSynchronize(side.stream()));
    return ws;
  }
  throw std::runtime_error("cpu_attention: every stream is being captured");
}

// The workspace tensor of (device, stream), at least nbytes long, zero-filled
// when made (the decode kernel leaves its tickets and counter at zero). One that
// has been outgrown stays: a captured graph may hold its address.
at::Tensor workspace(int64_t device, uintptr_t stream, int64_t nbytes) {
  std::lock_guard<std::mutex> lock(g_ws_mutex);
  const auto key = std::make_pair((int)device, stream);
  auto it = g_ws.find(key);
  if (it != g_ws.end() && it->second.numel() >= nbytes) return it->second;
  const int64_t grown = it == g_ws.end() ? 0 : 2 * it->second.numel();
  const int64_t size = std::max({nbytes, kMinWorkspace, grown});
  at::Tensor ws = zeroed(device, size);
  if (it != g_ws.end()) g_ws_outgrown.push_back(it->second);
  g_ws[key] = ws;
  return ws;
}

// The split decode's buffer: one per (device, stream) -- calls on a stream are
// ordered, and nothing in it outlives a call -- but one of its own for every
// captured call, since graphs may be replayed side by side.
std::map<std::pair<int, uintptr_t>, at::Tensor> g_split_ws;
at::Tensor split_workspace(int64_t device, uintptr_t stream, int64_t nbytes) {
  const auto options = at::TensorOptions().dtype(at::kByte).device(at::kCUDA, device);
  if (c10::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None)
    return at::empty({nbytes}, options);
  std::lock_guard<std::mutex> lock(g_ws_mutex);
  at::Tensor& ws = g_split_ws[std::make_pair((int)device, stream)];
  if (!ws.defined() || ws.numel() < nbytes) ws = at::empty({nbytes}, options);
  return ws;
}

at::Tensor py_workspace(int64_t device, int64_t stream, int64_t nbytes) {
  return workspace(device, (uintptr_t)stream, nbytes);
}

// dtype codes of the C ABI (`_kernel.py:17`: float32 0, bfloat16 1)
int dtype_code(at::ScalarType t) {
  if (t == at::kFloat) return 0;
  if (t == at::kBFloat16) return 1;
  return -1;
}

bool head_dim_ok(int64_t hd) { return hd == 32 || hd == 64 || hd == 128; }

// heads and dims contiguous; any token stride (`_C.mojo:68-71`)
bool rows_ok(const at::Tensor& t, int64_t hd) { return t.stride(-1) == 1 && t.stride(-2) == hd; }

bool int_vector(const at::Tensor& t, at::ScalarType dt, int64_t n) {
  return t.dim() == 1 && t.scalar_type() == dt && t.size(0) == n && t.is_contiguous();
}

// lse: absent, or float32 of `shape`, contiguous, on `device`
bool lse_ok(const c10::optional<at::Tensor>& lse, at::IntArrayRef shape, const c10::Device& device) {
  if (!lse) return true;
  const at::Tensor& t = *lse;
  return t.is_cuda() && t.device() == device && t.scalar_type() == at::kFloat && t.sizes() == shape &&
         t.is_contiguous();
}

// Returns the output tensor, or None when the call is declined.
py::object decode(const at::Tensor& q, const at::Tensor& kc, const at::Tensor& vc, const c10::optional<at::Tensor>& k,
                  const c10::optional<at::Tensor>& v, const c10::optional<at::Tensor>& slots, const at::Tensor& lens,
                  const at::Tensor& pt, const c10::optional<double>& scale, const c10::optional<at::Tensor>& dst,
                  const c10::optional<at::Tensor>& lse) {
  // one CUDA device for every tensor
  if (!q.is_cuda()) return py::none();
  const auto device = q.device();
  auto same = [&](const at::Tensor& t) { return t.is_cuda() && t.device() == device; };
  if (!same(kc) || !same(vc) || !same(lens) || !same(pt)) return py::none();
  if ((k && !same(*k)) || (v && !same(*v)) || (slots && !same(*slots)) || (dst && !same(*dst))) return py::none();

  const int64_t nd = q.dim();
  if ((nd != 3 && nd != 4) || (nd == 4 && q.size(1) != 1)) return py::none();
  const int64_t b = q.size(0), heads = q.size(-2), hd = q.size(-1);
  const int dt = dtype_code(q.scalar_type());
  if (dt < 0 || !head_dim_ok(hd) || !rows_ok(q, hd)) return py::none();
  // caches: [blocks, kv_heads, page, dim], contiguous, matching, page % 16 == 0
  // (`_C.mojo:74-80`); kv_heads divides heads
  if (kc.dim() != 4 || vc.sizes() != kc.sizes()) return py::none();
  const int64_t kvh = kc.size(1);
  if (kvh < 1 || heads % kvh) return py::none();
  if (kc.scalar_type() != q.scalar_type() || vc.scalar_type() != q.scalar_type() || kc.size(3) != hd ||
      kc.size(2) <= 0 || kc.size(2) % 16 || !kc.is_contiguous() || !vc.is_contiguous())
    return py::none();
  const int64_t page = kc.size(2);
  if (pt.dim() != 2 || pt.scalar_type() != at::kInt || pt.size(0) != b || !pt.is_contiguous()) return py::none();
  if (!int_vector(lens, at::kInt, b)) return py::none();
  const bool store = k.has_value();
  int64_t n_new = 0;
  if (store) {
    const at::Tensor& kk = *k;
    if (!v || kk.dim() != nd || v->sizes() != kk.sizes() || v->strides() != kk.strides()) return py::none();
    if (kk.size(0) != b || kk.size(-2) != kvh || kk.size(-1) != hd || (nd == 4 && kk.size(1) < 1))
      return py::none();
    n_new = nd == 4 ? kk.size(1) : 1;
    if (kk.scalar_type() != q.scalar_type() || v->scalar_type() != q.scalar_type() || !rows_ok(kk, hd) ||
        (slots && n_new != 1))
      return py::none();
  } else if (v) {
    return py::none();
  }
  if (slots && !(store && int_vector(*slots, at::kLong, b))) return py::none();
  if (!lse_ok(lse, {b, heads}, device)) return py::none();
  at::Tensor out;
  if (!dst) {
    out = at::empty(q.sizes(), q.options());
  } else {
    out = *dst;
    if (out.sizes() != q.sizes() || out.scalar_type() != q.scalar_type() || !out.is_contiguous()) return py::none();
  }
  if (b == 0) return py::cast(out);

  const int dev = device.index();
  const size_t need = ca_decode_workspace_bytes(b, heads, hd, page, dt, dev);
  if (need == 0) return py::none();
  const c10::cuda::CUDAGuard guard(device);
  cudaStream_t stream = c10::cuda::getCurrentCUDAStream(dev).stream();
  at::Tensor ws = workspace(dev, (uintptr_t)stream, (int64_t)need);
  const float sc = scale ? (float)*scale : std::nanf("");
  const int rc = ca_decode_ex(q.data_ptr(), q.stride(0), kc.data_ptr(), vc.data_ptr(), kc.size(0),
                             store ? k->data_ptr() : nullptr, store ? v->data_ptr() : nullptr,
                             store ? k->stride(0) : 0, store && nd == 4 ? k->stride(1) : 0, n_new,
                             slots ? slots->data_ptr<int64_t>() : nullptr, lens.data_ptr<int32_t>(),
                             pt.data_ptr<int32_t>(), pt.size(1), out.data_ptr(),
                             lse ? lse->data_ptr<float>() : nullptr, b, heads, kvh, hd, page, dt, sc, ws.data_ptr(),
                             (size_t)ws.numel(), stream);
  if (rc == CA_ECUDA) throw std::runtime_error(std::string("cpu_attention: ") + ca_last_cuda_error());
  if (rc != CA_OK) return py::none();
  return py::cast(out);
}

// flash_attn_func over q [batch, seq, heads, dim] and k/v [batch, seq_k,
// kv_heads, dim] (kv_heads divides heads; dims contiguous): the checks of
// cpu_attention/_native.py::flash (`_C.mojo:232-316`), then ca_flash_ex.
// Returns the output, or None when declined.
py::object flash(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const c10::optional<double>& scale,
                 bool causal) {
  if (!q.is_cuda()) return py::none();
  const auto device = q.device();
  if (!k.is_cuda() || k.device() != device || !v.is_cuda() || v.device() != device) return py::none();
  if (q.dim() != 4 || k.dim() != 4 || v.dim() != 4) return py::none();
  const int64_t b = q.size(0), sq = q.size(1), heads = q.size(2), hd = q.size(3), sk = k.size(1), kvh = k.size(2);
  const int dt = dtype_code(q.scalar_type());
  if (dt < 0 || !head_dim_ok(hd) || sq < 1 || sk < 1 || kvh < 1 || heads % kvh) return py::none();
  if (k.size(0) != b || k.size(3) != hd || k.scalar_type() != q.scalar_type() || v.scalar_type() != q.scalar_type())
    return py::none();
  if (v.sizes() != k.sizes() || q.stride(3) != 1 || k.stride(3) != 1 || v.stride(3) != 1) return py::none();
  at::Tensor out = at::empty({b, sq, heads, hd}, q.options().memory_format(at::MemoryFormat::Contiguous));
  if (b == 0) return py::cast(out);
  const int dev = device.index();
  const c10::cuda::CUDAGuard guard(device);
  cudaStream_t stream = c10::cuda::getCurrentCUDAStream(dev).stream();
  at::Tensor ws = workspace(dev, (uintptr_t)stream, 0);
  const int64_t qs[3] = {q.stride(0), q.stride(1), q.stride(2)};
  const int64_t ks[3] = {k.stride(0), k.stride(1), k.stride(2)};
  const int64_t vs[3] = {v.stride(0), v.stride(1), v.stride(2)};
  const float sc = scale ? (float)*scale : std::nanf("");
  const int rc = ca_flash_ex(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), nullptr, b, sq, sk, heads, kvh,
                             hd, qs, ks, vs, nullptr, nullptr, 0, 0, sc, causal ? 1 : 0, dt,
                             static_cast<int32_t*>(ws.data_ptr()), stream);
  if (rc == CA_ECUDA) throw std::runtime_error(std::string("cpu_attention: ") + ca_last_cuda_error());
  if (rc != CA_OK) return py::none();
  return py::cast(out);
}

// reshape_and_cache: token i of key/value [tokens, heads, dim] to slot
// slots[i] (int64; negative skips it): the checks of
// cpu_attention/_native.py::store (`_C.mojo:174-213`), then ca_store. True, or
// None when declined.
py::object store(const at::Tensor& key, const at::Tensor& value, const at::Tensor& kc, const at::Tensor& vc,
                 const at::Tensor& slots) {
  if (!key.is_cuda()) return py::none();
  const auto device = key.device();
  auto same = [&](const at::Tensor& t) { return t.is_cuda() && t.device() == device; };
  if (!same(value) || !same(kc) || !same(vc) || !same(slots)) return py::none();
  if (key.dim() != 3 || value.dim() != 3) return py::none();
  const int64_t n = key.size(0), heads = key.size(1), hd = key.size(2);
  const int dt = dtype_code(key.scalar_type());
  if (dt < 0 || !head_dim_ok(hd) || value.scalar_type() != key.scalar_type() || !rows_ok(key, hd)) return py::none();
  if (value.sizes() != key.sizes() || value.strides() != key.strides()) return py::none();
  if (kc.dim() != 4 || vc.sizes() != kc.sizes() || kc.scalar_type() != key.scalar_type() ||
      vc.scalar_type() != key.scalar_type() || kc.size(1) != heads || kc.size(3) != hd || kc.size(2) <= 0 ||
      kc.size(2) % 16 || !kc.is_contiguous() || !vc.is_contiguous())
    return py::none();
  if (!int_vector(slots, at::kLong, n)) return py::none();
  if (n == 0) return py::bool_(true);
  const int dev = device.index();
  const c10::cuda::CUDAGuard guard(device);
  cudaStream_t stream = c10::cuda::getCurrentCUDAStream(dev).stream();
  at::Tensor ws = workspace(dev, (uintptr_t)stream, 0);
  const int rc = ca_store(key.data_ptr(), value.data_ptr(), key.stride(0), kc.data_ptr(), vc.data_ptr(), kc.size(0),
                          slots.data_ptr<int64_t>(), n, heads, hd, kc.size(2), dt,
                          static_cast<int32_t*>(ws.data_ptr()), stream);
  if (rc == CA_ECUDA) throw std::runtime_error(std::string("cpu_attention: ") + ca_last_cuda_error());
  if (rc != CA_OK) return py::none();
  return py::bool_(true);
}

// ---- caches in 8 bits, windows, block moves ---------------------------------
// (the checks of cpu_attention/_native.py's functions of the same names)

// k_cache/v_cache [blocks, kv_heads, page, hd] of type `dt`, contiguous
bool caches_ok(const at::Tensor& kc, const at::Tensor& vc, at::ScalarType dt, int64_t hd) {
  return kc.dim() == 4 && vc.sizes() == kc.sizes() && kc.scalar_type() == dt && vc.scalar_type() == dt &&
         kc.size(1) >= 1 && kc.size(3) == hd && kc.size(2) > 0 && kc.size(2) % 16 == 0 && kc.is_contiguous() &&
         vc.is_contiguous();
}

// the scales of 8-bit caches: float32 [blocks, kv_heads], contiguous
bool scales_ok(const at::Tensor& t, const at::Tensor& kc) {
  return t.scalar_type() == at::kFloat && t.dim() == 2 && t.size(0) == kc.size(0) && t.size(1) == kc.size(1) &&
         t.is_contiguous();
}

py::object decode_split(const at::Tensor& q, const at::Tensor& kc, const at::Tensor& vc,
                        const c10::optional<at::Tensor>& k, const c10::optional<at::Tensor>& v,
                        const c10::optional<at::Tensor>& ks, const c10::optional<at::Tensor>& vs,
                        const at::Tensor& lens, const at::Tensor& pt, int64_t left, int64_t sinks,
                        const c10::optional<double>& scale, const c10::optional<at::Tensor>& lse) {
  if (!q.is_cuda()) return py::none();
  const auto device = q.device();
  auto same = [&](const at::Tensor& t) { return t.is_cuda() && t.device() == device; };
  if (!same(kc) || !same(vc) || !same(lens) || !same(pt)) return py::none();
  if ((k && !same(*k)) || (v && !same(*v)) || (ks && !same(*ks)) || (vs && !same(*vs))) return py::none();
  if (q.dim() != 4 || q.size(1) != 1) return py::none();
  const int64_t b = q.size(0), heads = q.size(2), hd = q.size(3);
  const int dt = dtype_code(q.scalar_type());
  if (dt < 0 || !head_dim_ok(hd) || !rows_ok(q, hd) || kc.dim() != 4) return py::none();
  const bool eight = kc.scalar_type() == at::kFloat8_e4m3fn;
  if (!caches_ok(kc, vc, eight ? at::kFloat8_e4m3fn : q.scalar_type(), hd)) return py::none();
  const int64_t kvh = kc.size(1), page = kc.size(2);
  if (heads < 1 || heads % kvh || eight != ks.has_value() || eight != vs.has_value()) return py::none();
  if (eight && (!scales_ok(*ks, kc) || !scales_ok(*vs, kc))) return py::none();
  if (pt.dim() != 2 || pt.scalar_type() != at::kInt || pt.size(0) != b || !pt.is_contiguous()) return py::none();
  if (!int_vector(lens, at::kInt, b) || !lse_ok(lse, {b, heads}, device)) return py::none();
  if (k.has_value() != v.has_value() || left < -1 || sinks < 0) return py::none();
  int64_t n_new = 0;
  if (k) {
    if (k->dim() != 4 || v->sizes() != k->sizes() || v->strides() != k->strides() || k->size(0) != b ||
        k->size(2) != kvh || k->size(3) != hd || k->scalar_type() != q.scalar_type() ||
        v->scalar_type() != q.scalar_type() || !rows_ok(*k, hd))
      return py::none();
    n_new = k->size(1);
  }
  at::Tensor out = at::empty(q.sizes(), q.options().memory_format(at::MemoryFormat::Contiguous));
  if (b == 0) return py::cast(out);
  const int dev = device.index();
  const c10::cuda::CUDAGuard guard(device);
  cudaStream_t stream = c10::cuda::getCurrentCUDAStream(dev).stream();
  const size_t need = ca_decode_split_workspace_bytes(hd, dev);
  at::Tensor scratch = split_workspace(dev, (uintptr_t)stream, (int64_t)need);
  at::Tensor ws = workspace(dev, (uintptr_t)stream, 0);
  const bool fresh = n_new > 0;
  const int rc = ca_decode_split(
      q.data_ptr(), q.stride(0), kc.data_ptr(), vc.data_ptr(), eight ? ks->data_ptr<float>() : nullptr,
      eight ? vs->data_ptr<float>() : nullptr, kc.size(0), fresh ? k->data_ptr() : nullptr,
      fresh ? v->data_ptr() : nullptr, fresh ? k->stride(0) : 0, fresh ? k->stride(1) : 0, n_new,
      lens.data_ptr<int32_t>(), pt.data_ptr<int32_t>(), pt.size(1), out.data_ptr(),
      lse ? lse->data_ptr<float>() : nullptr, b, heads, kvh, hd, page, dt, eight ? CA_DTYPE_E4M3 : dt, left, sinks,
      scale ? (float)*scale : std::nanf(""), scratch.data_ptr(), (size_t)scratch.numel(),
      static_cast<int32_t*>(ws.data_ptr()), stream);
  if (rc == CA_ECUDA) throw std::runtime_error(std::string("cpu_attention: ") + ca_last_cuda_error());
  if (rc != CA_OK) return py::none();
  return py::cast(out);
}

py::object append_8bit(const at::Tensor& key, const at::Tensor& value, const at::Tensor& kc, const at::Tensor& vc,
                       const at::Tensor& ks, const at::Tensor& vs, const at::Tensor& lens, const at::Tensor& pt,
                       const c10::optional<at::Tensor>& cu, int64_t max_new) {
  if (!key.is_cuda()) return py::none();
  const auto device = key.device();
  auto same = [&](const at::Tensor& t) { return t.is_cuda() && t.device() == device; };
  if (!same(value) || !same(kc) || !same(vc) || !same(ks) || !same(vs) || !same(lens) || !same(pt) ||
      (cu && !same(*cu)))
    return py::none();
  if (key.dim() != (cu ? 3 : 4) || value.sizes() != key.sizes() || value.strides() != key.strides()) return py::none();
  const int64_t heads = key.size(-2), hd = key.size(-1);
  const int dt = dtype_code(key.scalar_type());
  if (dt < 0 || value.scalar_type() != key.scalar_type() || !head_dim_ok(hd) || !rows_ok(key, hd)) return py::none();
  if (!caches_ok(kc, vc, at::kFloat8_e4m3fn, hd) || kc.size(1) != heads || !scales_ok(ks, kc) || !scales_ok(vs, kc))
    return py::none();
  if (lens.dim() != 1) return py::none();
  const int64_t b = lens.size(0);
  if (!int_vector(lens, at::kInt, b) || pt.dim() != 2 || pt.scalar_type() != at::kInt || pt.size(0) != b ||
      !pt.is_contiguous())
    return py::none();
  if (cu ? !int_vector(*cu, at::kInt, b + 1) || max_new < 0 : key.size(0) != b) return py::none();
  const int dev = device.index();
  const c10::cuda::CUDAGuard guard(device);
  cudaStream_t stream = c10::cuda::getCurrentCUDAStream(dev).stream();
  at::Tensor ws = workspace(dev, (uintptr_t)stream, 0);
  const int rc = ca_append_8bit(
      key.data_ptr(), value.data_ptr(), cu ? 0 : key.stride(0), cu ? key.stride(0) : key.stride(1),
      cu ? max_new : key.size(1), cu ? cu->data_ptr<int32_t>() : nullptr, cu ? key.size(0) : 0, kc.data_ptr(),
      vc.data_ptr(), ks.data_ptr<float>(), vs.data_ptr<float>(), kc.size(0), lens.data_ptr<int32_t>(),
      pt.data_ptr<int32_t>(), pt.size(1), b, heads, hd, kc.size(2), dt, static_cast<int32_t*>(ws.data_ptr()), stream);
  if (rc == CA_ECUDA) throw std::runtime_error(std::string("cpu_attention: ") + ca_last_cuda_error());
  if (rc != CA_OK) return py::none();
  return py::bool_(true);
}

// Prefill behind a window (flash_attn_func's and flash_attn_varlen_func's).
py::object flash_window(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                        const c10::optional<double>& scale, bool causal, int64_t left, int64_t right, int64_t sinks,
                        const c10::optional<at::Tensor>& lse, const c10::optional<at::Tensor>& cu_q,
                        const c10::optional<at::Tensor>& cu_k, int64_t max_q, int64_t max_k) {
  if (!q.is_cuda()) return py::none();
  const auto device = q.device();
  auto same = [&](const at::Tensor& t) { return t.is_cuda() && t.device() == device; };
  const bool var = cu_q.has_value();
  if (!same(k) || !same(v) || cu_k.has_value() != var || (var && (!same(*cu_q) || !same(*cu_k)))) return py::none();
  const int64_t nd = var ? 3 : 4;
  if (q.dim() != nd || k.dim() != nd || v.sizes() != k.sizes()) return py::none();
  const int64_t heads = q.size(-2), hd = q.size(-1), kvh = k.size(-2);
  const int dt = dtype_code(q.scalar_type());
  if (dt < 0 || !head_dim_ok(hd) || kvh < 1 || heads % kvh || k.size(-1) != hd) return py::none();
  if (k.scalar_type() != q.scalar_type() || v.scalar_type() != q.scalar_type()) return py::none();
  if (q.stride(-1) != 1 || k.stride(-1) != 1 || v.stride(-1) != 1) return py::none();
  if (left < -1 || right < -1 || sinks < 0) return py::none();
  int64_t b, sq, sk;
  if (var) {
    b = cu_q->numel() - 1;
    if (b < 0 || !int_vector(*cu_q, at::kInt, b + 1) || !int_vector(*cu_k, at::kInt, b + 1)) return py::none();
    sq = max_q;
    sk = max_k;
  } else {
    b = q.size(0);
    sq = q.size(1);
    sk = k.size(1);
    if (k.size(0) != b) return py::none();
  }
  if (sq < 1 || sk < 1) return py::none();
  if (var ? !lse_ok(lse, {heads, q.size(0)}, device) : !lse_ok(lse, {b, heads, sq}, device)) return py::none();
  at::Tensor out = at::empty(q.sizes(), q.options().memory_format(at::MemoryFormat::Contiguous));
  if (b == 0 || q.numel() == 0) return py::cast(out);
  const int dev = device.index();
  const c10::cuda::CUDAGuard guard(device);
  cudaStream_t stream = c10::cuda::getCurrentCUDAStream(dev).stream();
  at::Tensor ws = workspace(dev, (uintptr_t)stream, 0);
  int64_t st[3][3];
  const at::Tensor* ts[3] = {&q, &k, &v};
  for (int x = 0; x < 3; ++x) {
    st[x][0] = var ? 0 : ts[x]->stride(0);
    st[x][1] = ts[x]->stride(-3);
    st[x][2] = ts[x]->stride(-2);
  }
  const int rc = ca_flash_window(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(),
                                 lse ? lse->data_ptr<float>() : nullptr, b, sq, sk, heads, kvh, hd, st[0], st[1],
                                 st[2], var ? cu_q->data_ptr<int32_t>() : nullptr,
                                 var ? cu_k->data_ptr<int32_t>() : nullptr, var ? q.size(0) : 0, var ? k.size(0) : 0,
                                 scale ? (float)*scale : std::nanf(""), causal ? 1 : 0, left, right, sinks, dt,
                                 static_cast<int32_t*>(ws.data_ptr()), stream);
  if (rc == CA_ECUDA) throw std::runtime_error(std::string("cpu_attention: ") + ca_last_cuda_error());
  if (rc != CA_OK) return py::none();
  return py::cast(out);
}

// The caches of a block move: contiguous tensors [num_blocks, ...] on one
// device. Their bases and block sizes; false when one is not.
bool block_tensors(const std::vector<at::Tensor>& caches, const c10::Device& device, std::vector<void*>* base,
                   std::vector<int64_t>* bytes, int64_t* blocks) {
  *blocks = 0;
  for (const at::Tensor& t : caches) {
    if (!t.is_cuda() || t.device() != device || t.dim() < 1 || !t.is_contiguous()) return false;
    if (base->empty() && bytes->empty() && &t == &caches[0]) *blocks = t.size(0);
    if (t.size(0) != *blocks) return false;
    if (t.numel() == 0) continue;  // nothing to move
    base->push_back(t.data_ptr());
    bytes->push_back((int64_t)t.nbytes() / t.size(0));
  }
  return true;
}

py::object copy_blocks(const std::vector<at::Tensor>& caches, const at::Tensor& pairs) {
  if (!pairs.is_cuda() || pairs.scalar_type() != at::kLong || pairs.dim() != 2 || pairs.size(1) != 2 ||
      !pairs.is_contiguous())
    return py::none();
  const auto device = pairs.device();
  std::vector<void*> base;
  std::vector<int64_t> bytes;
  int64_t blocks;
  if (!block_tensors(caches, device, &base, &bytes, &blocks)) return py::none();
  const int dev = device.index();
  const c10::cuda::CUDAGuard guard(device);
  cudaStream_t stream = c10::cuda::getCurrentCUDAStream(dev).stream();
  at::Tensor ws = workspace(dev, (uintptr_t)stream, 0);
  const int rc = ca_copy_blocks(base.data(), bytes.data(), (int64_t)base.size(), blocks, pairs.data_ptr<int64_t>(),
                                pairs.size(0), static_cast<int32_t*>(ws.data_ptr()), stream);
  if (rc == CA_ECUDA) throw std::runtime_error(std::string("cpu_attention: ") + ca_last_cuda_error());
  if (rc != CA_OK) return py::none();
  return py::bool_(true);
}

py::object compact_blocks(const std::vector<at::Tensor>& caches, const at::Tensor& pt, const at::Tensor& lens,
                          int64_t page, int64_t left, int64_t sinks, const c10::optional<at::Tensor>& reserved) {
  if (!pt.is_cuda() || caches.empty()) return py::none();
  const auto device = pt.device();
  if (pt.dim() != 2 || pt.scalar_type() != at::kInt || !pt.is_contiguous() || !lens.is_cuda() ||
      lens.device() != device || !int_vector(lens, at::kInt, pt.size(0)))
    return py::none();
  if (reserved && (!reserved->is_cuda() || reserved->device() != device || !int_vector(*reserved, at::kInt, pt.size(0))))
    return py::none();
  std::vector<void*> base;
  std::vector<int64_t> bytes;
  int64_t blocks;
  if (!block_tensors(caches, device, &base, &bytes, &blocks)) return py::none();
  const int dev = device.index();
  const c10::cuda::CUDAGuard guard(device);
  cudaStream_t stream = c10::cuda::getCurrentCUDAStream(dev).stream();
  at::Tensor ws = workspace(dev, (uintptr_t)stream, 0);
  at::Tensor table = at::empty(pt.sizes(), pt.options()), used = at::empty({1}, pt.options());
  const size_t need = ca_compact_workspace_bytes(blocks);
  at::Tensor scratch = at::empty({(int64_t)need}, pt.options().dtype(at::kByte));
  const int rc = ca_compact_blocks_ex(
      base.data(), bytes.data(), (int64_t)base.size(), blocks, pt.data_ptr<int32_t>(), lens.data_ptr<int32_t>(),
      reserved ? reserved->data_ptr<int32_t>() : nullptr, pt.size(0), pt.size(1), page, left, sinks,
      table.data_ptr<int32_t>(), used.data_ptr<int32_t>(), scratch.data_ptr(), need,
      static_cast<int32_t*>(ws.data_ptr()), stream);
  if (rc == CA_ECUDA) throw std::runtime_error(std::string("cpu_attention: ") + ca_last_cuda_error());
  if (rc != CA_OK) return py::none();
  return py::make_tuple(table, used);
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.doc() = "cpu_attention's decode host path in C++ (argument checks and the C ABI call)";
  m.def("decode", &decode, "paged decode; the output tensor, or None when declined", py::arg("q"), py::arg("k_cache"),
        py::arg("v_cache"), py::arg("k"), py::arg("v"), py::arg("slots"), py::arg("lens"), py::arg("page_table"),
        py::arg("scale"), py::arg("dst"), py::arg("lse") = py::none());
  m.def("flash", &flash, "dense prefill; the output tensor, or None when declined", py::arg("q"), py::arg("k"),
        py::arg("v"), py::arg("scale"), py::arg("causal"));
  m.def("store", &store, "reshape_and_cache; True, or None when declined", py::arg("key"), py::arg("value"),
        py::arg("k_cache"), py::arg("v_cache"), py::arg("slots"));
  m.def("decode_split", &decode_split, "decode over 8-bit caches or behind a window; the output, or None", py::arg("q"),
        py::arg("k_cache"), py::arg("v_cache"), py::arg("k"), py::arg("v"), py::arg("k_scale"), py::arg("v_scale"),
        py::arg("lens"), py::arg("page_table"), py::arg("left"), py::arg("sinks"), py::arg("scale"), py::arg("lse"));
  m.def("append_8bit", &append_8bit, "new tokens into 8-bit caches; True, or None when declined", py::arg("key"),
        py::arg("value"), py::arg("k_cache"), py::arg("v_cache"), py::arg("k_scale"), py::arg("v_scale"),
        py::arg("lens"), py::arg("page_table"), py::arg("cu"), py::arg("max_new"));
  m.def("flash_window", &flash_window, "prefill behind a window; the output, or None when declined", py::arg("q"),
        py::arg("k"), py::arg("v"), py::arg("scale"), py::arg("causal"), py::arg("left"), py::arg("right"),
        py::arg("sinks"), py::arg("lse"), py::arg("cu_q"), py::arg("cu_k"), py::arg("max_q"), py::arg("max_k"));
  m.def("copy_blocks", &copy_blocks, "block copies; True, or None when declined", py::arg("caches"), py::arg("pairs"));
  m.def("compact_blocks", &compact_blocks, "pack the blocks in use; (table, used), or None when declined",
        py::arg("caches"), py::arg("page_table"), py::arg("lens"), py::arg("page"), py::arg("left"), py::arg("sinks"),
        py::arg("reserved") = py::none());
  m.def("workspace", &py_workspace, "the workspace tensor of (device, stream), at least nbytes long",
        py::arg("device"), py::arg("stream"), py::arg("nbytes"));
}
