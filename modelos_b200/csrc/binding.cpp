// The attention entry points as a Python module with their autograd node.
//
// Single tokens and small batches are bound by the host: a call through ctypes
// with its checks in Python took 16 us and a training step's two calls 150,
// for kernels of 2 to 10 us.  The module checks its arguments, allocates the
// outputs with torch's allocator and calls the C ABI on the current stream.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/extension.h>

#include "pkm_b200.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::tensor_list;
using OptTensor = std::optional<Tensor>;

#define REFUSE(ok, what) TORCH_CHECK_VALUE(ok, "modelos_b200 attention: " what)

int dtype_of(const Tensor& t) { return t.scalar_type() == at::kBFloat16 ? PKM_DT_BF16 : PKM_DT_F16; }
bool half_type(const Tensor& t) { return t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kHalf; }

void need_cuda(const Tensor& t) {
  TORCH_CHECK(t.is_cuda(), "modelos_b200 kernels need CUDA tensors (there is no CPU path)");
}

// A tensor with a forward-mode tangent, which the kernels would drop.
void no_dual(const Tensor& t) {
  TORCH_CHECK(!t.unsafeGetTensorImpl()->_fw_grad(0, t).defined(),
              "modelos_b200 attention: forward-mode derivatives are not implemented");
}

void check(int rc, const char* name) {
  TORCH_CHECK(rc == PKM_OK, name, " failed (", pkm_status_string(rc), "): ", pkm_last_error());
}

// The device's error word (modelos_b200._native.err_word keeps the tensor).
uint32_t* err_word(const Tensor& t) {
  static std::atomic<uint32_t*> words[64];
  const int dev = t.get_device();
  if (dev >= 64) return nullptr;
  uint32_t* w = words[dev].load(std::memory_order_acquire);
  if (!w) {
    py::gil_scoped_acquire gil;
    const Tensor word =
        py::module_::import("modelos_b200._native").attr("err_word")(py::cast(t.device())).cast<Tensor>();
    w = reinterpret_cast<uint32_t*>(word.data_ptr());
    words[dev].store(w, std::memory_order_release);
  }
  return w;
}

void* stream_of(const Tensor& t) { return at::cuda::getCurrentCUDAStream(t.get_device()).stream(); }
const int32_t* ints(const OptTensor& t) { return t ? t->const_data_ptr<int32_t>() : nullptr; }

// `t` itself if the kernels read it in place (unit channel stride, 16-byte
// aligned base and strides, no broadcast dimension), else a copy.
Tensor operand(const Tensor& t) {
  bool ok = t.stride(3) == 1 && reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 == 0;
  for (int i = 0; i < 3; ++i) ok = ok && (t.size(i) <= 1 || (t.stride(i) % 8 == 0 && t.stride(i) > 0));
  return ok ? t : t.clone(at::MemoryFormat::Contiguous);
}

OptTensor bounds(const OptTensor& t, int64_t B, const Tensor& like, const char* name) {
  if (!t) return t;
  const at::ScalarType type = t->scalar_type();
  TORCH_CHECK_VALUE(t->dim() == 1 && t->size(0) == B &&
                        (type == at::kInt || type == at::kLong || type == at::kShort || type == at::kChar ||
                         type == at::kByte),
                    "modelos_b200 attention: ", name, " must be integers [batch]");
  TORCH_CHECK_VALUE(t->device() == like.device(), "modelos_b200 attention: ", name,
                    " must be on the operands' device");
  // (64-bit numbers past 32 bits stay past every row)
  const Tensor in = t->scalar_type() == at::kLong ? t->clamp(INT32_MIN, INT32_MAX) : *t;
  return in.to(at::kInt).contiguous();
}

Tensor forward(const Tensor& q, const Tensor& k, const Tensor& v, double scale, int64_t window, int64_t sinks,
               const OptTensor& starts, const OptTensor& ends, Tensor* lse, Tensor* lo) {
  const c10::cuda::CUDAGuard guard(q.device());
  Tensor out = at::empty_like(q);
  if (lo) *lo = at::empty_like(out);
  if (lse) *lse = at::empty({q.size(0), q.size(1), q.size(2)}, q.options().dtype(at::kFloat));
  size_t bytes = 0;
  check(pkm_attn_fwd_workspace(q.size(0), q.size(1), k.size(1), q.size(2), k.size(2), q.size(3), window, sinks, &bytes),
        "pkm_attn_fwd_workspace");
  const Tensor ws = bytes ? at::empty({(int64_t)bytes}, q.options().dtype(at::kByte)) : Tensor();
  check(pkm_attn_fwd(q.const_data_ptr(), q.strides().data(), k.const_data_ptr(), k.strides().data(), v.const_data_ptr(),
                     v.strides().data(), dtype_of(q), q.size(0), q.size(1), k.size(1), q.size(2), k.size(2), q.size(3),
                     scale, window, sinks, ints(starts), ints(ends), out.data_ptr(), out.strides().data(),
                     lo ? lo->data_ptr() : nullptr, lse ? lse->data_ptr<float>() : nullptr,
                     bytes ? ws.data_ptr() : nullptr, bytes, err_word(q), stream_of(q)),
        "pkm_attn_fwd");
  return out;
}

struct WindowAttention : torch::autograd::Function<WindowAttention> {
  static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, double scale,
                        int64_t window, int64_t sinks, const OptTensor& starts, const OptTensor& ends) {
    Tensor lse, lo;
    Tensor out = ::forward(q, k, v, scale, window, sinks, starts, ends, &lse, &lo);
    ctx->save_for_backward({q, k, v, out, lo, lse, starts ? *starts : Tensor(), ends ? *ends : Tensor()});
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["window"] = window;
    ctx->saved_data["sinks"] = sinks;
    return out;
  }
  static tensor_list backward(AutogradContext* ctx, tensor_list grads) {
    const tensor_list s = ctx->get_saved_variables();
    tensor_list d(3);
    {
      const at::AutoGradMode off(false);
      const Tensor &q = s[0], &k = s[1], &v = s[2], &out = s[3], &lo = s[4], &lse = s[5];
      const c10::cuda::CUDAGuard guard(q.device());
      const Tensor dout = operand(grads[0]);
      for (int i = 0; i < 3; ++i) d[i] = at::empty_like(s[i]);
      size_t bytes = 0;
      check(pkm_attn_bwd_workspace(q.size(0), q.size(1), k.size(1), q.size(2), k.size(2), q.size(3),
                                   ctx->saved_data["window"].toInt(), ctx->saved_data["sinks"].toInt(), &bytes),
            "pkm_attn_bwd_workspace");
      const Tensor ws = at::empty({(int64_t)bytes}, q.options().dtype(at::kByte));
      check(pkm_attn_bwd(q.const_data_ptr(), q.strides().data(), k.const_data_ptr(), k.strides().data(),
                         v.const_data_ptr(), v.strides().data(), out.const_data_ptr(), out.strides().data(),
                         lo.const_data_ptr(), dout.const_data_ptr(), dout.strides().data(), lse.const_data_ptr<float>(), dtype_of(q),
                         q.size(0), q.size(1), k.size(1), q.size(2), k.size(2), q.size(3),
                         ctx->saved_data["scale"].toDouble(), ctx->saved_data["window"].toInt(),
                         ctx->saved_data["sinks"].toInt(), s[6].defined() ? s[6].const_data_ptr<int32_t>() : nullptr,
                         s[7].defined() ? s[7].const_data_ptr<int32_t>() : nullptr, d[0].data_ptr(),
                         d[0].strides().data(), d[1].data_ptr(), d[1].strides().data(), d[2].data_ptr(),
                         d[2].strides().data(), ws.data_ptr(), bytes, err_word(q), stream_of(q)),
            "pkm_attn_bwd");
    }
    if (at::GradMode::is_enabled()) {
      // under create_graph: what differentiates these gradients again has to fail
      for (auto& x : d) x.requires_grad_();
      const auto fail = std::make_shared<torch::autograd::DelayedError>(
          "modelos_b200 attention: window_attention is differentiable once", 3);
      d = (*fail)(tensor_list(d));
    }
    d.resize(8);
    return d;
  }
};

// A leaf's gradient is accumulated on the stream of the oldest graph that holds
// the leaf.  If that is the legacy default stream (an eager graph is alive), a
// captured backward pass would make that stream wait for a captured one, which
// CUDA answers by ending the capture and the autograd thread the process.
void check_capture(const Tensor& t) {
  if (!t.requires_grad() || !t.is_leaf()) return;
  const auto acc = torch::autograd::impl::try_get_grad_accumulator(t);
  if (!acc) return;
  const auto s = acc->stream();
  TORCH_CHECK(!s || c10::cuda::CUDAStream(*s).stream() != nullptr,
              "modelos_b200 attention: an eager graph of the default stream holds these leaves: release it before "
              "capturing their backward pass");
}

Tensor window_attention(const Tensor& q0, const Tensor& k0, const Tensor& v0, int64_t window, int64_t sinks,
                        std::optional<double> scale, const OptTensor& starts, const OptTensor& ends) {
  REFUSE(q0.dim() == 4 && k0.dim() == 4 && v0.dim() == 4, "q, k and v must be [batch, heads, tokens, head_dim]");
  REFUSE(k0.sizes() == v0.sizes(), "k and v must have one shape");
  const int64_t B = q0.size(0), Hq = q0.size(1), D = q0.size(3), Hk = k0.size(1);
  REFUSE(k0.size(0) == B && k0.size(3) == D, "q and k disagree in batch or head_dim");
  REFUSE(q0.scalar_type() == k0.scalar_type() && q0.scalar_type() == v0.scalar_type(), "q, k and v must share a type");
  REFUSE(half_type(q0), "only bf16 and fp16 are implemented");
  for (const Tensor* t : {&q0, &k0, &v0}) no_dual(*t);
  need_cuda(q0);
  need_cuda(k0);
  need_cuda(v0);
  REFUSE(q0.device() == k0.device() && q0.device() == v0.device(), "q, k and v must be on one device");
  REFUSE(D > 0 && D <= 128 && D % 8 == 0, "head_dim must be a multiple of 8 and at most 128");
  REFUSE(Hk > 0 && Hq > 0 && Hq % Hk == 0, "heads must be a multiple of kv_heads");
  REFUSE(k0.size(2) >= q0.size(2), "fewer keys than queries");
  REFUSE(window >= 0 && sinks >= 0, "window and sinks must not be negative");
  const OptTensor s = bounds(starts, B, q0, "starts"), e = bounds(ends, B, q0, "ends");
  const double c = scale ? *scale : 1.0 / std::sqrt((double)D);
  const Tensor q = operand(q0), k = operand(k0), v = operand(v0);
  if (at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || v.requires_grad())) {
    cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
    const cudaStream_t st = at::cuda::getCurrentCUDAStream(q.get_device()).stream();
    if (st) C10_CUDA_CHECK(cudaStreamIsCapturing(st, &capture));  // (the legacy stream cannot be captured)
    if (capture != cudaStreamCaptureStatusNone)
      for (const Tensor* t : {&q0, &k0, &v0}) check_capture(*t);
    return WindowAttention::apply(q, k, v, c, window, sinks, s, e);
  }
  return forward(q, k, v, c, window, sinks, s, e, nullptr, nullptr);
}

// ---------------------------------------------------------------------------
// the 4-bit cache: codes [B, Hk, cap, D/2], params [B, Hk, cap, D/32, 2]
// ---------------------------------------------------------------------------
// The cache's tensors are attributes that a caller can replace.
void check_cache(const Tensor& kc, const Tensor& kp, const Tensor& vc, const Tensor& vp) {
  bool ok = kc.dim() == 4 && kc.scalar_type() == at::kByte && (kc.size(3) == 32 || kc.size(3) == 64) &&
            vc.scalar_type() == at::kByte && vc.sizes() == kc.sizes() && kp.dim() == 5 && half_type(kp) &&
            vp.scalar_type() == kp.scalar_type() && vp.sizes() == kp.sizes();
  for (int i = 0; i < 3; ++i) ok = ok && kp.size(i) == kc.size(i);
  ok = ok && kp.size(3) == kc.size(3) / 16 && kp.size(4) == 2;
  for (const Tensor* t : {&kc, &kp, &vc, &vp}) ok = ok && t->is_contiguous() && t->device() == kc.device();
  REFUSE(ok, "the cache's codes and params do not fit together");
}

// Row numbers: a tensor [batch], or one number for all (-1: there is a tensor).
void check_rows(int64_t at0, const OptTensor& at, int64_t n, int64_t cap) {
  REFUSE(at || (at0 >= 0 && at0 <= cap - n), "rows outside the cache");
}

void kv4_write(const Tensor& k0, const Tensor& v0, const OptTensor& at, int64_t at0, const Tensor& kc, const Tensor& kp,
               const Tensor& vc, const Tensor& vp) {
  check_cache(kc, kp, vc, vp);
  const int64_t B = kc.size(0), Hk = kc.size(1), cap = kc.size(2), D = 2 * kc.size(3);
  REFUSE(k0.dim() == 4 && k0.sizes() == v0.sizes(), "k and v must be [batch, kv_heads, tokens, head_dim] of one shape");
  REFUSE(k0.size(0) == B && k0.size(1) == Hk && k0.size(3) == D, "k does not fit the cache");
  REFUSE(k0.scalar_type() == kp.scalar_type() && v0.scalar_type() == kp.scalar_type(),
         "k and v must have the cache's type");
  no_dual(k0);
  no_dual(v0);
  need_cuda(k0);
  need_cuda(v0);
  REFUSE(k0.device() == kc.device() && v0.device() == kc.device(), "k and v must be on the cache's device");
  check_rows(at0, at, k0.size(2), cap);
  const OptTensor rows = bounds(at, B, kc, "row numbers");
  const at::AutoGradMode off(false);
  const c10::cuda::CUDAGuard guard(kc.device());
  const Tensor k = operand(k0), v = operand(v0);
  check(pkm_kv4_write(k.const_data_ptr(), k.strides().data(), v.const_data_ptr(), v.strides().data(), dtype_of(k), B, Hk,
                      k.size(2), cap, D, ints(rows), at0, kc.data_ptr(), kp.data_ptr(), vc.data_ptr(), vp.data_ptr(),
                      err_word(kc), stream_of(kc)),
        "pkm_kv4_write");
}

std::tuple<Tensor, Tensor> kv4_read(const Tensor& kc, const Tensor& kp, const Tensor& vc, const Tensor& vp,
                                    const OptTensor& at, int64_t at0, int64_t n) {
  check_cache(kc, kp, vc, vp);
  const int64_t B = kc.size(0), Hk = kc.size(1), cap = kc.size(2), D = 2 * kc.size(3);
  REFUSE(n >= 0, "count must not be negative");
  need_cuda(kc);
  check_rows(at0, at, n, cap);
  const OptTensor rows = bounds(at, B, kc, "row numbers");
  const c10::cuda::CUDAGuard guard(kc.device());
  Tensor k = at::empty({B, Hk, n, D}, kp.options()), v = at::empty({B, Hk, n, D}, kp.options());
  check(pkm_kv4_read(kc.const_data_ptr(), kp.const_data_ptr(), vc.const_data_ptr(), vp.const_data_ptr(), dtype_of(kp),
                     B, Hk, n, cap, D, ints(rows), at0, k.data_ptr(), v.data_ptr(), err_word(kc), stream_of(kc)),
        "pkm_kv4_read");
  return {k, v};
}

Tensor kv4_attend(const Tensor& q0, const Tensor& kc, const Tensor& kp, const Tensor& vc, const Tensor& vp,
                  int64_t window, int64_t sinks, std::optional<double> scale, const OptTensor& starts,
                  const Tensor& lengths) {
  check_cache(kc, kp, vc, vp);
  const int64_t B = kc.size(0), Hk = kc.size(1), cap = kc.size(2), D = 2 * kc.size(3);
  REFUSE(lengths.dim() == 1 && lengths.size(0) == B && lengths.scalar_type() == at::kInt && lengths.is_contiguous() &&
             lengths.device() == kc.device(),
         "lengths must be int32 [batch] on the cache's device");
  REFUSE(q0.dim() == 4 && q0.size(0) == B && q0.size(3) == D, "q does not fit the cache");
  REFUSE(q0.scalar_type() == kp.scalar_type(), "q must have the cache's type");
  no_dual(q0);
  need_cuda(q0);
  REFUSE(q0.device() == kc.device(), "q must be on the cache's device");
  REFUSE(Hk > 0 && q0.size(1) % Hk == 0, "heads must be a multiple of kv_heads");
  REFUSE(q0.size(2) * (q0.size(1) / Hk) <= PKM_KV4_MAX_ROWS,
         "more than 64 query rows (tokens x grouped heads) to a KV head");
  REFUSE(window >= 0 && sinks >= 0, "window and sinks must not be negative");
  const OptTensor s = bounds(starts, B, kc, "starts");
  const at::AutoGradMode off(false);
  const c10::cuda::CUDAGuard guard(kc.device());
  const Tensor q = operand(q0);
  Tensor out = at::empty_like(q);
  check(pkm_kv4_attend(q.const_data_ptr(), q.strides().data(), kc.const_data_ptr(), kp.const_data_ptr(),
                       vc.const_data_ptr(), vp.const_data_ptr(), dtype_of(q), B, q.size(1), Hk, q.size(2), cap, D,
                       scale ? *scale : 1.0 / std::sqrt((double)D), window, sinks, ints(s),
                       lengths.const_data_ptr<int32_t>(), out.data_ptr(), out.strides().data(), err_word(kc),
                       stream_of(kc)),
        "pkm_kv4_attend");
  return out;
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("window_attention", &window_attention);
  m.def("kv4_write", &kv4_write);
  m.def("kv4_read", &kv4_read);
  m.def("kv4_attend", &kv4_attend);
}
