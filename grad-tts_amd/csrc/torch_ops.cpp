// PyTorch custom-op registration of the C ABI (include/gradtts.h): torch.ops.gradtts.*
//
//   gradtts::reverse_diffusion(int decoder, int dtype, Tensor z, Tensor mask, Tensor mu, int n_timesteps,
//                              Tensor? spk) -> Tensor          Diffusion.reverse_diffusion, model/diffusion.py:254-268
//   gradtts::estimator(int decoder, int dtype, Tensor x, Tensor mask, Tensor mu, Tensor t, Tensor? spk) -> Tensor
//                                                             GradLogPEstimator2d.forward, model/diffusion.py:174-216
//   gradtts::maximum_path(Tensor value, Tensor mask) -> Tensor monotonic_align.maximum_path, __init__.py:8-23
//   gradtts::bucket_attention / bucket_attention_backward, gradtts::residual_norm / residual_norm_backward
//                                                             operators of transformer blocks (gradtts_amd.attention, .norm)
//   gradtts::bind(str library_path) -> ()                     resolve the C ABI (once per process)
//
// `decoder` is the gt_decoder* of the module that owns the weights (gradtts_amd.diffusion keeps it and syncs the
// parameters before the call); `dtype` is GT_F32 / GT_BF16 / GT_BF16_W8. The HIP (dispatch key CUDA) kernels
// run on the current HIP stream with workspace from PyTorch's caching allocator on that stream; the Meta kernels
// give shapes and dtypes to torch.compile's fake tensors. Errors raise (TORCH_CHECK) with gt_last_error().
// The C ABI is looked up with dlsym in the library libgradtts.so that the Python package loaded (the same path,
// so the same instance: no second copy of the decoder state and no link-time dependency).
#include <dlfcn.h>

#include <ATen/ATen.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/library.h>

#include <unordered_set>

#include "gradtts.h"

namespace {

struct Api {
  decltype(&gt_last_error) last_error = nullptr;
  decltype(&gt_decoder_workspace_bytes) ws_bytes = nullptr;
  decltype(&gt_reverse_diffusion) reverse = nullptr;
  decltype(&gt_estimator_forward) estimator = nullptr;
  decltype(&gt_maximum_path_workspace_bytes) mas_ws = nullptr;
  decltype(&gt_maximum_path) mas = nullptr;
  decltype(&gt_bucket_attention_workspace_bytes) ba_ws = nullptr;
  decltype(&gt_bucket_attention_forward) ba_fwd = nullptr;
  decltype(&gt_bucket_attention_backward_workspace_bytes) ba_bwd_ws = nullptr;
  decltype(&gt_bucket_attention_backward) ba_bwd = nullptr;
  decltype(&gt_residual_norm_forward) rn_fwd = nullptr;
  decltype(&gt_residual_norm_backward_workspace_bytes) rn_bwd_ws = nullptr;
  decltype(&gt_residual_norm_backward) rn_bwd = nullptr;
};
Api g_api;

const Api& api() {
  TORCH_CHECK(g_api.reverse != nullptr, "gradtts ops: call torch.ops.gradtts.bind(<path of libgradtts.so>) first");
  return g_api;
}

void bind(c10::string_view path) {
  void* h = dlopen(std::string(path).c_str(), RTLD_NOW | RTLD_GLOBAL);
  TORCH_CHECK(h != nullptr, "gradtts ops: dlopen failed: ", dlerror());
  Api a;
  auto sym = [&](const char* n) {
    void* p = dlsym(h, n);
    TORCH_CHECK(p != nullptr, "gradtts ops: missing symbol ", n);
    return p;
  };
  a.last_error = reinterpret_cast<decltype(a.last_error)>(sym("gt_last_error"));
  a.ws_bytes = reinterpret_cast<decltype(a.ws_bytes)>(sym("gt_decoder_workspace_bytes"));
  a.reverse = reinterpret_cast<decltype(a.reverse)>(sym("gt_reverse_diffusion"));
  a.estimator = reinterpret_cast<decltype(a.estimator)>(sym("gt_estimator_forward"));
  a.mas_ws = reinterpret_cast<decltype(a.mas_ws)>(sym("gt_maximum_path_workspace_bytes"));
  a.mas = reinterpret_cast<decltype(a.mas)>(sym("gt_maximum_path"));
  a.ba_ws = reinterpret_cast<decltype(a.ba_ws)>(sym("gt_bucket_attention_workspace_bytes"));
  a.ba_fwd = reinterpret_cast<decltype(a.ba_fwd)>(sym("gt_bucket_attention_forward"));
  a.ba_bwd_ws = reinterpret_cast<decltype(a.ba_bwd_ws)>(sym("gt_bucket_attention_backward_workspace_bytes"));
  a.ba_bwd = reinterpret_cast<decltype(a.ba_bwd)>(sym("gt_bucket_attention_backward"));
  a.rn_fwd = reinterpret_cast<decltype(a.rn_fwd)>(sym("gt_residual_norm_forward"));
  a.rn_bwd_ws = reinterpret_cast<decltype(a.rn_bwd_ws)>(sym("gt_residual_norm_backward_workspace_bytes"));
  a.rn_bwd = reinterpret_cast<decltype(a.rn_bwd)>(sym("gt_residual_norm_backward"));
  g_api = a;
}

void check_decoder_io(const at::Tensor& x, const at::Tensor& mask, const at::Tensor& mu, const char* xname) {
  TORCH_CHECK(x.dim() == 3 && x.size(1) == 80, "gradtts: ", xname, " must be [B, 80, T], got ", x.sizes());
  TORCH_CHECK(mu.sizes() == x.sizes(), "gradtts: mu must match ", xname, " ", x.sizes(), ", got ", mu.sizes());
  TORCH_CHECK(mask.dim() == 3 && mask.size(0) == x.size(0) && mask.size(1) == 1 && mask.size(2) == x.size(2),
              "gradtts: mask must be [B, 1, T], got ", mask.sizes());
  TORCH_CHECK(x.size(2) % 4 == 0, "gradtts: T must be a multiple of 4 (fix_len_compatibility, model/utils.py:13-17)");
  TORCH_CHECK(x.is_floating_point() && mu.is_floating_point() && mask.is_floating_point(),
              "gradtts: floating-point inputs expected");
}

at::Tensor f32c(const at::Tensor& t, const at::Device& dev) { return t.to(dev, at::kFloat).contiguous(); }

hipStream_t stream_of(const at::Device& dev) { return c10::hip::getCurrentHIPStream(dev.index()).stream(); }

// Masks are 0/1 (sequence_mask, model/utils.py:6-10; the reference's callers never build others). The decoder's fused
// kernels rely on it: the reference masks some operands twice (Block: (Mish(GN(h))*m + tb)*m, diffusion.py:56-58,
// 74-77), which the library computes as one multiply -- exact for 0/1 masks, 40-60 % off for fractional ones. A
// fractional mask is therefore rejected here instead of decoded wrongly. The check reads one flag back (a host
// sync); inside a HIP-graph capture, where no host read is allowed, it is skipped (the captured call was checked when
// its inputs were made, or is the caller's contract).
void check_binary_mask(const at::Tensor& m32, hipStream_t s) {
  hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
  if (hipStreamIsCapturing(s, &st) != hipSuccess || st != hipStreamCaptureStatusNone) return;
  const bool bad = (m32.ne(0) & m32.ne(1)).any().item<bool>();
  TORCH_CHECK(!bad, "gradtts: mask values must be 0 or 1 (sequence_mask); fractional masks are not supported by the "
              "fused decoder (the reference's double masking x*m*m is computed as x*m)");
}

at::Tensor reverse_diffusion_hip(int64_t decoder, int64_t dtype, const at::Tensor& z, const at::Tensor& mask,
                                 const at::Tensor& mu, int64_t n_timesteps, const std::optional<at::Tensor>& spk) {
  check_decoder_io(z, mask, mu, "z");
  TORCH_CHECK(n_timesteps >= 0 && n_timesteps < (int64_t(1) << 31), "gradtts: bad n_timesteps ", n_timesteps);
  const at::Device dev = z.device();
  c10::DeviceGuard guard(dev);
  const int64_t B = z.size(0), T = z.size(2);
  at::Tensor z32 = f32c(z, dev), m32 = f32c(mask, dev), mu32 = f32c(mu, dev);
  at::Tensor s32;
  if (spk.has_value()) s32 = f32c(*spk, dev);
  at::Tensor out = at::empty({B, 80, T}, z32.options());
  if (B == 0) return out.to(z.scalar_type());
  check_binary_mask(m32, stream_of(dev));
  auto* d = reinterpret_cast<gt_decoder*>(decoder);
  const Api& A = api();
  const size_t nb = A.ws_bytes(d, (int)dtype, B, T, (int32_t)n_timesteps);
  at::Tensor ws = at::empty({(int64_t)nb}, z32.options().dtype(at::kByte));
  const int rc = A.reverse(d, (int)dtype, z32.data_ptr<float>(), m32.data_ptr<float>(), mu32.data_ptr<float>(),
                           s32.defined() ? s32.data_ptr<float>() : nullptr, B, T, (int32_t)n_timesteps,
                           out.data_ptr<float>(), ws.data_ptr(), nb, stream_of(dev));
  TORCH_CHECK(rc == GT_OK, "gt_reverse_diffusion failed (code ", rc, "): ", A.last_error());
  return out.to(z.scalar_type());
}

at::Tensor estimator_hip(int64_t decoder, int64_t dtype, const at::Tensor& x, const at::Tensor& mask,
                         const at::Tensor& mu, const at::Tensor& t, const std::optional<at::Tensor>& spk) {
  check_decoder_io(x, mask, mu, "x");
  const at::Device dev = x.device();
  c10::DeviceGuard guard(dev);
  const int64_t B = x.size(0), T = x.size(2);
  TORCH_CHECK(t.numel() == B || t.numel() == 1, "gradtts: t must have B or 1 elements, got ", t.numel());
  at::Tensor x32 = f32c(x, dev), m32 = f32c(mask, dev), mu32 = f32c(mu, dev);
  at::Tensor t32 = f32c(t.reshape({-1}).expand({B}), dev);
  at::Tensor s32;
  if (spk.has_value()) s32 = f32c(*spk, dev);
  at::Tensor out = at::empty({B, 80, T}, x32.options());
  if (B == 0) return out.to(x.scalar_type());
  check_binary_mask(m32, stream_of(dev));
  auto* d = reinterpret_cast<gt_decoder*>(decoder);
  const Api& A = api();
  const size_t nb = A.ws_bytes(d, (int)dtype, B, T, 0);
  at::Tensor ws = at::empty({(int64_t)nb}, x32.options().dtype(at::kByte));
  const int rc = A.estimator(d, (int)dtype, x32.data_ptr<float>(), m32.data_ptr<float>(), mu32.data_ptr<float>(),
                             t32.data_ptr<float>(), s32.defined() ? s32.data_ptr<float>() : nullptr, B, T,
                             out.data_ptr<float>(), ws.data_ptr(), nb, stream_of(dev));
  TORCH_CHECK(rc == GT_OK, "gt_estimator_forward failed (code ", rc, "): ", A.last_error());
  return out.to(x.scalar_type());
}

// maximum_path (monotonic_align/__init__.py:8-23): value * mask in fp32, t_x = mask.sum(1)[:, 0],
// t_y = mask.sum(2)[:, 0], the DP on device; the path comes back as value.dtype.
at::Tensor maximum_path_hip(const at::Tensor& value, const at::Tensor& mask) {
  TORCH_CHECK(value.dim() == 3 && mask.sizes() == value.sizes(), "gradtts: value and mask must both be [b, t_x, t_y]");
  const at::Device dev = value.device();
  c10::DeviceGuard guard(dev);
  at::Tensor v = (value * mask.to(dev)).to(at::kFloat).contiguous();
  at::Tensor m = mask.to(dev);
  at::Tensor t_x = m.sum(1).select(1, 0).to(at::kInt).contiguous();
  at::Tensor t_y = m.sum(2).select(1, 0).to(at::kInt).contiguous();
  at::Tensor path = at::empty(v.sizes(), v.options().dtype(at::kInt));
  if (v.numel() > 0) {
    const Api& A = api();
    const int64_t b = v.size(0), tx = v.size(1), ty = v.size(2);
    const size_t nb = A.mas_ws(b, tx, ty);
    at::Tensor ws = at::empty({(int64_t)std::max<size_t>(nb, 1)}, v.options().dtype(at::kByte));
    const int rc = A.mas(path.data_ptr<int32_t>(), v.data_ptr<float>(), t_x.data_ptr<int32_t>(),
                         t_y.data_ptr<int32_t>(), b, tx, ty, -1e9f, ws.data_ptr(), (size_t)ws.numel(), stream_of(dev));
    TORCH_CHECK(rc == GT_OK, "gt_maximum_path failed (code ", rc, "): ", A.last_error());
  }
  return path.to(value.scalar_type());
}

// ---- Meta kernels (shapes / dtypes only)
at::Tensor reverse_diffusion_meta(int64_t, int64_t, const at::Tensor& z, const at::Tensor& mask, const at::Tensor& mu,
                                  int64_t, const std::optional<at::Tensor>&) {
  check_decoder_io(z, mask, mu, "z");
  return at::empty_like(z);
}
at::Tensor estimator_meta(int64_t, int64_t, const at::Tensor& x, const at::Tensor& mask, const at::Tensor& mu,
                          const at::Tensor&, const std::optional<at::Tensor>&) {
  check_decoder_io(x, mask, mu, "x");
  return at::empty_like(x);
}
at::Tensor maximum_path_meta(const at::Tensor& value, const at::Tensor& mask) {
  TORCH_CHECK(value.dim() == 3 && mask.sizes() == value.sizes(), "gradtts: value and mask must both be [b, t_x, t_y]");
  return at::empty_like(value);
}

// ================================================================ operators of transformer blocks
using OptTensor = std::optional<at::Tensor>;

int elem_of(const at::Tensor& t, const char* name) {
  switch (t.scalar_type()) {
    case at::kFloat: return GT_ELEM_F32;
    case at::kBFloat16: return GT_ELEM_BF16;
    case at::kHalf: return GT_ELEM_F16;
    default: TORCH_CHECK(false, "gradtts: ", name, " must be float32, bfloat16 or float16, got ", t.scalar_type());
  }
}
// lengths and starts: integers [B], int64 on the operator's device (copied there if they are not)
void check_ints(const OptTensor& t, int64_t B, const char* name) {
  if (!t.has_value()) return;
  TORCH_CHECK(t->dim() == 1 && t->size(0) == B && !t->is_floating_point() && !t->is_complex() && t->scalar_type() != at::kBool,
              "gradtts: ", name, " must be integers [", B, "], got ", t->scalar_type(), " ", t->sizes());
}
at::Tensor ints_on(const OptTensor& t, const at::Device& dev) {
  return t.has_value() ? t->to(dev, at::kLong).contiguous() : at::Tensor();
}
const int64_t* ints_ptr(const at::Tensor& t) { return t.defined() ? t.data_ptr<int64_t>() : nullptr; }
at::Tensor unit_channels(const at::Tensor& t) { return t.size(3) <= 1 || t.stride(3) == 1 ? t : t.contiguous(); }
gt_stride stride3(const at::Tensor& t) { return {t.stride(0), t.stride(1), t.stride(2)}; }

void check_attention(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& table,
                     const OptTensor& lengths, const OptTensor& q_lengths, const OptTensor& q_start) {
  TORCH_CHECK(q.dim() == 4 && k.dim() == 4, "gradtts: q must be [B, Tq, Hq, D] and k [B, Tk, Hkv, D], got ", q.sizes(),
              " and ", k.sizes());
  TORCH_CHECK(v.sizes() == k.sizes(), "gradtts: v must match k ", k.sizes(), ", got ", v.sizes());
  TORCH_CHECK(k.size(0) == q.size(0) && k.size(3) == q.size(3), "gradtts: q ", q.sizes(), " and k ", k.sizes(),
              " differ in batch or head size");
  TORCH_CHECK(k.size(2) > 0 && q.size(2) > 0 && q.size(2) % k.size(2) == 0, "gradtts: query heads ", q.size(2),
              " must be a multiple of key / value heads ", k.size(2));
  TORCH_CHECK(table.dim() == 2 && table.size(1) == q.size(2), "gradtts: table must be [n_buckets, ", q.size(2), "], got ",
              table.sizes());
  elem_of(q, "q");
  for (const at::Tensor* t : {&k, &v, &table}) {
    TORCH_CHECK(t->scalar_type() == q.scalar_type(), "gradtts: q, k, v and table must have one type, got ",
                q.scalar_type(), " and ", t->scalar_type());
    TORCH_CHECK(t->device() == q.device(), "gradtts: q, k, v and table must be on one device, got ", q.device(), " and ",
                t->device());
  }
  check_ints(lengths, q.size(0), "lengths");
  check_ints(q_lengths, q.size(0), "q_lengths");
  check_ints(q_start, q.size(0), "q_start");
}

gt_bucket_attention attention_args(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& table,
                                   const at::Tensor& len, const at::Tensor& qlen, const at::Tensor& qstart, bool causal,
                                   int64_t max_distance, double scale, const at::Tensor& out) {
  gt_bucket_attention a{};
  a.dtype = elem_of(q, "q");
  a.causal = causal;
  a.n_buckets = (int32_t)std::min<int64_t>(table.size(0), INT32_MAX);
  a.max_distance = (int32_t)std::max<int64_t>(std::min<int64_t>(max_distance, INT32_MAX), 0);
  a.scale = (float)scale;
  a.B = q.size(0); a.Tq = q.size(1); a.Hq = q.size(2); a.D = q.size(3); a.Tk = k.size(1); a.Hkv = k.size(2);
  a.q = q.data_ptr(); a.k = k.data_ptr(); a.v = v.data_ptr(); a.table = table.data_ptr();
  a.q_stride = stride3(q); a.k_stride = stride3(k); a.v_stride = stride3(v); a.out_stride = stride3(out);
  a.lengths = ints_ptr(len); a.q_lengths = ints_ptr(qlen); a.q_start = ints_ptr(qstart);
  return a;
}
at::Tensor workspace(size_t bytes, const at::Tensor& like) {
  return at::empty({(int64_t)bytes}, like.options().dtype(at::kByte));
}

std::tuple<at::Tensor, at::Tensor> bucket_attention_hip(const at::Tensor& q0, const at::Tensor& k0, const at::Tensor& v0,
                                                        const at::Tensor& table0, const OptTensor& lengths,
                                                        const OptTensor& q_lengths, const OptTensor& q_start, bool causal,
                                                        int64_t max_distance, double scale) {
  check_attention(q0, k0, v0, table0, lengths, q_lengths, q_start);
  const at::Device dev = q0.device();
  c10::DeviceGuard guard(dev);
  const at::Tensor q = unit_channels(q0), k = unit_channels(k0), v = unit_channels(v0), table = table0.contiguous();
  const at::Tensor len = ints_on(lengths, dev), qlen = ints_on(q_lengths, dev), qs = ints_on(q_start, dev);
  at::Tensor out = at::empty(q.sizes(), q.options());
  at::Tensor lse = at::empty({q.size(0), q.size(2), q.size(1)}, q.options().dtype(at::kFloat));
  const gt_bucket_attention a = attention_args(q, k, v, table, len, qlen, qs, causal, max_distance, scale, out);
  const Api& A = api();
  const size_t nb = A.ba_ws(&a);
  at::Tensor ws;
  if (nb) ws = workspace(nb, q);
  const int rc = A.ba_fwd(&a, out.data_ptr(), lse.data_ptr<float>(), nb ? ws.data_ptr() : nullptr, nb, stream_of(dev));
  TORCH_CHECK(rc == GT_OK, "gt_bucket_attention_forward failed (code ", rc, "): ", A.last_error());
  return {out, lse};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> bucket_attention_backward_hip(
    const at::Tensor& dout0, const at::Tensor& q0, const at::Tensor& k0, const at::Tensor& v0, const at::Tensor& table0,
    const OptTensor& lengths, const OptTensor& q_lengths, const OptTensor& q_start, const at::Tensor& out0,
    const at::Tensor& lse0, bool causal, int64_t max_distance, double scale) {
  check_attention(q0, k0, v0, table0, lengths, q_lengths, q_start);
  TORCH_CHECK(dout0.sizes() == q0.sizes() && dout0.scalar_type() == q0.scalar_type() && dout0.device() == q0.device() &&
              out0.sizes() == q0.sizes() && out0.scalar_type() == q0.scalar_type() && out0.device() == q0.device(),
              "gradtts: out and its gradient must match q");
  TORCH_CHECK(lse0.scalar_type() == at::kFloat && lse0.dim() == 3 && lse0.size(0) == q0.size(0) && lse0.size(1) == q0.size(2) &&
              lse0.size(2) == q0.size(1) && lse0.device() == q0.device(), "gradtts: lse must be float32 [B, Hq, Tq]");
  const at::Device dev = q0.device();
  c10::DeviceGuard guard(dev);
  const at::Tensor q = unit_channels(q0), k = unit_channels(k0), v = unit_channels(v0), table = table0.contiguous();
  const at::Tensor len = ints_on(lengths, dev), qlen = ints_on(q_lengths, dev), qs = ints_on(q_start, dev);
  const at::Tensor out = unit_channels(out0), dout = unit_channels(dout0), lse = lse0.contiguous();
  at::Tensor dq = at::empty(q.sizes(), q.options()), dk = at::empty(k.sizes(), k.options()),
             dv = at::empty(v.sizes(), v.options()), dtable = at::empty(table.sizes(), table.options());
  const gt_bucket_attention a = attention_args(q, k, v, table, len, qlen, qs, causal, max_distance, scale, out);
  const Api& A = api();
  const size_t nb = A.ba_bwd_ws(&a);
  at::Tensor ws = workspace(nb, q);
  gt_bucket_attention_grads g{dout.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), dtable.data_ptr(),
                              stride3(dout), stride3(dq), stride3(dk), stride3(dv)};
  const int rc = A.ba_bwd(&a, out.data_ptr(), lse.data_ptr<float>(), &g, ws.data_ptr(), nb, stream_of(dev));
  TORCH_CHECK(rc == GT_OK, "gt_bucket_attention_backward failed (code ", rc, "): ", A.last_error());
  return {dq, dk, dv, dtable};
}

void check_norm(const at::Tensor& x, const at::Tensor& y, const OptTensor& gate, const at::Tensor& w1, const OptTensor& b1,
                const at::Tensor& w2, const OptTensor& b2, const OptTensor& lengths) {
  TORCH_CHECK(x.dim() == 3, "gradtts: x must be [B, T, C], got ", x.sizes());
  TORCH_CHECK(y.sizes() == x.sizes() && y.scalar_type() == x.scalar_type() && y.device() == x.device(),
              "gradtts: y must match x ", x.sizes(), " ", x.scalar_type(), ", got ", y.sizes(), " ", y.scalar_type());
  elem_of(x, "x");
  const int64_t C = x.size(2);
  auto param = [&](const at::Tensor& t, const char* name, bool batch) {
    TORCH_CHECK(t.scalar_type() == at::kFloat && t.device() == x.device() &&
                ((t.dim() == 1 && t.size(0) == C) || (batch && t.dim() == 2 && t.size(0) == x.size(0) && t.size(1) == C)),
                "gradtts: ", name, " must be float32 [", C, "]", batch ? " or [B, C]" : "", " on x's device, got ",
                t.scalar_type(), " ", t.sizes());
  };
  param(w1, "post_weight", false);
  param(w2, "pre_weight", false);
  if (b1.has_value()) param(*b1, "post_bias", false);
  if (b2.has_value()) param(*b2, "pre_bias", false);
  if (gate.has_value()) param(*gate, "gate", true);
  check_ints(lengths, x.size(0), "lengths");
}

struct NormArgs {   // the call's contiguous tensors, kept alive, and their parameter block
  at::Tensor x, y, gate, w1, b1, w2, b2, len;
  gt_residual_norm a{};
  NormArgs(const at::Tensor& x0, const at::Tensor& y0, const OptTensor& gate0, const at::Tensor& w10, const OptTensor& b10,
           const at::Tensor& w20, const OptTensor& b20, const OptTensor& lengths, double scale, double eps, bool rms) {
    auto c = [](const OptTensor& t) { return t.has_value() ? t->contiguous() : at::Tensor(); };
    auto f = [](const at::Tensor& t) { return t.defined() ? t.data_ptr<float>() : nullptr; };
    x = x0.contiguous(); y = y0.contiguous(); w1 = w10.contiguous(); w2 = w20.contiguous();
    gate = c(gate0); b1 = c(b10); b2 = c(b20); len = ints_on(lengths, x.device());
    a.dtype = elem_of(x, "x"); a.rms = rms; a.gate_per_batch = gate.defined() && gate.dim() == 2;
    a.scale = (float)scale; a.eps = (float)eps;
    a.B = x.size(0); a.T = x.size(1); a.C = x.size(2);
    a.x = x.data_ptr(); a.y = y.data_ptr();
    a.gate = f(gate); a.post_weight = f(w1); a.post_bias = f(b1); a.pre_weight = f(w2); a.pre_bias = f(b2);
    a.lengths = ints_ptr(len);
  }
};

std::tuple<at::Tensor, at::Tensor, at::Tensor> residual_norm_hip(
    const at::Tensor& x, const at::Tensor& y, const OptTensor& gate, const at::Tensor& w1, const OptTensor& b1,
    const at::Tensor& w2, const OptTensor& b2, const OptTensor& lengths, double scale, double eps, bool rms) {
  check_norm(x, y, gate, w1, b1, w2, b2, lengths);
  c10::DeviceGuard guard(x.device());
  const NormArgs n(x, y, gate, w1, b1, w2, b2, lengths, scale, eps, rms);
  at::Tensor out = at::empty(x.sizes(), x.options()), h = at::empty(x.sizes(), x.options());
  at::Tensor stats = at::empty({x.size(0), x.size(1), 4}, x.options().dtype(at::kFloat));
  const Api& A = api();
  const int rc = A.rn_fwd(&n.a, out.data_ptr(), h.data_ptr(), stats.data_ptr<float>(), stream_of(x.device()));
  TORCH_CHECK(rc == GT_OK, "gt_residual_norm_forward failed (code ", rc, "): ", A.last_error());
  return {out, h, stats};
}

// dx, dy, dgate, dpost_weight, dpost_bias, dpre_weight, dpre_bias (empty for an absent parameter)
std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor> residual_norm_backward_hip(
    const at::Tensor& dout0, const at::Tensor& dh0, const at::Tensor& x, const at::Tensor& y, const OptTensor& gate,
    const at::Tensor& w1, const OptTensor& b1, const at::Tensor& w2, const OptTensor& b2, const OptTensor& lengths,
    const at::Tensor& stats0, double scale, double eps, bool rms) {
  check_norm(x, y, gate, w1, b1, w2, b2, lengths);
  for (const at::Tensor* t : {&dout0, &dh0})
    TORCH_CHECK(t->sizes() == x.sizes() && t->scalar_type() == x.scalar_type() && t->device() == x.device(),
                "gradtts: the outputs' gradients must match x");
  TORCH_CHECK(stats0.scalar_type() == at::kFloat && stats0.dim() == 3 && stats0.size(0) == x.size(0) &&
              stats0.size(1) == x.size(1) && stats0.size(2) == 4 && stats0.device() == x.device(),
              "gradtts: stats must be float32 [B, T, 4]");
  c10::DeviceGuard guard(x.device());
  const NormArgs n(x, y, gate, w1, b1, w2, b2, lengths, scale, eps, rms);
  const at::Tensor dout = dout0.contiguous(), dh = dh0.contiguous(), stats = stats0.contiguous();
  const auto f32 = x.options().dtype(at::kFloat);
  auto like = [&](const at::Tensor& t) { return t.defined() ? at::empty(t.sizes(), f32) : at::empty({0}, f32); };
  at::Tensor dx = at::empty(x.sizes(), x.options()), dy = at::empty(x.sizes(), x.options());
  at::Tensor dg = like(n.gate), dw1 = like(n.w1), db1 = like(n.b1), dw2 = like(n.w2), db2 = like(n.b2);
  auto f = [](const at::Tensor& has, const at::Tensor& t) { return has.defined() ? t.data_ptr<float>() : nullptr; };
  const Api& A = api();
  const size_t nb = A.rn_bwd_ws(&n.a);
  at::Tensor ws = workspace(nb, x);
  gt_residual_norm_grads g{dout.data_ptr(), dh.data_ptr(), dx.data_ptr(), dy.data_ptr(), f(n.gate, dg), f(n.w1, dw1),
                           f(n.b1, db1), f(n.w2, dw2), f(n.b2, db2)};
  const int rc = A.rn_bwd(&n.a, stats.data_ptr<float>(), &g, ws.data_ptr(), nb, stream_of(x.device()));
  TORCH_CHECK(rc == GT_OK, "gt_residual_norm_backward failed (code ", rc, "): ", A.last_error());
  return {dx, dy, dg, dw1, db1, dw2, db2};
}

std::tuple<at::Tensor, at::Tensor> bucket_attention_meta(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                                                         const at::Tensor& table, const OptTensor& lengths,
                                                         const OptTensor& q_lengths, const OptTensor& q_start, bool,
                                                         int64_t, double) {
  check_attention(q, k, v, table, lengths, q_lengths, q_start);
  return {at::empty_symint(q.sym_sizes(), q.options()),
          at::empty_symint({q.sym_size(0), q.sym_size(2), q.sym_size(1)}, q.options().dtype(at::kFloat))};
}
std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> bucket_attention_backward_meta(
    const at::Tensor&, const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& table,
    const OptTensor&, const OptTensor&, const OptTensor&, const at::Tensor&, const at::Tensor&, bool, int64_t, double) {
  auto e = [](const at::Tensor& t) { return at::empty_symint(t.sym_sizes(), t.options()); };
  return {e(q), e(k), e(v), e(table)};
}
std::tuple<at::Tensor, at::Tensor, at::Tensor> residual_norm_meta(
    const at::Tensor& x, const at::Tensor& y, const OptTensor& gate, const at::Tensor& w1, const OptTensor& b1,
    const at::Tensor& w2, const OptTensor& b2, const OptTensor& lengths, double, double, bool) {
  check_norm(x, y, gate, w1, b1, w2, b2, lengths);
  auto e = [&] { return at::empty_symint(x.sym_sizes(), x.options()); };
  return {e(), e(), at::empty_symint({x.sym_size(0), x.sym_size(1), 4}, x.options().dtype(at::kFloat))};
}
std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor> residual_norm_backward_meta(
    const at::Tensor&, const at::Tensor&, const at::Tensor& x, const at::Tensor& y, const OptTensor& gate,
    const at::Tensor& w1, const OptTensor& b1, const at::Tensor& w2, const OptTensor& b2, const OptTensor&,
    const at::Tensor&, double, double, bool) {
  auto e = [](const at::Tensor& t) { return at::empty_symint(t.sym_sizes(), t.options()); };
  auto o = [&](const OptTensor& t) { return t.has_value() ? e(*t) : at::empty({0}, w1.options()); };
  return {e(x), e(y), o(gate), e(w1), o(b1), e(w2), o(b2)};
}

// ---- autograd
// A backward pass captured into a HIP graph must not meet a gradient accumulator that an eager graph of the same leaf
// still holds: it belongs to the eager graph's stream, and autograd's wait on that stream ends the capture, and with it
// the process. Such a capture is refused here, where the caller can still handle it.
void check_capture(std::initializer_list<const at::Tensor*> inputs) {
  const at::Tensor& first = **inputs.begin();
  if (!first.is_cuda() || !at::GradMode::is_enabled()) return;
  const auto cur = c10::hip::getCurrentHIPStream(first.device().index());
  hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
  if (hipStreamIsCapturing(cur.stream(), &st) != hipSuccess || st == hipStreamCaptureStatusNone) return;
  auto check = [&](torch::autograd::Node* acc) {
    const auto s = acc->stream();
    TORCH_CHECK(!s.has_value() || *s == cur.unwrap(),
                "gradtts: a graph capture with gradients while an eager autograd graph of the same parameters is alive "
                "(its gradient accumulators run on another stream); free that graph (its loss and outputs) first");
  };
  // the inputs that are leaves, and the leaves that the others were made from
  std::vector<torch::autograd::Node*> todo;
  std::unordered_set<torch::autograd::Node*> seen;
  for (const at::Tensor* t : inputs) {
    if (!t->defined() || !t->requires_grad()) continue;
    if (t->is_leaf()) {
      if (const auto acc = torch::autograd::impl::try_get_grad_accumulator(*t)) check(acc.get());
    } else if (t->grad_fn()) {
      todo.push_back(t->grad_fn().get());
    }
  }
  while (!todo.empty()) {
    torch::autograd::Node* n = todo.back();
    todo.pop_back();
    if (!seen.insert(n).second) continue;
    if (dynamic_cast<torch::autograd::AccumulateGrad*>(n)) check(n);
    for (const auto& e : n->next_edges())
      if (e.function) todo.push_back(e.function.get());
  }
}

using torch::autograd::AutogradContext;
using torch::autograd::Variable;
using torch::autograd::variable_list;

OptTensor opt(const at::Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); }
at::Tensor undef(const OptTensor& t) { return t.has_value() ? *t : at::Tensor(); }

// The gradients carry a node of their own where grad mode is on (create_graph): it refuses to be differentiated, where
// operators without one would pass zeros on.
std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> bucket_attention_backward_below(
    const at::Tensor& dout, const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& table,
    const OptTensor& lengths, const OptTensor& q_lengths, const OptTensor& q_start, const at::Tensor& out,
    const at::Tensor& lse, bool causal, int64_t max_distance, double scale) {
  static auto op = c10::Dispatcher::singleton().findSchemaOrThrow("gradtts::bucket_attention_backward", "")
                       .typed<decltype(bucket_attention_backward_hip)>();
  at::AutoDispatchBelowADInplaceOrView below;
  return op.call(dout, q, k, v, table, lengths, q_lengths, q_start, out, lse, causal, max_distance, scale);
}
struct BucketAttentionBackwardFn : torch::autograd::Function<BucketAttentionBackwardFn> {
  static variable_list forward(AutogradContext*, const at::Tensor& dout, const at::Tensor& q, const at::Tensor& k,
                               const at::Tensor& v, const at::Tensor& table, const OptTensor& lengths,
                               const OptTensor& q_lengths, const OptTensor& q_start, const at::Tensor& out,
                               const at::Tensor& lse, bool causal, int64_t max_distance, double scale) {
    auto [dq, dk, dv, dt] = bucket_attention_backward_below(dout, q, k, v, table, lengths, q_lengths, q_start, out, lse,
                                                            causal, max_distance, scale);
    return {dq, dk, dv, dt};
  }
  static variable_list backward(AutogradContext*, variable_list) {
    TORCH_CHECK_NOT_IMPLEMENTED(false, "gradtts: bucket_attention has no second derivatives");
  }
};
std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> bucket_attention_backward_autograd(
    const at::Tensor& dout, const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& table,
    const OptTensor& lengths, const OptTensor& q_lengths, const OptTensor& q_start, const at::Tensor& out,
    const at::Tensor& lse, bool causal, int64_t max_distance, double scale) {
  if (!at::GradMode::is_enabled())
    return bucket_attention_backward_below(dout, q, k, v, table, lengths, q_lengths, q_start, out, lse, causal,
                                           max_distance, scale);
  const auto r = BucketAttentionBackwardFn::apply(dout, q, k, v, table, lengths, q_lengths, q_start, out, lse, causal,
                                                  max_distance, scale);
  return {r[0], r[1], r[2], r[3]};
}

struct BucketAttentionFn : torch::autograd::Function<BucketAttentionFn> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                               const at::Tensor& table, const OptTensor& lengths, const OptTensor& q_lengths,
                               const OptTensor& q_start, bool causal, int64_t max_distance, double scale) {
    static auto op = c10::Dispatcher::singleton().findSchemaOrThrow("gradtts::bucket_attention", "")
                         .typed<decltype(bucket_attention_hip)>();
    at::AutoDispatchBelowADInplaceOrView below;
    auto [out, lse] = op.call(q, k, v, table, lengths, q_lengths, q_start, causal, max_distance, scale);
    ctx->save_for_backward({q, k, v, table, undef(lengths), undef(q_lengths), undef(q_start), out, lse});
    ctx->saved_data["causal"] = causal;
    ctx->saved_data["max_distance"] = max_distance;
    ctx->saved_data["scale"] = scale;
    ctx->mark_non_differentiable({lse});
    return {out, lse};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto s = ctx->get_saved_variables();
    auto [dq, dk, dv, dt] = bucket_attention_backward_autograd(
        grads[0], s[0], s[1], s[2], s[3], opt(s[4]), opt(s[5]), opt(s[6]), s[7], s[8], ctx->saved_data["causal"].toBool(),
        ctx->saved_data["max_distance"].toInt(), ctx->saved_data["scale"].toDouble());
    return {dq, dk, dv, dt, Variable(), Variable(), Variable(), Variable(), Variable(), Variable()};
  }
};
std::tuple<at::Tensor, at::Tensor> bucket_attention_autograd(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                                                             const at::Tensor& table, const OptTensor& lengths,
                                                             const OptTensor& q_lengths, const OptTensor& q_start,
                                                             bool causal, int64_t max_distance, double scale) {
  check_capture({&q, &k, &v, &table});
  const auto r = BucketAttentionFn::apply(q, k, v, table, lengths, q_lengths, q_start, causal, max_distance, scale);
  return {r[0], r[1]};
}

using NormGrads = std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor>;
NormGrads residual_norm_backward_below(const at::Tensor& dout, const at::Tensor& dh, const at::Tensor& x,
                                       const at::Tensor& y, const OptTensor& gate, const at::Tensor& w1,
                                       const OptTensor& b1, const at::Tensor& w2, const OptTensor& b2,
                                       const OptTensor& lengths, const at::Tensor& stats, double scale, double eps,
                                       bool rms) {
  static auto op = c10::Dispatcher::singleton().findSchemaOrThrow("gradtts::residual_norm_backward", "")
                       .typed<decltype(residual_norm_backward_hip)>();
  at::AutoDispatchBelowADInplaceOrView below;
  return op.call(dout, dh, x, y, gate, w1, b1, w2, b2, lengths, stats, scale, eps, rms);
}
struct ResidualNormBackwardFn : torch::autograd::Function<ResidualNormBackwardFn> {
  static variable_list forward(AutogradContext*, const at::Tensor& dout, const at::Tensor& dh, const at::Tensor& x,
                               const at::Tensor& y, const OptTensor& gate, const at::Tensor& w1, const OptTensor& b1,
                               const at::Tensor& w2, const OptTensor& b2, const OptTensor& lengths,
                               const at::Tensor& stats, double scale, double eps, bool rms) {
    auto [dx, dy, dg, dw1, db1, dw2, db2] =
        residual_norm_backward_below(dout, dh, x, y, gate, w1, b1, w2, b2, lengths, stats, scale, eps, rms);
    return {dx, dy, dg, dw1, db1, dw2, db2};
  }
  static variable_list backward(AutogradContext*, variable_list) {
    TORCH_CHECK_NOT_IMPLEMENTED(false, "gradtts: residual_norm has no second derivatives");
  }
};
NormGrads residual_norm_backward_autograd(const at::Tensor& dout, const at::Tensor& dh, const at::Tensor& x,
                                          const at::Tensor& y, const OptTensor& gate, const at::Tensor& w1,
                                          const OptTensor& b1, const at::Tensor& w2, const OptTensor& b2,
                                          const OptTensor& lengths, const at::Tensor& stats, double scale, double eps,
                                          bool rms) {
  if (!at::GradMode::is_enabled())
    return residual_norm_backward_below(dout, dh, x, y, gate, w1, b1, w2, b2, lengths, stats, scale, eps, rms);
  const auto r = ResidualNormBackwardFn::apply(dout, dh, x, y, gate, w1, b1, w2, b2, lengths, stats, scale, eps, rms);
  return {r[0], r[1], r[2], r[3], r[4], r[5], r[6]};
}

struct ResidualNormFn : torch::autograd::Function<ResidualNormFn> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& y, const OptTensor& gate,
                               const at::Tensor& w1, const OptTensor& b1, const at::Tensor& w2, const OptTensor& b2,
                               const OptTensor& lengths, double scale, double eps, bool rms) {
    static auto op = c10::Dispatcher::singleton().findSchemaOrThrow("gradtts::residual_norm", "")
                         .typed<decltype(residual_norm_hip)>();
    at::AutoDispatchBelowADInplaceOrView below;
    auto [out, h, stats] = op.call(x, y, gate, w1, b1, w2, b2, lengths, scale, eps, rms);
    ctx->save_for_backward({x, y, undef(gate), w1, undef(b1), w2, undef(b2), undef(lengths), stats});
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["rms"] = rms;
    ctx->mark_non_differentiable({stats});
    return {out, h, stats};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto s = ctx->get_saved_variables();
    auto [dx, dy, dg, dw1, db1, dw2, db2] = residual_norm_backward_autograd(
        grads[0], grads[1], s[0], s[1], opt(s[2]), s[3], opt(s[4]), s[5], opt(s[6]), opt(s[7]), s[8],
        ctx->saved_data["scale"].toDouble(), ctx->saved_data["eps"].toDouble(), ctx->saved_data["rms"].toBool());
    auto of = [](const at::Tensor& has, const at::Tensor& g) { return has.defined() ? g : Variable(); };
    return {dx, dy, of(s[2], dg), dw1, of(s[4], db1), dw2, of(s[6], db2), Variable(), Variable(), Variable(), Variable()};
  }
};
std::tuple<at::Tensor, at::Tensor, at::Tensor> residual_norm_autograd(
    const at::Tensor& x, const at::Tensor& y, const OptTensor& gate, const at::Tensor& w1, const OptTensor& b1,
    const at::Tensor& w2, const OptTensor& b2, const OptTensor& lengths, double scale, double eps, bool rms) {
  const at::Tensor g = undef(gate), c1 = undef(b1), c2 = undef(b2);
  check_capture({&x, &y, &g, &w1, &c1, &w2, &c2});
  const auto r = ResidualNormFn::apply(x, y, gate, w1, b1, w2, b2, lengths, scale, eps, rms);
  return {r[0], r[1], r[2]};
}

}  // namespace

TORCH_LIBRARY(gradtts, m) {
  m.def("bind(str library_path) -> ()", &bind);
  m.def("reverse_diffusion(int decoder, int dtype, Tensor z, Tensor mask, Tensor mu, int n_timesteps, Tensor? spk) -> Tensor");
  m.def("estimator(int decoder, int dtype, Tensor x, Tensor mask, Tensor mu, Tensor t, Tensor? spk) -> Tensor");
  m.def("maximum_path(Tensor value, Tensor mask) -> Tensor");
  m.def("bucket_attention(Tensor q, Tensor k, Tensor v, Tensor table, Tensor? lengths, Tensor? q_lengths, "
        "Tensor? q_start, bool causal, int max_distance, float scale) -> (Tensor, Tensor)");
  m.def("bucket_attention_backward(Tensor dout, Tensor q, Tensor k, Tensor v, Tensor table, Tensor? lengths, "
        "Tensor? q_lengths, Tensor? q_start, Tensor out, Tensor lse, bool causal, int max_distance, float scale) -> "
        "(Tensor, Tensor, Tensor, Tensor)");
  m.def("residual_norm(Tensor x, Tensor y, Tensor? gate, Tensor post_weight, Tensor? post_bias, Tensor pre_weight, "
        "Tensor? pre_bias, Tensor? lengths, float scale, float eps, bool rms) -> (Tensor, Tensor, Tensor)");
  m.def("residual_norm_backward(Tensor dout, Tensor dh, Tensor x, Tensor y, Tensor? gate, Tensor post_weight, "
        "Tensor? post_bias, Tensor pre_weight, Tensor? pre_bias, Tensor? lengths, Tensor stats, float scale, float eps, "
        "bool rms) -> (Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(gradtts, CUDA, m) {
  m.impl("reverse_diffusion", &reverse_diffusion_hip);
  m.impl("estimator", &estimator_hip);
  m.impl("maximum_path", &maximum_path_hip);
  m.impl("bucket_attention", &bucket_attention_hip);
  m.impl("bucket_attention_backward", &bucket_attention_backward_hip);
  m.impl("residual_norm", &residual_norm_hip);
  m.impl("residual_norm_backward", &residual_norm_backward_hip);
}

TORCH_LIBRARY_IMPL(gradtts, Autograd, m) {
  m.impl("bucket_attention", &bucket_attention_autograd);
  m.impl("bucket_attention_backward", &bucket_attention_backward_autograd);
  m.impl("residual_norm", &residual_norm_autograd);
  m.impl("residual_norm_backward", &residual_norm_backward_autograd);
}

TORCH_LIBRARY_IMPL(gradtts, Meta, m) {
  m.impl("reverse_diffusion", &reverse_diffusion_meta);
  m.impl("estimator", &estimator_meta);
  m.impl("maximum_path", &maximum_path_meta);
  m.impl("bucket_attention", &bucket_attention_meta);
  m.impl("bucket_attention_backward", &bucket_attention_backward_meta);
  m.impl("residual_norm", &residual_norm_meta);
  m.impl("residual_norm_backward", &residual_norm_backward_meta);
}
