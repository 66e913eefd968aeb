// PyTorch-facing glue for the gfx950 kernels in csrc/kernels.
//
// Each function validates shapes / dtypes / alignment on the host (a kernel
// that reads out of bounds can take the whole node down, so nothing is
// launched on operands the kernels were not written for), allocates outputs
// through the caching allocator, and launches on the current HIP stream.
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/extension.h>

#include <algorithm>
#include <optional>
#include <vector>

#include "kernels/pda_kernels.h"

namespace py = pybind11;

namespace {

pda::DType dtype_of(const at::Tensor& t) {
  if (t.scalar_type() == at::kBFloat16) return pda::kBF16;
  TORCH_CHECK(t.scalar_type() == at::kFloat, "expected a float32 or bfloat16 tensor, got ", t.scalar_type());
  return pda::kF32;
}

void check_gpu(const at::Tensor& t, const char* name) {
  TORCH_CHECK(t.defined(), name, " is undefined");
  TORCH_CHECK(t.is_cuda(), name, " must live on the GPU");
  TORCH_CHECK(t.is_contiguous(), name, " must be contiguous");
  TORCH_CHECK(reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0, name, " must be 16-byte aligned");
}

// Kernels launch on PyTorch's current stream of the current device (set by the DeviceGuard
// each binding takes on its first tensor argument).
hipStream_t current_stream() { return c10::hip::getCurrentHIPStream().stream(); }

void check_launch(const char* what) {
  hipError_t err = hipGetLastError();
  TORCH_CHECK(err == hipSuccess, what, " launch failed: ", hipGetErrorString(err));
}

// ------------------------------------------------------------------ norms --
std::vector<at::Tensor> norm_forward(const at::Tensor& x, const std::optional<at::Tensor>& residual,
                                     const at::Tensor& weight, const std::optional<at::Tensor>& bias,
                                     double eps, bool rms, double dropout_p, uint64_t seed) {
  check_gpu(x, "x");
  TORCH_CHECK(dropout_p >= 0.0 && dropout_p < 1.0, "norm: dropout probability must be in [0, 1)");
  TORCH_CHECK(dropout_p == 0.0 || !rms, "norm: fused dropout is implemented for LayerNorm only");
  check_gpu(weight, "weight");
  const c10::DeviceGuard guard(x.device());
  const int64_t d = x.size(-1);
  const int64_t rows = x.numel() / d;
  const auto dt = dtype_of(x);
  const int vec = dt == pda::kBF16 ? 8 : 4;
  TORCH_CHECK(d % vec == 0 && d <= 64 * 16 * vec, "norm: unsupported row length ", d);
  TORCH_CHECK(weight.numel() == d && weight.scalar_type() == x.scalar_type(), "norm: bad weight");
  const void* bias_ptr = nullptr;
  if (!rms) {
    TORCH_CHECK(bias.has_value(), "layernorm needs a bias");
    check_gpu(*bias, "bias");
    TORCH_CHECK(bias->numel() == d && bias->scalar_type() == x.scalar_type(), "norm: bad bias");
    bias_ptr = bias->data_ptr();
  }
  const void* res_ptr = nullptr;
  at::Tensor sum_out;
  if (residual.has_value()) {
    check_gpu(*residual, "residual");
    TORCH_CHECK(residual->sizes() == x.sizes() && residual->scalar_type() == x.scalar_type(),
                "norm: residual must match x");
    res_ptr = residual->data_ptr();
    sum_out = at::empty_like(x);
  } else if (dropout_p > 0.0) {
    sum_out = at::empty_like(x);  // the normalised row is dropout(x), not x: it is emitted too
  }
  at::Tensor y = at::empty_like(x);
  auto stat_opts = x.options().dtype(at::kFloat);
  at::Tensor rstd = at::empty({rows}, stat_opts);
  at::Tensor mean = rms ? at::Tensor() : at::empty({rows}, stat_opts);
  pda::norm_forward(dt, rms, x.data_ptr(), res_ptr, weight.data_ptr(), bias_ptr, y.data_ptr(),
                    sum_out.defined() ? sum_out.data_ptr() : nullptr,
                    rms ? nullptr : mean.data_ptr<float>(), rstd.data_ptr<float>(), rows, (int)d,
                    (float)eps, (float)dropout_p, seed, current_stream());
  check_launch("norm_forward");
  return {y, sum_out, mean, rstd};
}

std::vector<at::Tensor> norm_backward(const at::Tensor& dy, const at::Tensor& x,
                                      const at::Tensor& weight, const std::optional<at::Tensor>& mean,
                                      const at::Tensor& rstd, const std::optional<at::Tensor>& dresidual,
                                      bool rms, const std::optional<at::Tensor>& dweight_out, bool accumulate_w,
                                      const std::optional<at::Tensor>& dbias_out, bool accumulate_b,
                                      double dropout_p, uint64_t seed) {
  TORCH_CHECK(dropout_p >= 0.0 && dropout_p < 1.0, "norm: dropout probability must be in [0, 1)");
  TORCH_CHECK(dropout_p == 0.0 || !rms, "norm: fused dropout is implemented for LayerNorm only");
  check_gpu(dy, "dy");
  check_gpu(x, "x");
  check_gpu(weight, "weight");
  check_gpu(rstd, "rstd");
  const c10::DeviceGuard guard(x.device());
  const int64_t d = x.size(-1);
  const int64_t rows = x.numel() / d;
  const auto dt = dtype_of(x);
  const int vec = dt == pda::kBF16 ? 8 : 4;
  TORCH_CHECK(d % vec == 0 && d <= 64 * 16 * vec, "norm: unsupported row length ", d);
  TORCH_CHECK(dy.sizes() == x.sizes() && dy.scalar_type() == x.scalar_type(), "norm: dy must match x");
  TORCH_CHECK(weight.numel() == d && weight.scalar_type() == x.scalar_type(), "norm: bad weight");
  TORCH_CHECK(rstd.numel() == rows && rstd.scalar_type() == at::kFloat, "norm: bad rstd");
  const float* mean_ptr = nullptr;
  if (!rms) {
    TORCH_CHECK(mean.has_value() && mean->defined(), "layernorm backward needs mean");
    check_gpu(*mean, "mean");
    TORCH_CHECK(mean->numel() == rows && mean->scalar_type() == at::kFloat, "norm: bad mean");
    mean_ptr = mean->data_ptr<float>();
  }
  const void* dres_ptr = nullptr;
  if (dresidual.has_value() && dresidual->defined()) {
    check_gpu(*dresidual, "dresidual");
    TORCH_CHECK(dresidual->sizes() == x.sizes() && dresidual->scalar_type() == x.scalar_type(),
                "norm: dresidual must match x");
    dres_ptr = dresidual->data_ptr();
  }
  at::Tensor dx = at::empty_like(x);
  // With dropout the branch input gets the masked gradient, the residual stream the full one.
  at::Tensor dx_branch = dropout_p > 0.0 ? at::empty_like(x) : at::Tensor();
  const int prow = pda::norm_backward_partial_rows(rows);
  auto f32 = x.options().dtype(at::kFloat);
  at::Tensor dwp = at::empty({prow, d}, f32);
  at::Tensor dbp = rms ? at::Tensor() : at::empty({prow, d}, f32);
  hipStream_t stream = current_stream();
  pda::norm_backward(dt, rms, dy.data_ptr(), x.data_ptr(), weight.data_ptr(), mean_ptr,
                     rstd.data_ptr<float>(), dres_ptr, dx.data_ptr(),
                     dx_branch.defined() ? dx_branch.data_ptr() : nullptr, dwp.data_ptr<float>(),
                     rms ? nullptr : dbp.data_ptr<float>(), rows, (int)d, (float)dropout_p, seed, stream);
  check_launch("norm_backward");
  // Parameter gradients go into fresh tensors, or (written / accumulated) into the tensors the
  // caller supplies: slices of a reducer's flat gradient buffer, or existing .grad tensors.
  auto sink = [&](const std::optional<at::Tensor>& out, bool accumulate, const char* what) {
    if (!out.has_value() || !out->defined()) {
      TORCH_CHECK(!accumulate, "norm: accumulate needs ", what);
      return at::empty_like(weight);
    }
    TORCH_CHECK(out->is_cuda() && out->is_contiguous() && out->numel() == d &&
                    (out->scalar_type() == at::kBFloat16 || out->scalar_type() == at::kFloat),
                "norm: ", what, " must be a contiguous bf16/fp32 GPU tensor with ", d, " elements");
    return *out;
  };
  at::Tensor dw = sink(dweight_out, accumulate_w, "dweight_out");
  at::Tensor db = rms ? at::Tensor() : sink(dbias_out, accumulate_b, "dbias_out");
  pda::norm_reduce_partials(dwp.data_ptr<float>(), rms ? nullptr : dbp.data_ptr<float>(), prow, (int)d,
                            dtype_of(dw), dw.data_ptr(), accumulate_w, rms ? pda::kF32 : dtype_of(db),
                            rms ? nullptr : db.data_ptr(), accumulate_b, stream);
  check_launch("norm_reduce_partials");
  return {dx, dw, db, dx_branch};
}

// ------------------------------------------------------------ activations --
at::Tensor gelu_forward(const at::Tensor& u) {
  check_gpu(u, "u");
  const c10::DeviceGuard guard(u.device());
  at::Tensor y = at::empty_like(u);
  pda::gelu_forward(dtype_of(u), u.data_ptr(), y.data_ptr(), u.numel(), current_stream());
  check_launch("gelu_forward");
  return y;
}

at::Tensor gelu_backward(const at::Tensor& dy, const at::Tensor& u) {
  check_gpu(dy, "dy");
  check_gpu(u, "u");
  TORCH_CHECK(dy.sizes() == u.sizes() && dy.scalar_type() == u.scalar_type(), "gelu: dy must match u");
  const c10::DeviceGuard guard(u.device());
  at::Tensor du = at::empty_like(u);
  pda::gelu_backward(dtype_of(u), dy.data_ptr(), u.data_ptr(), du.data_ptr(), u.numel(), current_stream());
  check_launch("gelu_backward");
  return du;
}

at::Tensor swiglu_forward(const at::Tensor& x) {
  check_gpu(x, "x");
  const c10::DeviceGuard guard(x.device());
  const int64_t f2 = x.size(-1);
  const auto dt = dtype_of(x);
  const int vec = dt == pda::kBF16 ? 8 : 4;
  TORCH_CHECK(f2 % 2 == 0 && (f2 / 2) % vec == 0, "swiglu: last dim must be 2*f with f % ", vec, " == 0");
  auto sizes = x.sizes().vec();
  sizes.back() = f2 / 2;
  at::Tensor y = at::empty(sizes, x.options());
  pda::swiglu_forward(dt, x.data_ptr(), y.data_ptr(), x.numel() / f2, (int)(f2 / 2), current_stream());
  check_launch("swiglu_forward");
  return y;
}

at::Tensor swiglu_backward(const at::Tensor& dy, const at::Tensor& x) {
  check_gpu(dy, "dy");
  check_gpu(x, "x");
  const c10::DeviceGuard guard(x.device());
  const int64_t f2 = x.size(-1);
  const auto dt = dtype_of(x);
  const int vec = dt == pda::kBF16 ? 8 : 4;
  TORCH_CHECK(f2 % 2 == 0 && (f2 / 2) % vec == 0, "swiglu: bad last dim");
  TORCH_CHECK(dy.scalar_type() == x.scalar_type() && dy.numel() * 2 == x.numel(), "swiglu: dy mismatch");
  at::Tensor dx = at::empty_like(x);
  pda::swiglu_backward(dt, dy.data_ptr(), x.data_ptr(), dx.data_ptr(), x.numel() / f2, (int)(f2 / 2),
                       current_stream());
  check_launch("swiglu_backward");
  return dx;
}

// ---------------------------------------------------------- cross entropy --
// logits: [rows, ld] view (stride(0) = ld >= vocab, stride(1) = 1); overwritten with the gradient.
at::Tensor cross_entropy_fwd_bwd(at::Tensor logits, const at::Tensor& targets, int64_t vocab,
                                 const at::Tensor& grad_scale, int64_t ignore_index) {
  TORCH_CHECK(logits.is_cuda() && logits.dim() == 2 && logits.stride(1) == 1, "ce: bad logits layout");
  TORCH_CHECK(targets.is_cuda() && targets.scalar_type() == at::kLong && targets.is_contiguous(),
              "ce: targets must be contiguous int64 on the GPU");
  TORCH_CHECK(grad_scale.is_cuda() && grad_scale.scalar_type() == at::kFloat && grad_scale.numel() == 1,
              "ce: grad_scale must be a 1-element float32 GPU tensor");
  const int64_t rows = logits.size(0);
  const int64_t ld = logits.stride(0);
  TORCH_CHECK(targets.numel() == rows, "ce: one target per row");
  TORCH_CHECK(vocab > 0 && vocab <= ld && vocab <= logits.size(1) + (ld - logits.size(1)),
              "ce: vocab exceeds the row");
  // The kernel rewrites the whole padded row [0, ld); the storage must own it.
  const int64_t elt = logits.element_size();
  const int64_t end_byte = (logits.storage_offset() + (rows - 1) * ld + ld) * elt;
  TORCH_CHECK(rows == 0 || end_byte <= (int64_t)logits.storage().nbytes(),
              "ce: padded rows run past the end of the logits storage");
  const c10::DeviceGuard guard(logits.device());
  at::Tensor row_loss = at::empty({rows}, logits.options().dtype(at::kFloat));
  pda::cross_entropy_fwd_bwd(dtype_of(logits), logits.data_ptr(), targets.data_ptr<int64_t>(),
                             row_loss.data_ptr<float>(), grad_scale.data_ptr<float>(), rows, (int)vocab,
                             ld, ignore_index, current_stream());
  check_launch("cross_entropy_fwd_bwd");
  return row_loss;
}

// ------------------------------------------------------------------ AdamW --
void adamw_step(const std::vector<at::Tensor>& params, const std::vector<std::optional<at::Tensor>>& lowp,
                const std::vector<at::Tensor>& grads, const std::vector<at::Tensor>& exp_avg,
                const std::vector<at::Tensor>& exp_avg_sq, double lr, double beta1, double beta2,
                double eps, double weight_decay, int64_t step, double grad_scale, bool zero_grad,
                const std::optional<at::Tensor>& dynamic) {
  const size_t n = params.size();
  TORCH_CHECK(grads.size() == n && exp_avg.size() == n && exp_avg_sq.size() == n && lowp.size() == n,
              "adamw: list lengths differ");
  if (n == 0) return;
  TORCH_CHECK(step >= 1, "adamw: step counts from 1");
  const c10::DeviceGuard guard(params[0].device());
  std::vector<pda::AdamWTensor> ts;
  ts.reserve(n);
  const pda::DType gdt = dtype_of(grads[0]);
  for (size_t i = 0; i < n; ++i) {
    check_gpu(params[i], "param");
    check_gpu(grads[i], "grad");
    check_gpu(exp_avg[i], "exp_avg");
    check_gpu(exp_avg_sq[i], "exp_avg_sq");
    TORCH_CHECK(params[i].scalar_type() == at::kFloat && exp_avg[i].scalar_type() == at::kFloat &&
                    exp_avg_sq[i].scalar_type() == at::kFloat,
                "adamw: param / state must be float32");
    TORCH_CHECK(dtype_of(grads[i]) == gdt, "adamw: mixed gradient dtypes in one call");
    const int64_t numel = params[i].numel();
    TORCH_CHECK(grads[i].numel() == numel && exp_avg[i].numel() == numel && exp_avg_sq[i].numel() == numel,
                "adamw: size mismatch at tensor ", i);
    pda::AdamWTensor t;
    t.param = params[i].data_ptr<float>();
    t.lowp = nullptr;
    if (lowp[i].has_value() && lowp[i]->defined()) {
      check_gpu(*lowp[i], "lowp");
      TORCH_CHECK(lowp[i]->scalar_type() == at::kBFloat16 && lowp[i]->numel() == numel, "adamw: bad bf16 mirror");
      t.lowp = lowp[i]->data_ptr();
    }
    t.grad = grads[i].data_ptr();
    t.exp_avg = exp_avg[i].data_ptr<float>();
    t.exp_avg_sq = exp_avg_sq[i].data_ptr<float>();
    t.numel = numel;
    ts.push_back(t);
  }
  pda::AdamWHyper hp;
  hp.lr = (float)lr;
  hp.beta1 = (float)beta1;
  hp.beta2 = (float)beta2;
  hp.eps = (float)eps;
  hp.weight_decay = (float)weight_decay;
  hp.bias_correction1 = (float)(1.0 - std::pow(beta1, (double)step));
  hp.bias_correction2 = (float)(1.0 - std::pow(beta2, (double)step));
  hp.grad_scale = (float)grad_scale;
  if (dynamic.has_value()) {  // device-resident {1 - lr*wd, lr/bc1, 1/sqrt(bc2)}: HIP-graph capture
    TORCH_CHECK(dynamic->is_cuda() && dynamic->scalar_type() == at::kFloat && dynamic->numel() >= 3 &&
                    dynamic->is_contiguous(),
                "adamw: dynamic must be a contiguous float32 GPU tensor with 3 elements");
    hp.dynamic = dynamic->data_ptr<float>();
  }
  pda::adamw_step(ts.data(), (int)n, gdt, hp, zero_grad, current_stream());
  check_launch("adamw_step");
}

void accumulate_bf16_into_f32(const at::Tensor& src, at::Tensor dst, double scale) {
  check_gpu(src, "src");
  check_gpu(dst, "dst");
  TORCH_CHECK(src.scalar_type() == at::kBFloat16 && dst.scalar_type() == at::kFloat &&
                  src.numel() == dst.numel(),
              "accumulate: expected bf16 src and float32 dst of equal size");
  const c10::DeviceGuard guard(src.device());
  pda::accumulate_bf16_into_f32(src.data_ptr(), dst.data_ptr<float>(), src.numel(), (float)scale,
                                current_stream());
  check_launch("accumulate_bf16_into_f32");
}

// -------------------------------------------------------------- attention --
std::vector<at::Tensor> attention_forward(const at::Tensor& qkv, int64_t num_heads, double softmax_scale,
                                          double dropout_p, uint64_t seed) {
  check_gpu(qkv, "qkv");
  TORCH_CHECK(qkv.scalar_type() == at::kBFloat16, "attention: bf16 only");
  TORCH_CHECK(qkv.dim() == 3, "attention: qkv must be [B, T, 3*H*D]");
  const int64_t B = qkv.size(0), T = qkv.size(1), three_hd = qkv.size(2);
  TORCH_CHECK(three_hd % (3 * num_heads) == 0, "attention: bad qkv width");
  const int64_t D = three_hd / (3 * num_heads);
  TORCH_CHECK(D == 64 || D == 128, "attention: head_dim must be 64 or 128, got ", D);
  TORCH_CHECK(T >= 1 && B >= 1, "attention: empty input");
  TORCH_CHECK(dropout_p >= 0.0 && dropout_p < 1.0, "attention: dropout_p must be in [0, 1)");
  const c10::DeviceGuard guard(qkv.device());
  at::Tensor out = at::empty({B, T, num_heads * D}, qkv.options());
  at::Tensor lse = at::empty({B, num_heads, T}, qkv.options().dtype(at::kFloat));
  pda::attention_forward(qkv.data_ptr(), out.data_ptr(), lse.data_ptr<float>(), (int)B, (int)T,
                         (int)num_heads, (int)D, (float)softmax_scale, (float)dropout_p, seed, current_stream());
  check_launch("attention_forward");
  return {out, lse};
}

at::Tensor attention_backward(const at::Tensor& qkv, const at::Tensor& out, const at::Tensor& dout,
                              const at::Tensor& lse, int64_t num_heads, double softmax_scale,
                              double dropout_p, uint64_t seed) {
  check_gpu(qkv, "qkv");
  check_gpu(out, "out");
  check_gpu(dout, "dout");
  check_gpu(lse, "lse");
  TORCH_CHECK(qkv.scalar_type() == at::kBFloat16 && out.scalar_type() == at::kBFloat16 &&
                  dout.scalar_type() == at::kBFloat16 && lse.scalar_type() == at::kFloat,
              "attention backward: dtype mismatch");
  const int64_t B = qkv.size(0), T = qkv.size(1);
  const int64_t D = qkv.size(2) / (3 * num_heads);
  TORCH_CHECK(D == 64 || D == 128, "attention: head_dim must be 64 or 128");
  TORCH_CHECK(out.numel() == B * T * num_heads * D && dout.numel() == out.numel() &&
                  lse.numel() == B * num_heads * T,
              "attention backward: shape mismatch");
  const c10::DeviceGuard guard(qkv.device());
  at::Tensor dqkv = at::empty_like(qkv);
  at::Tensor delta = at::empty_like(lse);
  pda::attention_backward(qkv.data_ptr(), out.data_ptr(), dout.data_ptr(), lse.data_ptr<float>(),
                          delta.data_ptr<float>(), dqkv.data_ptr(), (int)B, (int)T, (int)num_heads,
                          (int)D, (float)softmax_scale, (float)dropout_p, seed, current_stream());
  check_launch("attention_backward");
  return dqkv;
}

// Checks of both window-attention passes; returns {B, T, D} and clamps window and sinks to the length.
struct WindowShape {
  int64_t B, T, H, D, window, sinks;
};
WindowShape check_window(const at::Tensor& qkv, int64_t num_heads, int64_t window, int64_t sinks, double dropout_p) {
  check_gpu(qkv, "qkv");
  TORCH_CHECK(qkv.scalar_type() == at::kBFloat16, "window attention: bf16 only");
  TORCH_CHECK(qkv.dim() == 3, "window attention: qkv must be [B, T, 3*H*D]");
  TORCH_CHECK(num_heads >= 1 && qkv.size(2) % (3 * num_heads) == 0, "window attention: bad qkv width");
  TORCH_CHECK(window >= 1, "window attention: window must be at least 1, got ", window);
  TORCH_CHECK(sinks >= 0, "window attention: sinks must not be negative, got ", sinks);
  TORCH_CHECK(dropout_p >= 0.0 && dropout_p < 1.0, "window attention: dropout_p must be in [0, 1)");
  WindowShape w{qkv.size(0), qkv.size(1), num_heads, qkv.size(2) / (3 * num_heads), window, sinks};
  TORCH_CHECK(w.D == 64 || w.D == 128, "window attention: head_dim must be 64 or 128, got ", w.D);
  TORCH_CHECK(w.B >= 1 && w.T >= 1, "window attention: empty input");
  w.window = std::min(window, w.T);
  w.sinks = std::min(sinks, w.T);
  // (a launch takes less than 2^32 threads: workgroups of 256, one for 128 rows of a head, in the backward one for 32 sinks)
  const int64_t most = std::max((w.T + 127) / 128, w.window < w.T ? (w.sinks + 31) / 32 : 0);
  TORCH_CHECK(w.T <= (1 << 30) && w.B < (1 << 30) && w.H < (1 << 30) && w.B * w.H < (int64_t(1) << 24) &&
                  most * w.B * w.H < (int64_t(1) << 24) && 64 * qkv.size(2) * 2 < (int64_t(1) << 31),
              "window attention: sizes exceed the kernels' 32-bit indices");
  return w;
}

// Contiguous and on a 16-byte boundary, as vector loads need it.
at::Tensor packed16(const at::Tensor& t) {
  const at::Tensor c = t.contiguous();
  return reinterpret_cast<uintptr_t>(c.data_ptr()) % 16 == 0 ? c : c.clone();
}

// {out, out_rest, neg_lse}; out_rest (only with `for_backward`) and neg_lse are the backward's.
std::vector<at::Tensor> window_attention_forward(const at::Tensor& qkv, int64_t num_heads, int64_t window, int64_t sinks,
                                                 double softmax_scale, double dropout_p, uint64_t seed, bool for_backward) {
  const WindowShape w = check_window(qkv, num_heads, window, sinks, dropout_p);
  const c10::DeviceGuard guard(qkv.device());
  at::Tensor out = at::empty({w.B, w.T, w.H * w.D}, qkv.options());
  at::Tensor rest;
  if (for_backward) rest = at::empty(out.sizes(), qkv.options().dtype(at::kByte));
  at::Tensor neg_lse = at::empty({w.B, w.H, w.T}, qkv.options().dtype(at::kFloat));
  pda::window_attention_forward(qkv.data_ptr(), out.data_ptr(), for_backward ? rest.data_ptr() : nullptr, neg_lse.data_ptr<float>(),
                                (int)w.B, (int)w.T, (int)w.H, (int)w.D, (int)w.window, (int)w.sinks, (float)softmax_scale,
                                (float)dropout_p, seed, current_stream());
  check_launch("window_attention_forward");
  return {out, rest, neg_lse};
}

at::Tensor window_attention_backward(const at::Tensor& qkv, const at::Tensor& out, const at::Tensor& out_rest, const at::Tensor& dout,
                                     const at::Tensor& neg_lse, int64_t num_heads, int64_t window, int64_t sinks, double softmax_scale,
                                     double dropout_p, uint64_t seed) {
  const WindowShape w = check_window(qkv, num_heads, window, sinks, dropout_p);
  check_gpu(out, "out");
  check_gpu(out_rest, "out_rest");
  check_gpu(dout, "dout");
  check_gpu(neg_lse, "neg_lse");
  TORCH_CHECK(out.scalar_type() == at::kBFloat16 && dout.scalar_type() == at::kBFloat16 && out_rest.scalar_type() == at::kByte &&
                  neg_lse.scalar_type() == at::kFloat,
              "window attention backward: dtype mismatch");
  TORCH_CHECK(out.numel() == w.B * w.T * w.H * w.D && dout.numel() == out.numel() && out_rest.numel() == out.numel() &&
                  neg_lse.numel() == w.B * w.H * w.T,
              "window attention backward: shape mismatch");
  TORCH_CHECK(out.device() == qkv.device() && dout.device() == qkv.device() && neg_lse.device() == qkv.device() &&
                  out_rest.device() == qkv.device(),
              "window attention backward: tensors on different devices");
  const c10::DeviceGuard guard(qkv.device());
  at::Tensor dqkv = at::empty_like(qkv);
  const size_t bytes = pda::window_attention_backward_workspace_bytes((int)w.B, (int)w.T, (int)w.H, (int)w.D, (int)w.window, (int)w.sinks);
  const int64_t delta_bytes = (w.B * w.H * w.T * 4 + 255) / 256 * 256;  // -delta, then the sinks' partial sums
  at::Tensor scratch = at::empty({delta_bytes + (int64_t)bytes}, qkv.options().dtype(at::kByte));
  float* neg_delta = reinterpret_cast<float*>(scratch.data_ptr());
  void* workspace = bytes ? static_cast<char*>(scratch.data_ptr()) + delta_bytes : nullptr;
  pda::window_attention_dq(qkv.data_ptr(), out.data_ptr(), out_rest.data_ptr(), dout.data_ptr(), neg_lse.data_ptr<float>(),
                           neg_delta, dqkv.data_ptr(), (int)w.B, (int)w.T, (int)w.H, (int)w.D, (int)w.window,
                           (int)w.sinks, (float)softmax_scale, (float)dropout_p, seed, current_stream());
  pda::window_attention_dkv(qkv.data_ptr(), dout.data_ptr(), neg_lse.data_ptr<float>(), neg_delta, dqkv.data_ptr(),
                            workspace, (int)w.B, (int)w.T, (int)w.H, (int)w.D, (int)w.window,
                            (int)w.sinks, (float)softmax_scale, (float)dropout_p, seed, current_stream());
  check_launch("window_attention_backward");
  return dqkv;
}

struct WindowAttentionFn : public torch::autograd::Function<WindowAttentionFn> {
  static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& qkv, int64_t num_heads, int64_t window,
                            int64_t sinks, double softmax_scale, double dropout_p, int64_t seed, bool for_backward) {
    const at::Tensor packed = packed16(qkv);
    auto got = window_attention_forward(packed, num_heads, window, sinks, softmax_scale, dropout_p, (uint64_t)seed, for_backward);
    if (!for_backward) return got[0];
    ctx->save_for_backward({packed, got[0], got[1], got[2]});
    auto& d = ctx->saved_data;
    d["args"] = std::vector<int64_t>{num_heads, window, sinks, seed};
    d["floats"] = std::vector<double>{softmax_scale, dropout_p};
    return got[0];
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    TORCH_CHECK(!at::GradMode::is_enabled(), "window_attention has no second derivative (create_graph=True)");
    const auto saved = ctx->get_saved_variables();
    const auto i = ctx->saved_data["args"].toIntVector();
    const auto f = ctx->saved_data["floats"].toDoubleVector();
    at::Tensor dqkv = window_attention_backward(saved[0], saved[1], saved[2], packed16(grads[0]), saved[3], i[0], i[1], i[2], f[0], f[1], (uint64_t)i[3]);
    const at::Tensor none;
    return {dqkv, none, none, none, none, none, none, none};
  }
};

at::Tensor window_attention(const at::Tensor& qkv, int64_t num_heads, int64_t window, int64_t sinks, double softmax_scale,
                            double dropout_p, int64_t seed) {
  return WindowAttentionFn::apply(qkv, num_heads, window, sinks, softmax_scale, dropout_p, seed,
                                  at::GradMode::is_enabled() && qkv.requires_grad());
}

// keep[B, H, T, T] (bool): the attention-dropout mask the kernels apply for (dropout_p, seed).
at::Tensor attention_dropout_mask(int64_t B, int64_t H, int64_t T, double dropout_p, uint64_t seed,
                                  const at::Device& device) {
  TORCH_CHECK(device.is_cuda(), "attention_dropout_mask: GPU device expected");
  const c10::DeviceGuard guard(device);
  at::Tensor keep = at::empty({B, H, T, T}, at::TensorOptions().dtype(at::kByte).device(device));
  pda::attention_dropout_mask(keep.data_ptr<uint8_t>(), (int)B, (int)T, (int)H, (float)dropout_p, seed,
                              current_stream());
  check_launch("attention_dropout_mask");
  return keep.to(at::kBool);
}

// ------------------------------------------------------------------- rotary --
// [rows, cols] bf16 (unit column stride, any 8-aligned row pitch) -> [cols, rows_padded], rows_padded
// = rows rounded up to pad_rows_to, with the padding columns zero.
at::Tensor transpose_2d(const at::Tensor& src, int64_t pad_rows_to) {
  TORCH_CHECK(src.defined() && src.is_cuda() && src.dim() == 2, "transpose_2d: expected a 2-D GPU tensor");
  TORCH_CHECK(src.scalar_type() == at::kBFloat16, "transpose_2d: bf16 only");
  const int64_t rows = src.size(0), cols = src.size(1);
  TORCH_CHECK(rows > 0 && cols > 0 && rows < (int64_t(1) << 30) && cols < (int64_t(1) << 30), "transpose_2d: bad shape");
  TORCH_CHECK(src.stride(1) == 1 && src.stride(0) >= cols && src.stride(0) % 8 == 0 && cols % 8 == 0,
              "transpose_2d: rows must be contiguous, 16-byte aligned and a multiple of 8 long");
  TORCH_CHECK(reinterpret_cast<uintptr_t>(src.data_ptr()) % 16 == 0, "transpose_2d: source must be 16-byte aligned");
  TORCH_CHECK(pad_rows_to >= 8 && pad_rows_to % 8 == 0, "transpose_2d: pad_rows_to must be a multiple of 8");
  const c10::DeviceGuard guard(src.device());
  const int64_t rows_padded = (rows + pad_rows_to - 1) / pad_rows_to * pad_rows_to;
  at::Tensor out = at::empty({cols, rows_padded}, src.options());
  pda::transpose_bf16(src.data_ptr(), src.stride(0), out.data_ptr(), rows_padded, (int)rows, (int)cols,
                      (int)rows_padded, current_stream());
  check_launch("transpose_2d");
  return out;
}

at::Tensor rope_apply(const at::Tensor& qkv, const at::Tensor& cos, const at::Tensor& sin, int64_t num_heads,
                      bool inverse, bool in_place) {
  check_gpu(qkv, "qkv");
  check_gpu(cos, "cos");
  check_gpu(sin, "sin");
  TORCH_CHECK(qkv.dim() == 3, "rope: qkv must be [B, T, 3*H*D]");
  const int64_t B = qkv.size(0), T = qkv.size(1);
  TORCH_CHECK(qkv.size(2) % (3 * num_heads) == 0, "rope: bad qkv width");
  const int64_t D = qkv.size(2) / (3 * num_heads);
  const auto dt = dtype_of(qkv);
  const int vec = dt == pda::kBF16 ? 8 : 4;
  TORCH_CHECK(D % 2 == 0 && (D / 2) % vec == 0, "rope: head_dim / 2 must be a multiple of ", vec);
  TORCH_CHECK(cos.scalar_type() == at::kFloat && sin.scalar_type() == at::kFloat && cos.dim() == 2 &&
                  sin.sizes() == cos.sizes() && cos.size(0) >= T && cos.size(1) == D / 2,
              "rope: cos / sin must be float32 [>= T, D/2] tables");
  TORCH_CHECK(B * T < (int64_t(1) << 31) && T * D < (int64_t(1) << 31) && 3 * num_heads * D < (int64_t(1) << 31),
              "rope: token count and row length must fit 32-bit indices");
  const c10::DeviceGuard guard(qkv.device());
  at::Tensor out = in_place ? qkv : at::empty_like(qkv);
  pda::rope_apply(dt, qkv.data_ptr(), out.data_ptr(), cos.data_ptr<float>(), sin.data_ptr<float>(), (int)B, (int)T,
                  (int)num_heads, (int)D, inverse, current_stream());
  check_launch("rope_apply");
  return out;
}

// ---------------------------------------------------------------- weight grad --
bool wgrad_supported(int64_t M, int64_t I, int64_t J) { return pda::wgrad_supported((int)M, (int)I, (int)J); }

// Can `n` pairs of `rows` rows each go through linear_wgrad_segments?
bool wgrad_segments_supported(int64_t rows, int64_t I, int64_t J, int64_t n) {
  if (n < 1 || n > pda::wgrad_max_segments() || rows < 32 || rows % 32 != 0) return false;
  const int64_t steps = rows / 32;
  if ((steps & (steps - 1)) != 0 || rows * n >= (int64_t(1) << 31)) return false;
  return pda::wgrad_supported((int)(rows * n), (int)I, (int)J);
}

// dW[I, J] = dy[M, I]^T . x[M, J] and (optionally) db[I] = column sums of dy, both bf16.
// With `out` the weight gradient is written into that tensor (a slice of a reducer's flat
// gradient buffer) instead of a fresh one — added to its contents when `accumulate` is set.
// `out_rows` (default: all I): only the leading rows of dW are produced — for a dy whose trailing
// columns are zero padding (the LM head's logits gradient, V = 50257 in a 50304-column buffer).
std::vector<at::Tensor> linear_wgrad(const at::Tensor& dy, const at::Tensor& x, bool want_bias,
                                     const std::optional<at::Tensor>& out, bool accumulate,
                                     const std::optional<at::Tensor>& bias_out, bool bias_accumulate,
                                     int64_t out_rows) {
  TORCH_CHECK(dy.is_cuda() && x.is_cuda() && dy.dim() == 2 && x.dim() == 2, "wgrad: 2-D GPU tensors");
  TORCH_CHECK(dy.scalar_type() == at::kBFloat16 && x.scalar_type() == at::kBFloat16, "wgrad: bf16 only");
  TORCH_CHECK(dy.stride(1) == 1 && x.stride(1) == 1, "wgrad: rows must be contiguous");
  const int64_t M = dy.size(0), I = dy.size(1), J = x.size(1);
  TORCH_CHECK(x.size(0) == M, "wgrad: row counts differ");
  TORCH_CHECK(pda::wgrad_supported((int)M, (int)I, (int)J), "wgrad: unsupported shape ", M, "x", I, "x", J);
  TORCH_CHECK(dy.stride(0) % 8 == 0 && x.stride(0) % 8 == 0 &&
                  reinterpret_cast<uintptr_t>(dy.data_ptr()) % 16 == 0 &&
                  reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 == 0,
              "wgrad: operands must be 16-byte aligned with row strides that are multiples of 8");
  if (out_rows < 0) out_rows = I;
  TORCH_CHECK(out_rows >= 1 && out_rows <= I && (out_rows * J) % 4 == 0, "wgrad: bad out_rows ", out_rows);
  TORCH_CHECK(out_rows == I || !want_bias, "wgrad: out_rows and the bias gradient are not combined");
  const c10::DeviceGuard guard(dy.device());
  const int S = pda::wgrad_pick_slices((int)M, (int)I, (int)J);
  auto f32 = dy.options().dtype(at::kFloat);
  at::Tensor partial = at::empty({S, I, J}, f32);
  at::Tensor bpartial = want_bias ? at::empty({S, I}, f32) : at::Tensor();
  hipStream_t stream = current_stream();
  pda::wgrad_gemm(dy.data_ptr(), dy.stride(0), x.data_ptr(), x.stride(0), partial.data_ptr<float>(),
                  want_bias ? bpartial.data_ptr<float>() : nullptr, (int)M, (int)I, (int)J, S, stream);
  check_launch("wgrad_gemm");
  at::Tensor dw;
  if (out.has_value()) {
    dw = *out;
    TORCH_CHECK(dw.is_cuda() && dw.is_contiguous() && dw.numel() == out_rows * J &&
                    (dw.scalar_type() == at::kBFloat16 || dw.scalar_type() == at::kFloat),
                "wgrad: out must be a contiguous bf16/fp32 GPU tensor with ", out_rows * J, " elements");
  } else {
    TORCH_CHECK(!accumulate, "wgrad: accumulate needs an out tensor");
    dw = at::empty({out_rows, J}, dy.options());
  }
  at::Tensor db;
  if (want_bias) {
    if (bias_out.has_value() && bias_out->defined()) {
      db = *bias_out;
      TORCH_CHECK(db.is_cuda() && db.is_contiguous() && db.numel() == I &&
                      (db.scalar_type() == at::kBFloat16 || db.scalar_type() == at::kFloat),
                  "wgrad: bias_out must be a contiguous bf16/fp32 GPU tensor with ", I, " elements");
    } else {
      TORCH_CHECK(!bias_accumulate, "wgrad: bias_accumulate needs a bias_out tensor");
      db = at::empty({I}, dy.options());
    }
  }
  pda::wgrad_reduce(partial.data_ptr<float>(), S, out_rows * J, I * J, dtype_of(dw), dw.data_ptr(), accumulate,
                    want_bias ? bpartial.data_ptr<float>() : nullptr, I, want_bias ? dtype_of(db) : pda::kBF16,
                    want_bias ? db.data_ptr() : nullptr, want_bias && bias_accumulate, stream);
  check_launch("wgrad_reduce");
  return {dw, db};
}

// The same product over the row-wise concatenation of up to wgrad_max_segments() (dy, x) pairs that
// live in separate buffers (the micro-batches of a gradient-accumulation window): ONE long-K GEMM and
// one slice reduction instead of one of each per micro-batch. Every pair has the same shape and row
// strides; rows per pair / 32 must be a power of two (the kernel finds a stage's pair with a shift).
std::vector<at::Tensor> linear_wgrad_segments(const std::vector<at::Tensor>& dys, const std::vector<at::Tensor>& xs,
                                              bool want_bias, const std::optional<at::Tensor>& out, bool accumulate,
                                              const std::optional<at::Tensor>& bias_out, bool bias_accumulate) {
  const int64_t n = (int64_t)dys.size();
  TORCH_CHECK(n >= 1 && n <= pda::wgrad_max_segments() && (int64_t)xs.size() == n, "wgrad segments: need 1..",
              pda::wgrad_max_segments(), " (dy, x) pairs, got ", n, " and ", xs.size());
  if (n == 1) return linear_wgrad(dys[0], xs[0], want_bias, out, accumulate, bias_out, bias_accumulate, -1);
  const at::Tensor& dy0 = dys[0];
  const at::Tensor& x0 = xs[0];
  TORCH_CHECK(dy0.is_cuda() && dy0.dim() == 2 && x0.dim() == 2, "wgrad segments: 2-D GPU tensors");
  const int64_t rows = dy0.size(0), I = dy0.size(1), J = x0.size(1);
  TORCH_CHECK(wgrad_segments_supported(rows, I, J, n), "wgrad segments: unsupported shape ", n, "x", rows, "x", I, "x", J);
  const void* a[4];
  const void* b[4];
  for (int64_t k = 0; k < n; ++k) {
    const at::Tensor& dy = dys[k];
    const at::Tensor& x = xs[k];
    TORCH_CHECK(dy.is_cuda() && x.is_cuda() && dy.device() == dy0.device() && x.device() == dy0.device() &&
                    dy.scalar_type() == at::kBFloat16 && x.scalar_type() == at::kBFloat16,
                "wgrad segments: bf16 tensors on one GPU");
    TORCH_CHECK(dy.dim() == 2 && x.dim() == 2 && dy.size(0) == rows && x.size(0) == rows && dy.size(1) == I &&
                    x.size(1) == J && dy.stride(1) == 1 && x.stride(1) == 1 && dy.stride(0) == dy0.stride(0) &&
                    x.stride(0) == x0.stride(0),
                "wgrad segments: pair ", k, " differs in shape or strides from pair 0");
    TORCH_CHECK(dy.stride(0) % 8 == 0 && x.stride(0) % 8 == 0 && reinterpret_cast<uintptr_t>(dy.data_ptr()) % 16 == 0 &&
                    reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 == 0,
                "wgrad segments: operands must be 16-byte aligned with row strides that are multiples of 8");
    a[k] = dy.data_ptr();
    b[k] = x.data_ptr();
  }
  const c10::DeviceGuard guard(dy0.device());
  const int64_t M = rows * n;
  const int S = pda::wgrad_pick_slices((int)M, (int)I, (int)J);
  auto f32 = dy0.options().dtype(at::kFloat);
  at::Tensor partial = at::empty({S, I, J}, f32);
  at::Tensor bpartial = want_bias ? at::empty({S, I}, f32) : at::Tensor();
  hipStream_t stream = current_stream();
  pda::wgrad_gemm_segments(a, dy0.stride(0), b, x0.stride(0), (int)n, partial.data_ptr<float>(),
                           want_bias ? bpartial.data_ptr<float>() : nullptr, (int)rows, (int)I, (int)J, S, stream);
  check_launch("wgrad_gemm_segments");
  at::Tensor dw;
  if (out.has_value()) {
    dw = *out;
    TORCH_CHECK(dw.is_cuda() && dw.is_contiguous() && dw.numel() == I * J &&
                    (dw.scalar_type() == at::kBFloat16 || dw.scalar_type() == at::kFloat),
                "wgrad segments: out must be a contiguous bf16/fp32 GPU tensor with ", I * J, " elements");
  } else {
    TORCH_CHECK(!accumulate, "wgrad segments: accumulate needs an out tensor");
    dw = at::empty({I, J}, dy0.options());
  }
  at::Tensor db;
  if (want_bias) {
    if (bias_out.has_value() && bias_out->defined()) {
      db = *bias_out;
      TORCH_CHECK(db.is_cuda() && db.is_contiguous() && db.numel() == I &&
                      (db.scalar_type() == at::kBFloat16 || db.scalar_type() == at::kFloat),
                  "wgrad segments: bias_out must be a contiguous bf16/fp32 GPU tensor with ", I, " elements");
    } else {
      TORCH_CHECK(!bias_accumulate, "wgrad segments: bias_accumulate needs a bias_out tensor");
      db = at::empty({I}, dy0.options());
    }
  }
  pda::wgrad_reduce(partial.data_ptr<float>(), S, I * J, I * J, dtype_of(dw), dw.data_ptr(), accumulate,
                    want_bias ? bpartial.data_ptr<float>() : nullptr, I, want_bias ? dtype_of(db) : pda::kBF16,
                    want_bias ? db.data_ptr() : nullptr, want_bias && bias_accumulate, stream);
  check_launch("wgrad_reduce");
  return {dw, db};
}

// -------------------------------------------------------- 8-bit floating point --
// (e4m3 values with a scale byte e + 127 per block of 128; layouts in kernels/pda_kernels.h)
int64_t round_up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }

struct Fp8Pair {
  at::Tensor q, scale;
};

// A quantised matrix of `rows` rows of `cols` values by address.
struct Fp8Buffer {
  uint8_t *q = nullptr, *scale = nullptr;
  int64_t rows = 0, cols = 0;
  bool tiles = false;
  int64_t ld() const { return round_up(cols, 128); }
  int64_t ld_scale() const { return round_up((cols + 127) / 128, 4); }
  int64_t scale_rows() const { return tiles ? (rows + 127) / 128 : rows; }
  pda::Fp8Operand operand() const { return pda::Fp8Operand{q, scale, ld(), ld_scale(), (int)rows, tiles}; }
};

// One allocation for what a call needs only until its kernels have run.
struct Scratch {
  size_t size = 0;
  at::Tensor memory;
  std::vector<std::pair<uint8_t**, size_t>> wanted;
  void want(uint8_t** p, int64_t bytes) {
    wanted.emplace_back(p, size);
    size += (size_t)round_up(bytes, 256);
  }
  Fp8Buffer& want(Fp8Buffer& b, int64_t rows, int64_t cols, bool tiles) {
    b.rows = rows, b.cols = cols, b.tiles = tiles;
    want(&b.q, rows * b.ld());
    want(&b.scale, b.scale_rows() * b.ld_scale());
    return b;
  }
  void allocate(const at::TensorOptions& options) {
    memory = at::empty({(int64_t)size}, options.dtype(at::kByte));
    for (auto& [p, at] : wanted) *p = memory.data_ptr<uint8_t>() + at;
  }
};

// A bf16 / fp32 GPU matrix whose rows are contiguous (any row pitch).
void check_fp8_source(const at::Tensor& x, const char* name) {
  TORCH_CHECK(x.is_cuda(), "fp8: ", name, " must live on the GPU");
  TORCH_CHECK(x.dim() == 2, "fp8: ", name, " must be a matrix, got ", x.dim(), " dimensions");
  (void)dtype_of(x);
  TORCH_CHECK(x.numel() == 0 || x.size(1) == 1 || x.stride(1) == 1, "fp8: rows of ", name, " must be contiguous");
  TORCH_CHECK(x.numel() == 0 || x.size(0) == 1 || x.stride(0) >= x.size(1), "fp8: rows of ", name, " must not overlap");
  TORCH_CHECK(x.size(0) <= (1 << 22) && x.size(1) <= (1 << 22), "fp8: ", name, " is larger than 2^22 rows or columns");
  TORCH_CHECK(((x.size(0) + 127) / 128) * ((x.size(1) + 127) / 128) < (1 << 29), "fp8: ", name, " has too many tiles");
}

// `x` [..., C] as a matrix [rows, C] that check_fp8_source accepts, copied only if it has to be.
at::Tensor fp8_source(const at::Tensor& x) {
  int64_t rows = 1;
  for (int64_t i = 0; i + 1 < x.dim(); ++i) rows *= x.size(i);
  at::Tensor m = x.dim() == 2 ? x : x.reshape({rows, x.size(-1)});
  const bool ok = (m.size(1) <= 1 || m.stride(1) == 1) && (m.size(0) <= 1 || m.stride(0) >= m.size(1));
  return ok ? m : m.contiguous();
}

// Matrices to be quantised in one launch.
struct Fp8Quantizer {
  pda::Fp8QuantProblem problems[3];
  int n = 0;
  pda::DType dtype = pda::kBF16;

  // x [R, C] by rows and / or columns, or by tiles (then both layouts share the scales); an output that is not
  // wanted is null. `sums`: fp32 [ceil(R / 128), C] partial column sums (not with tiles).
  void add(const at::Tensor& x, bool tiles, const Fp8Buffer* rows, const Fp8Buffer* cols, float* sums) {
    const int64_t R = x.size(0), C = x.size(1);
    if (R == 0 || C == 0) return;  // every output is empty
    dtype = dtype_of(x);
    problems[n++] = {x.data_ptr(), R > 1 ? x.stride(0) : C, (int)R, (int)C, tiles, rows ? rows->q : nullptr,
                     rows ? rows->scale : nullptr, cols ? cols->q : nullptr, cols ? cols->scale : nullptr, sums};
  }
  void run() {
    if (n == 0) return;
    pda::fp8_quantize(dtype, problems, n, current_stream());
    check_launch("fp8_quantize");
  }
};

// Tensors for a quantised matrix, and where they are.
Fp8Pair fp8_pair(int64_t rows, int64_t cols, bool tiles, const at::TensorOptions& options, Fp8Buffer* at) {
  *at = Fp8Buffer{nullptr, nullptr, rows, cols, tiles};
  Fp8Pair p{at::empty({rows, at->ld()}, options.dtype(at::kFloat8_e4m3fn)), at::empty({at->scale_rows(), at->ld_scale()}, options.dtype(at::kByte))};
  at->q = reinterpret_cast<uint8_t*>(p.q.data_ptr());
  at->scale = reinterpret_cast<uint8_t*>(p.scale.data_ptr());
  return p;
}

std::vector<at::Tensor> fp8_quantize(const at::Tensor& x, bool want_rows, bool want_cols, bool tiles) {
  check_fp8_source(x, "x");
  TORCH_CHECK(want_rows || want_cols, "fp8_quantize: no output asked for");
  const c10::DeviceGuard guard(x.device());
  Fp8Pair rows, cols;
  Fp8Buffer r, c;
  if (want_rows) rows = fp8_pair(x.size(0), x.size(1), tiles, x.options(), &r);
  if (want_cols) cols = fp8_pair(x.size(1), x.size(0), tiles, x.options(), &c);
  Fp8Quantizer quantizer;
  quantizer.add(x, tiles, want_rows ? &r : nullptr, want_cols ? &c : nullptr, nullptr);
  quantizer.run();
  std::vector<at::Tensor> out;
  if (want_rows) out.insert(out.end(), {rows.q, rows.scale});
  if (want_cols) out.insert(out.end(), {cols.q, cols.scale});
  return out;
}

// Checks a quantised operand with `K` values in a row and describes it to the kernel.
pda::Fp8Operand fp8_operand(const at::Tensor& q, const at::Tensor& scale, bool tiles, int64_t K, const char* name) {
  TORCH_CHECK(q.is_cuda() && scale.is_cuda() && q.device() == scale.device(), "fp8: ", name, " must live on one GPU");
  TORCH_CHECK(q.scalar_type() == at::kFloat8_e4m3fn && scale.scalar_type() == at::kByte, "fp8: ", name,
              " needs float8_e4m3fn values and uint8 scales, got ", q.scalar_type(), " and ", scale.scalar_type());
  TORCH_CHECK(q.dim() == 2 && scale.dim() == 2 && q.is_contiguous() && scale.is_contiguous(), "fp8: ", name,
              " needs contiguous matrices");
  const int64_t Kp = round_up(K, 128), rows = q.size(0);
  TORCH_CHECK(q.size(1) == Kp, "fp8: ", name, " has rows of ", q.size(1), " values, ", Kp, " expected (", K, " padded to 128)");
  TORCH_CHECK(scale.size(0) == (tiles ? (rows + 127) / 128 : rows) && scale.size(1) == round_up(Kp / 128, 4), "fp8: ", name,
              " has scales ", scale.sizes(), ", expected [", tiles ? (rows + 127) / 128 : rows, ", ", round_up(Kp / 128, 4), "]");
  TORCH_CHECK(rows <= (1 << 22) && Kp <= (1 << 22), "fp8: ", name, " is larger than 2^22 rows or columns");
  TORCH_CHECK(reinterpret_cast<uintptr_t>(q.data_ptr()) % 16 == 0 && reinterpret_cast<uintptr_t>(scale.data_ptr()) % 4 == 0,
              "fp8: ", name, " must be 16-byte aligned");
  return pda::Fp8Operand{q.data_ptr(), scale.data_ptr(), Kp, scale.size(1), (int)rows, tiles};
}

// Independent products in one launch, their partial sums (and column sums) folded in another.
struct Fp8Products {
  pda::Fp8GemmProblem problems[2];
  int n = 0;
  at::TensorOptions partial_options;

  // out[M, N] = (out +) bias + x . w^T over K; `out` fresh in `dtype` unless given.
  at::Tensor add(const pda::Fp8Operand& X, const pda::Fp8Operand& W, int64_t K, const std::optional<at::Tensor>& bias,
                 const at::TensorOptions& options, const std::optional<at::Tensor>& out, bool accumulate) {
    const int64_t M = X.rows, N = W.rows;
    at::Tensor y;
    if (out.has_value()) {
      y = *out;
      TORCH_CHECK(y.device() == options.device() && y.is_contiguous() && y.numel() == M * N, "fp8_matmul: out must be a contiguous tensor with ",
                  M * N, " elements on the operands' device");
    } else {
      TORCH_CHECK(!accumulate, "fp8_matmul: accumulate needs an out tensor");
      y = at::empty({M, N}, options);
    }
    const pda::DType out_dtype = dtype_of(y);
    if (bias.has_value())
      TORCH_CHECK(bias->device() == options.device() && bias->is_contiguous() && bias->numel() == N, "fp8_matmul: bias must be a contiguous tensor with ",
                  N, " elements on the operands' device");
    const pda::DType bias_dtype = bias.has_value() ? dtype_of(*bias) : pda::kBF16;
    if (M == 0 || N == 0) return y;
    if (K == 0) {  // a sum over nothing
      if (!accumulate) y.zero_();
      if (bias.has_value()) y.view({M, N}).add_(*bias);
      return y;
    }
    problems[n++] = {X, W, (int)X.ld, bias.has_value() ? bias->data_ptr() : nullptr, bias_dtype, y.data_ptr(), out_dtype, accumulate, {}, nullptr};
    partial_options = options.dtype(at::kFloat);
    return y;
  }
  void run(const pda::Fp8ColumnSums* sums = nullptr) {
    if (n == 0 && !sums) return;
    at::Tensor partials[2];
    pda::fp8_gemm_plan(problems, n);
    for (int i = 0; i < n; ++i) {
      pda::Fp8GemmProblem& p = problems[i];
      if (p.plan.slices == 1 && !p.accumulate) continue;
      partials[i] = at::empty({p.plan.slices, p.x.rows, p.w.rows}, partial_options);
      p.partial = partials[i].data_ptr<float>();
    }
    pda::fp8_gemm(problems, n, sums, current_stream());
    check_launch("fp8_gemm");
  }
};

at::Tensor fp8_matmul(const at::Tensor& xq, const at::Tensor& xs, bool x_tiles, const at::Tensor& wq, const at::Tensor& ws,
                      bool w_tiles, int64_t K, const std::optional<at::Tensor>& bias, bool out_f32) {
  TORCH_CHECK(xq.is_cuda(), "fp8_matmul: operands must live on the GPU");
  const c10::DeviceGuard guard(xq.device());
  const pda::Fp8Operand X = fp8_operand(xq, xs, x_tiles, K, "the left operand");
  const pda::Fp8Operand W = fp8_operand(wq, ws, w_tiles, K, "the right operand");
  TORCH_CHECK(xq.device() == wq.device(), "fp8_matmul: operands on different devices");
  Fp8Products products;
  at::Tensor y = products.add(X, W, K, bias, xq.options().dtype(out_f32 ? at::kFloat : at::kBFloat16), std::nullopt, false);
  products.run();
  return y;
}

// What the products of one call (at most two) are planned as: {tile, slices} each, for {M, N, K, fp32 result, accumulate}.
std::vector<std::vector<int64_t>> fp8_plan(const std::vector<std::vector<int64_t>>& products) {
  TORCH_CHECK(products.size() <= 2, "fp8_plan: at most two products share a call, got ", products.size());
  pda::Fp8GemmProblem problems[2] = {};
  for (size_t i = 0; i < products.size(); ++i) {
    const auto& p = products[i];
    TORCH_CHECK(p.size() == 5 && p[0] >= 1 && p[1] >= 1 && p[2] >= 1 && p[0] <= (1 << 22) && p[1] <= (1 << 22) && p[2] <= (1 << 22),
                "fp8_plan: a product is {M, N, K, fp32, accumulate} with sizes between 1 and 2^22");
    problems[i].x.rows = (int)p[0];
    problems[i].w.rows = (int)p[1];
    problems[i].K = (int)round_up(p[2], 128);
    problems[i].out_dtype = p[3] ? pda::kF32 : pda::kBF16;
    problems[i].accumulate = p[4] != 0;
  }
  pda::fp8_gemm_plan(problems, (int)products.size());
  std::vector<std::vector<int64_t>> plans;
  for (size_t i = 0; i < products.size(); ++i) plans.push_back({problems[i].plan.tile, problems[i].plan.slices});
  return plans;
}

// y = x . w^T + bias with x [..., K] quantised by rows and w [N, K] by tiles. `keep`: also x quantised by
// columns (from the same read of x), which is all that the weight gradient needs of it.
std::vector<at::Tensor> fp8_linear_forward(const at::Tensor& x, const at::Tensor& weight, const std::optional<at::Tensor>& bias,
                                           bool keep) {
  const at::Tensor x2 = fp8_source(x), w2 = fp8_source(weight);
  check_fp8_source(x2, "x");
  check_fp8_source(w2, "weight");
  TORCH_CHECK(x2.scalar_type() == w2.scalar_type() && x2.device() == w2.device() && x2.size(1) == w2.size(1), "fp8_linear: x ",
              x.sizes(), " ", x.scalar_type(), " and weight ", weight.sizes(), " ", weight.scalar_type(), " do not match");
  const c10::DeviceGuard guard(x.device());
  const int64_t M = x2.size(0), K = x2.size(1), N = w2.size(0);
  Fp8Pair kept;
  Fp8Buffer xr, xc, wr;
  Scratch scratch;
  scratch.want(xr, M, K, false);
  scratch.want(wr, N, K, true);
  scratch.allocate(x.options());
  if (keep) kept = fp8_pair(K, M, false, x.options(), &xc);
  Fp8Quantizer quantizer;
  quantizer.add(x2, false, &xr, keep ? &xc : nullptr, nullptr);
  quantizer.add(w2, true, &wr, nullptr, nullptr);
  quantizer.run();
  Fp8Products products;
  std::optional<at::Tensor> b;
  if (bias.has_value()) b = bias->contiguous();
  // allocated in its final shape, not returned as a view: a following op may work on it in place (the rotary one does)
  std::vector<int64_t> shape(x.sizes().begin(), x.sizes().end());
  shape.back() = weight.size(0);
  at::Tensor y = at::empty(shape, x.options());
  products.add(xr.operand(), wr.operand(), K, b, x.options(), y, false);
  products.run();
  if (keep) return {y, kept.q, kept.scale};
  return {y};
}

// Gradients of that: dx = dy . w (dy by rows, w by tiles), dw = dy^T . x (both by columns), db = column sums of
// dy before quantisation. xq / xs: x by columns (fp8_linear_forward's `keep`), or `x` itself, quantised here.
// dx has dy's leading dimensions.
std::vector<at::Tensor> fp8_linear_backward(const at::Tensor& dy, const at::Tensor& weight, const std::optional<at::Tensor>& x,
                                            const std::optional<at::Tensor>& xq, const std::optional<at::Tensor>& xs, bool want_x,
                                            bool want_w, bool want_b, const std::optional<at::Tensor>& w_out, bool w_accumulate,
                                            const std::optional<at::Tensor>& b_out, bool b_accumulate) {
  const at::Tensor g2 = fp8_source(dy), w2 = fp8_source(weight);
  check_fp8_source(g2, "dy");
  check_fp8_source(w2, "weight");
  const int64_t M = g2.size(0), N = g2.size(1), K = w2.size(1);
  TORCH_CHECK(dy.scalar_type() == weight.scalar_type() && dy.device() == weight.device() && w2.size(0) == N,
              "fp8_linear backward: dy ", dy.sizes(), " ", dy.scalar_type(), " and weight ", weight.sizes(), " ", weight.scalar_type(), " do not match");
  const c10::DeviceGuard guard(dy.device());
  at::Tensor dx, dw, db, x2;
  const bool rows = want_x || !want_w;  // (the bias gradient alone still needs the pass: rows are the cheaper by-product)
  const bool anew = want_w && x.has_value();
  if (anew) {
    x2 = fp8_source(*x);
    check_fp8_source(x2, "x");
    TORCH_CHECK(x2.size(0) == M && x2.size(1) == K && x2.scalar_type() == dy.scalar_type() && x2.device() == dy.device(),
                "fp8_linear backward: x ", x->sizes(), " does not match dy ", dy.sizes());
  } else if (want_w) {
    TORCH_CHECK(xq.has_value() && xs.has_value(), "fp8_linear backward: the weight gradient needs x");
  }
  Fp8Buffer gr, gc, wc, xc;
  uint8_t* sums = nullptr;
  Scratch scratch;
  if (rows) scratch.want(gr, M, N, false);
  if (want_w) scratch.want(gc, N, M, false);
  if (want_b) scratch.want(&sums, (M + 127) / 128 * N * 4);
  if (want_x) scratch.want(wc, K, N, true);
  if (anew) scratch.want(xc, K, M, false);
  scratch.allocate(dy.options());
  Fp8Quantizer quantizer;
  if (want_x || want_w || want_b) quantizer.add(g2, false, rows ? &gr : nullptr, want_w ? &gc : nullptr, (float*)sums);
  if (want_x) quantizer.add(w2, true, nullptr, &wc, nullptr);
  if (anew) quantizer.add(x2, false, nullptr, &xc, nullptr);
  quantizer.run();
  Fp8Products products;
  if (want_x) {
    dx = products.add(gr.operand(), wc.operand(), N, std::nullopt, dy.options(), std::nullopt, false);
    std::vector<int64_t> shape(dy.sizes().begin(), dy.sizes().end());
    shape.back() = K;
    dx = dx.view(shape);
  }
  if (want_w) {
    const pda::Fp8Operand X = anew ? xc.operand() : fp8_operand(*xq, *xs, false, M, "x");
    TORCH_CHECK(X.rows == K, "fp8_linear backward: x has ", X.rows, " features, ", K, " expected");
    dw = products.add(gc.operand(), X, M, std::nullopt, dy.options(), w_out, w_accumulate);
  }
  pda::Fp8ColumnSums fold{};
  if (want_b) {
    if (b_out.has_value()) {
      db = *b_out;
      TORCH_CHECK(db.device() == dy.device() && db.is_contiguous() && db.numel() == N,
                  "fp8_linear backward: bias_out must be a contiguous tensor with ", N, " elements");
    } else {
      TORCH_CHECK(!b_accumulate, "fp8_linear backward: accumulating the bias gradient needs its tensor");
      db = at::empty({N}, dy.options());
    }
    fold = {(const float*)sums, (int)((M + 127) / 128), (int)N, db.data_ptr(), dtype_of(db), b_accumulate};
  }
  products.run(want_b && N > 0 ? &fold : nullptr);
  return {dx, dw, db};
}

// The layer as one autograd node, for gradients that autograd itself takes (no gradient sink, no recipe for x).
struct Fp8LinearFn : public torch::autograd::Function<Fp8LinearFn> {
  static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& x, const at::Tensor& weight,
                            const std::optional<at::Tensor>& bias, bool keep) {
    std::vector<at::Tensor> got = fp8_linear_forward(x, weight, bias, keep);
    if (keep) ctx->save_for_backward({weight, got[1], got[2]});
    else ctx->save_for_backward({weight});
    ctx->saved_data["bias"] = bias.has_value();
    return got[0];
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    TORCH_CHECK(!at::GradMode::is_enabled(), "fp8_linear has no second derivative (create_graph=True)");
    const auto saved = ctx->get_saved_variables();
    const bool keep = saved.size() == 3;
    const bool want_b = ctx->saved_data["bias"].toBool() && ctx->needs_input_grad(2);
    std::optional<at::Tensor> xq, xs;
    if (keep) xq = saved[1], xs = saved[2];
    auto got = fp8_linear_backward(grads[0], saved[0], std::nullopt, xq, xs, ctx->needs_input_grad(0), keep && ctx->needs_input_grad(1),
                                   want_b, std::nullopt, false, std::nullopt, false);
    return {got[0], got[1], got[2], at::Tensor()};
  }
};

at::Tensor fp8_linear(const at::Tensor& x, const at::Tensor& weight, const std::optional<at::Tensor>& bias) {
  return Fp8LinearFn::apply(x, weight, bias, at::GradMode::is_enabled() && weight.requires_grad());
}

}  // namespace

// ------------------------------------------------------- fused-epilogue GEMM --
void check_bf16_matrix(const at::Tensor& t, const char* name) {
  TORCH_CHECK(t.defined() && t.is_cuda() && t.scalar_type() == at::kBFloat16, name, " must be a bf16 GPU tensor");
  TORCH_CHECK(t.dim() == 2 && t.stride(1) == 1 && t.stride(0) >= t.size(1) && t.stride(0) % 8 == 0, name,
              " must be a row-major matrix with unit column stride and a row stride that is a multiple of 8");
  TORCH_CHECK(reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0, name, " must be 16-byte aligned");
}

bool gemm_fused_supported(int64_t M, int64_t N, int64_t K) {
  return M < (int64_t(1) << 31) && N < (int64_t(1) << 31) && pda::gemm_fused_supported((int)M, (int)N, (int)K);
}

// epilogue: "none" | "bias" | "bias_gelu" (returns [u, gelu(u)]) | "mul_gelu_grad" (aux = u, returns [acc * gelu'(u)]).
std::vector<at::Tensor> gemm_fused(const at::Tensor& x, const at::Tensor& w, const std::optional<at::Tensor>& bias,
                                   const std::string& epilogue, const std::optional<at::Tensor>& aux) {
  check_bf16_matrix(x, "x");
  check_bf16_matrix(w, "w");
  const c10::DeviceGuard guard(x.device());
  const int64_t M = x.size(0), K = x.size(1), N = w.size(0);
  TORCH_CHECK(w.size(1) == K, "gemm_fused: x is [M, K], w must be [N, K]");
  TORCH_CHECK(gemm_fused_supported(M, N, K), "gemm_fused: unsupported shape M=", M, " N=", N, " K=", K,
              " (needs K % 32 == 0 and N % 8 == 0)");
  int epi = pda::kEpiNone;
  if (epilogue == "bias") epi = pda::kEpiBias;
  else if (epilogue == "bias_gelu") epi = pda::kEpiBiasGelu;
  else if (epilogue == "mul_gelu_grad") epi = pda::kEpiMulGeluGrad;
  else TORCH_CHECK(epilogue == "none", "gemm_fused: unknown epilogue '", epilogue, "'");
  const void* bias_ptr = nullptr;
  if (epi == pda::kEpiBias || epi == pda::kEpiBiasGelu) {
    TORCH_CHECK(bias.has_value() && bias->is_cuda() && bias->scalar_type() == at::kBFloat16 && bias->is_contiguous() &&
                    bias->numel() == N && reinterpret_cast<uintptr_t>(bias->data_ptr()) % 8 == 0,
                "gemm_fused: bias must be a contiguous, 8-byte aligned bf16 GPU vector of length ", N);
    bias_ptr = bias->data_ptr();
  }
  at::Tensor out = at::empty({M, N}, x.options());
  std::vector<at::Tensor> result{out};
  void* aux_ptr = nullptr;
  int64_t ldaux = N;
  if (epi == pda::kEpiBiasGelu) {
    at::Tensor act = at::empty({M, N}, x.options());
    aux_ptr = act.data_ptr();
    result.push_back(act);
  } else if (epi == pda::kEpiMulGeluGrad) {
    TORCH_CHECK(aux.has_value(), "gemm_fused: 'mul_gelu_grad' needs the pre-activation as aux");
    check_bf16_matrix(*aux, "aux");
    TORCH_CHECK(aux->size(0) == M && aux->size(1) == N, "gemm_fused: aux must be [M, N]");
    aux_ptr = aux->data_ptr();
    ldaux = aux->stride(0);
  }
  pda::gemm_fused(x.data_ptr(), x.stride(0), w.data_ptr(), w.stride(0), bias_ptr, out.data_ptr(), N, aux_ptr, ldaux, (int)M,
                  (int)N, (int)K, epi, current_stream());
  check_launch("gemm_fused");
  return result;
}

// -------------------------------------------------------------- embedding --
at::Tensor embedding_forward(const at::Tensor& ids, const at::Tensor& wte, const std::optional<at::Tensor>& wpe) {
  check_gpu(wte, "wte");
  TORCH_CHECK(ids.is_cuda() && ids.is_contiguous() && ids.scalar_type() == at::kLong, "embedding: ids must be a contiguous int64 GPU tensor");
  TORCH_CHECK(ids.dim() == 2 && wte.dim() == 2, "embedding: ids [B, T], wte [V, d]");
  const c10::DeviceGuard guard(wte.device());
  const auto dt = dtype_of(wte);
  const int64_t d = wte.size(1), T = ids.size(1);
  TORCH_CHECK(d % (dt == pda::kBF16 ? 8 : 4) == 0, "embedding: row length ", d, " is not a multiple of the 16-byte vector");
  TORCH_CHECK(wte.size(0) < (int64_t(1) << 31) && ids.numel() < (int64_t(1) << 31), "embedding: table or batch too large");
  const void* wpe_ptr = nullptr;
  if (wpe.has_value()) {
    check_gpu(*wpe, "wpe");
    TORCH_CHECK(wpe->dim() == 2 && wpe->size(1) == d && wpe->size(0) >= T && wpe->scalar_type() == wte.scalar_type(),
                "embedding: wpe must be [>= T, d] in the dtype of wte");
    wpe_ptr = wpe->data_ptr();
  }
  at::Tensor out = at::empty({ids.size(0), T, d}, wte.options());
  pda::embedding_forward(dt, ids.data_ptr<int64_t>(), wte.data_ptr(), wpe_ptr, out.data_ptr(), ids.numel(), (int)T, (int)d,
                         (int)wte.size(0), current_stream());
  check_launch("embedding_forward");
  return out;
}

// Gradients of embedding_forward. dwte_out / dwpe_out (optional): existing gradient buffers to
// write (accumulate = false) or add into (accumulate = true); without them fresh tensors are
// returned (dwte zero-initialised, then the rows of occurring tokens written).
std::vector<at::Tensor> embedding_backward(const at::Tensor& ids, const at::Tensor& dout, int64_t vocab, bool need_wpe,
                                           int64_t wpe_rows, const std::optional<at::Tensor>& dwte_out, bool wte_accumulate,
                                           const std::optional<at::Tensor>& dwpe_out, bool wpe_accumulate) {
  check_gpu(dout, "dout");
  TORCH_CHECK(ids.is_cuda() && ids.is_contiguous() && ids.scalar_type() == at::kLong && ids.dim() == 2,
              "embedding: ids must be a contiguous int64 [B, T] GPU tensor");
  const c10::DeviceGuard guard(dout.device());
  const auto dt = dtype_of(dout);
  const int64_t B = ids.size(0), T = ids.size(1), d = dout.size(-1);
  TORCH_CHECK(dout.numel() == B * T * d, "embedding: dout must be [B, T, d]");
  TORCH_CHECK(d % (dt == pda::kBF16 ? 8 : 4) == 0, "embedding: bad row length ", d);
  TORCH_CHECK(vocab > 0 && vocab < (int64_t(1) << 31) && B * T < (int64_t(1) << 31), "embedding: table or batch too large");
  at::Tensor dwte;
  bool acc_w = false;
  if (dwte_out.has_value()) {
    dwte = *dwte_out;
    check_gpu(dwte, "dwte_out");
    TORCH_CHECK(dwte.scalar_type() == dout.scalar_type() && dwte.numel() == vocab * d, "embedding: dwte_out must be [V, d] in dout's dtype");
    acc_w = wte_accumulate;
    if (!acc_w) dwte.zero_();
  } else {
    dwte = at::zeros({vocab, d}, dout.options());
  }
  const size_t ws_bytes = pda::embedding_backward_workspace_bytes((int)(B * T), (int)vocab);
  at::Tensor ws = at::empty({(int64_t)ws_bytes}, dout.options().dtype(at::kByte));
  pda::embedding_backward_wte(dt, ids.data_ptr<int64_t>(), dout.data_ptr(), dwte.data_ptr(), acc_w, (int)(B * T), (int)d,
                              (int)vocab, ws.data_ptr(), ws_bytes, current_stream());
  check_launch("embedding_backward_wte");
  std::vector<at::Tensor> result{dwte};
  if (need_wpe) {
    TORCH_CHECK(wpe_rows >= T, "embedding: position table shorter than the sequence");
    at::Tensor dwpe;
    bool acc_p = false;
    if (dwpe_out.has_value()) {
      dwpe = *dwpe_out;
      check_gpu(dwpe, "dwpe_out");
      TORCH_CHECK(dwpe.scalar_type() == dout.scalar_type() && dwpe.numel() == wpe_rows * d, "embedding: dwpe_out must be [n_ctx, d]");
      acc_p = wpe_accumulate;
      if (!acc_p && wpe_rows > T) dwpe.narrow(0, T, wpe_rows - T).zero_();
    } else {
      dwpe = wpe_rows > T ? at::zeros({wpe_rows, d}, dout.options()) : at::empty({wpe_rows, d}, dout.options());
    }
    pda::embedding_backward_wpe(dt, dout.data_ptr(), dwpe.data_ptr(), acc_p, (int)B, (int)T, (int)d, current_stream());
    check_launch("embedding_backward_wpe");
    result.push_back(dwpe);
  }
  return result;
}

void bind_ops(py::module_& m) {
  m.def("gemm_fused_supported", &gemm_fused_supported);
  m.def("gemm_fused", &gemm_fused, py::arg("x"), py::arg("w"), py::arg("bias") = py::none(), py::arg("epilogue") = "none",
        py::arg("aux") = py::none());
  m.def("embedding_forward", &embedding_forward, py::arg("ids"), py::arg("wte"), py::arg("wpe") = py::none());
  m.def("embedding_backward", &embedding_backward, py::arg("ids"), py::arg("dout"), py::arg("vocab"), py::arg("need_wpe"),
        py::arg("wpe_rows") = 0, py::arg("dwte_out") = py::none(), py::arg("wte_accumulate") = false,
        py::arg("dwpe_out") = py::none(), py::arg("wpe_accumulate") = false);
  m.def("rope_apply", &rope_apply, py::arg("qkv"), py::arg("cos"), py::arg("sin"), py::arg("num_heads"),
        py::arg("inverse"), py::arg("in_place"));
  m.def("transpose_2d", &transpose_2d, py::arg("src"), py::arg("pad_rows_to") = 8);
  m.def("wgrad_supported", &wgrad_supported);
  m.def("linear_wgrad", &linear_wgrad, py::arg("dy"), py::arg("x"), py::arg("want_bias"),
        py::arg("out") = py::none(), py::arg("accumulate") = false, py::arg("bias_out") = py::none(),
        py::arg("bias_accumulate") = false, py::arg("out_rows") = -1);
  m.def("wgrad_segments_supported", &wgrad_segments_supported, py::arg("rows"), py::arg("I"), py::arg("J"), py::arg("n"));
  m.def("wgrad_max_segments", []() { return pda::wgrad_max_segments(); });
  m.def("linear_wgrad_segments", &linear_wgrad_segments, py::arg("dys"), py::arg("xs"), py::arg("want_bias"),
        py::arg("out") = py::none(), py::arg("accumulate") = false, py::arg("bias_out") = py::none(),
        py::arg("bias_accumulate") = false);
  m.def("norm_forward", &norm_forward, py::arg("x"), py::arg("residual"), py::arg("weight"),
        py::arg("bias"), py::arg("eps"), py::arg("rms"), py::arg("dropout_p") = 0.0, py::arg("seed") = 0);
  m.def("norm_backward", &norm_backward, py::arg("dy"), py::arg("x"), py::arg("weight"), py::arg("mean"),
        py::arg("rstd"), py::arg("dresidual"), py::arg("rms"), py::arg("dweight_out") = py::none(),
        py::arg("accumulate_w") = false, py::arg("dbias_out") = py::none(), py::arg("accumulate_b") = false,
        py::arg("dropout_p") = 0.0, py::arg("seed") = 0);
  m.def("gelu_forward", &gelu_forward);
  m.def("gelu_backward", &gelu_backward);
  m.def("swiglu_forward", &swiglu_forward);
  m.def("swiglu_backward", &swiglu_backward);
  m.def("cross_entropy_fwd_bwd", &cross_entropy_fwd_bwd, py::arg("logits"), py::arg("targets"),
        py::arg("vocab"), py::arg("grad_scale"), py::arg("ignore_index"));
  m.def("adamw_step", &adamw_step, py::arg("params"), py::arg("lowp"), py::arg("grads"),
        py::arg("exp_avg"), py::arg("exp_avg_sq"), py::arg("lr"), py::arg("beta1"), py::arg("beta2"),
        py::arg("eps"), py::arg("weight_decay"), py::arg("step"), py::arg("grad_scale"),
        py::arg("zero_grad"), py::arg("dynamic") = py::none());
  m.def("accumulate_bf16_into_f32", &accumulate_bf16_into_f32);
  m.def("fp8_quantize", &fp8_quantize, py::arg("x"), py::arg("rows"), py::arg("columns"), py::arg("tiles"));
  m.def("fp8_matmul", &fp8_matmul, py::arg("xq"), py::arg("xs"), py::arg("x_tiles"), py::arg("wq"), py::arg("ws"),
        py::arg("w_tiles"), py::arg("K"), py::arg("bias"), py::arg("out_f32"));
  m.def("fp8_plan", &fp8_plan, py::arg("products"));
  m.def("fp8_linear", &fp8_linear, py::arg("x"), py::arg("weight"), py::arg("bias"));
  m.def("fp8_linear_forward", &fp8_linear_forward, py::arg("x"), py::arg("weight"), py::arg("bias"), py::arg("keep"));
  m.def("fp8_linear_backward", &fp8_linear_backward, py::arg("dy"), py::arg("weight"), py::arg("x"), py::arg("xq"), py::arg("xs"),
        py::arg("want_x"), py::arg("want_w"), py::arg("want_b"), py::arg("w_out"), py::arg("w_accumulate"), py::arg("b_out"),
        py::arg("b_accumulate"));
  m.def("attention_forward", &attention_forward, py::arg("qkv"), py::arg("num_heads"),
        py::arg("softmax_scale"), py::arg("dropout_p") = 0.0, py::arg("seed") = 0);
  m.def("attention_backward", &attention_backward, py::arg("qkv"), py::arg("out"), py::arg("dout"),
        py::arg("lse"), py::arg("num_heads"), py::arg("softmax_scale"), py::arg("dropout_p") = 0.0,
        py::arg("seed") = 0);
  m.def("window_attention", &window_attention, py::arg("qkv"), py::arg("num_heads"), py::arg("window"), py::arg("sinks"),
        py::arg("softmax_scale"), py::arg("dropout_p"), py::arg("seed"));
  m.def("window_attention_forward", &window_attention_forward, py::arg("qkv"), py::arg("num_heads"), py::arg("window"),
        py::arg("sinks"), py::arg("softmax_scale"), py::arg("dropout_p"), py::arg("seed"), py::arg("for_backward") = false);
  m.def("window_attention_backward", &window_attention_backward, py::arg("qkv"), py::arg("out"), py::arg("out_rest"),
        py::arg("dout"), py::arg("neg_lse"),
        py::arg("num_heads"), py::arg("window"), py::arg("sinks"), py::arg("softmax_scale"), py::arg("dropout_p"), py::arg("seed"));
  m.def("attention_dropout_mask", &attention_dropout_mask, py::arg("B"), py::arg("H"), py::arg("T"),
        py::arg("dropout_p"), py::arg("seed"), py::arg("device"));
}
