// The classification tail and the optimizers of the training scripts
// (reference tests/gcn/graphcuda_impl.py:24,45,55-56,63-68).
#include <torch/csrc/autograd/custom_function.h>

#include <vector>

#include "host.h"

namespace gch {

namespace {
// One byte per row, non-zero where the row counts; bool and uint8 selections are used as they are.
Tensor bytes_of(const Tensor& m) {
  if (m.scalar_type() == at::kBool || m.scalar_type() == at::kByte) return m.contiguous();
  return m.to(at::kByte).contiguous();
}
}  // namespace

NllForward nll_forward(const Tensor& Zin, const Tensor& labels, const OptTensor& row_mask, double scale) {
  require(Zin.dim() == 2 && Zin.is_cuda() && Zin.scalar_type() == at::kFloat, "logits must be a float32 CUDA matrix");
  require(labels.device() == Zin.device() && labels.scalar_type() == at::kLong && labels.numel() == Zin.size(0),
          "labels must be a CUDA int64 vector with one entry per row, on the logits' device");
  NllForward f;
  f.masked = row_mask && row_mask->defined();
  Tensor mask8;
  if (f.masked) {
    require(row_mask->device() == Zin.device() && row_mask->numel() == Zin.size(0),
            "row_mask must have one entry per row, on the logits' device");
    mask8 = bytes_of(*row_mask);
  }
  f.Z = Zin.stride(1) == 1 ? Zin : Zin.contiguous();
  f.labels = labels.contiguous();
  const int64_t M = f.Z.size(0), C = f.Z.size(1);
  const at::Device dev = f.Z.device();
  const c10::cuda::CUDAGuard guard(dev);
  const size_t wsb = std::max<size_t>(abi.gc_nll_workspace_bytes(M), 4);
  f.ws = at::empty({int64_t(wsb)}, at::TensorOptions().dtype(at::kByte).device(dev));
  f.loss = at::empty({}, at::TensorOptions().dtype(at::kFloat).device(dev));
  check(abi.gc_logsoftmax_nll_forward_f32(
            f.Z.const_data_ptr<float>(), M > 1 ? f.Z.stride(0) : std::max<int64_t>(C, 1),
            f.labels.const_data_ptr<int64_t>(), f.masked ? static_cast<const uint8_t*>(mask8.data_ptr()) : nullptr, M, C,
            float(scale), f.loss.data_ptr<float>(), f.ws.data_ptr(), wsb, stream_of(dev)),
        "gc_logsoftmax_nll_forward_f32");
  return f;
}

// masked: the rows are those of the forward pass's selection, of which the workspace holds a copy
Tensor nll_backward(const Tensor& grad, const Tensor& Z, const Tensor& labels, const Tensor& ws, bool masked,
                    double scale) {
  const int64_t M = Z.size(0), C = Z.size(1);
  const at::Device dev = Z.device();
  const c10::cuda::CUDAGuard guard(dev);
  const int64_t ldz = M > 1 ? Z.stride(0) : std::max<int64_t>(C, 1);
  int64_t lddz = std::max<int64_t>(C, 1);
  Tensor dZ;
  if (M > 1 && C < ldz && ldz <= C + 3 && ldz % 4 == 0 && reinterpret_cast<uintptr_t>(Z.data_ptr()) % 16 == 0) {
    // The logits are a view of a matrix padded to 16-byte rows (an odd class count): give the gradient the same
    // pitch with zero pad columns, so the layer below can aggregate it without re-padding a copy.
    lddz = ldz;
    Tensor buf = empty_f32(M, ldz, dev);
    register_zero_padded(buf);
    dZ = buf.narrow(1, 0, C);
  } else {
    dZ = empty_f32(M, C, dev);
  }
  const Tensor g = grad.to(at::kFloat).contiguous();
  const uint8_t* mask =
      masked ? static_cast<const uint8_t*>(ws.data_ptr()) + abi.gc_nll_workspace_bytes(M) - M : nullptr;
  check((lddz == C ? abi.gc_logsoftmax_nll_backward_f32 : abi.gc_logsoftmax_nll_backward_pad_f32)(
            Z.const_data_ptr<float>(), ldz, labels.const_data_ptr<int64_t>(), mask, M, C, float(scale),
            g.const_data_ptr<float>(), dZ.data_ptr<float>(), lddz, ws.data_ptr(), stream_of(dev)),
        "gc_logsoftmax_nll_backward_f32");
  return dZ;
}

namespace {
struct NllFunction : torch::autograd::Function<NllFunction> {
  static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& Z, const Tensor& labels,
                        const OptTensor& row_mask, double scale) {
    const NllForward f = nll_forward(Z, labels, row_mask, scale);
    ctx->save_for_backward({f.Z, f.labels, f.ws});
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["masked"] = f.masked;
    return f.loss;
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    return {nll_backward(grads[0], saved[0], saved[1], saved[2], ctx->saved_data["masked"].toBool(),
                         ctx->saved_data["scale"].toDouble()),
            Tensor(), Tensor(), Tensor()};
  }
};

}  // namespace

Tensor nll_loss(const Tensor& Z, const Tensor& labels, const OptTensor& row_mask, double scale) {
  return NllFunction::apply(Z, labels, row_mask, scale);
}

// ------------------------------------------------------------------ distillation
namespace {
bool f32_or_bf16(const Tensor& t) { return t.scalar_type() == at::kFloat || t.scalar_type() == at::kBFloat16; }
int type_of(const Tensor& t) { return t.scalar_type() == at::kFloat ? GC_TYPE_F32 : GC_TYPE_BF16; }
int bits_of(const Tensor& index) { return index.scalar_type() == at::kLong ? 64 : 32; }
// The gradient's buffer.  Its rows start as many bytes behind a 16-byte boundary as the logits' own, so that both go in vectors.  Where
// the logits are a view of a matrix padded to 16-byte rows (an odd class count), its `pad` columns become zero, so that the layer below
// can aggregate it without re-padding a copy (as in nll_backward).
struct GradientRows {
  int64_t ld, pad;
};
GradientRows gradient_rows(const Tensor& Z) {
  const int64_t C = Z.size(1), ldz = ld_of(Z), vec = 16 / Z.element_size();
  GradientRows g{C + (ldz - C) % vec, 0};
  if (Z.size(0) > 1 && C < g.ld && ldz == g.ld && g.ld % 4 == 0 && g.ld <= C + 3 && Z.scalar_type() == at::kFloat &&
      reinterpret_cast<uintptr_t>(Z.data_ptr()) % 16 == 0)
    g.pad = g.ld - C;
  return g;
}
}  // namespace

DistillForward distill_forward(const Tensor& Zin, const Tensor& top, const Tensor& index, const OptTensor& row_mask,
                               double temperature, double scale, bool want_gradient) {
  require(Zin.dim() == 2 && Zin.is_cuda() && f32_or_bf16(Zin), "distill_loss: logits must be a float32 or bfloat16 CUDA matrix");
  const at::Device dev = Zin.device();
  const int64_t M = Zin.size(0), C = Zin.size(1);
  require(C >= 1, "distill_loss: logits have no classes");
  require(top.dim() == 2 && top.device() == dev && f32_or_bf16(top) && top.size(0) == M,
          "distill_loss: top_logits must be a float32 or bfloat16 matrix with a row per row of the logits, on their device");
  require(index.device() == dev && (index.scalar_type() == at::kLong || index.scalar_type() == at::kInt) &&
              index.sizes() == top.sizes(),
          "distill_loss: top_index must be int64 or int32 of top_logits' shape, on its device");
  require(top.size(1) <= 1024, "distill_loss: at most 1024 entries to a row");
  Tensor mask8;
  if (row_mask && row_mask->defined()) {
    require(row_mask->device() == dev && row_mask->numel() == M,
            "distill_loss: row_mask must have one entry per row, on the logits' device");
    require(row_mask->scalar_type() == at::kBool || row_mask->scalar_type() == at::kByte,
            "distill_loss: row_mask must be bool or uint8");
    mask8 = row_mask->contiguous();
  }
  const c10::cuda::CUDAGuard guard(dev);
  DistillForward f;
  f.Z = row_major(Zin);
  f.top = row_major(top);
  f.index = row_major(index);
  const auto f32 = at::TensorOptions().dtype(at::kFloat).device(dev);
  f.stats = at::empty({M, 4}, f32);
  f.loss = at::empty({}, f32);
  GradientRows rows{C, 0};
  if (want_gradient) {
    rows = gradient_rows(f.Z);
    f.pad = rows.pad;
    if (abi.gc_distill_one_pass(f.Z.const_data_ptr(), type_of(f.Z), ld_of(f.Z), rows.ld, M, C, top.size(1)))
      f.dz = at::empty({M, rows.ld}, f.Z.options());
  }
  const Scratch ws = scratch(kSpmm, abi.gc_distill_workspace_bytes(M, C), dev);
  check(abi.gc_distill_forward(f.Z.const_data_ptr(), type_of(f.Z), ld_of(f.Z), f.top.const_data_ptr(), type_of(f.top), ld_of(f.top),
                               f.index.const_data_ptr(), bits_of(f.index), ld_of(f.index),
                               mask8.defined() ? static_cast<const uint8_t*>(mask8.data_ptr()) : nullptr, M, C, top.size(1),
                               float(temperature), float(scale), f.loss.data_ptr<float>(), f.stats.data_ptr<float>(),
                               f.dz.defined() ? f.dz.data_ptr() : nullptr, rows.ld, rows.pad, ws.ptr, ws.bytes, stream_of(dev)),
        "gc_distill_forward");
  return f;
}

// dz: the buffer that the forward pass has filled, or undefined; its rows are as they were then (a hook may give Z back with other strides)
Tensor distill_backward(const Tensor& grad, const Tensor& Z, const Tensor& top, const Tensor& index, const Tensor& stats, const Tensor& dz,
                        int64_t dz_pad, double temperature, double scale) {
  const int64_t M = Z.size(0), C = Z.size(1);
  const at::Device dev = Z.device();
  const c10::cuda::CUDAGuard guard(dev);
  const GradientRows rows = dz.defined() ? GradientRows{dz.size(1), dz_pad} : gradient_rows(Z);
  const Tensor buf = dz.defined() ? dz : at::empty({M, rows.ld}, Z.options());
  if (rows.pad) register_zero_padded(buf);
  const Tensor dZ = rows.ld == C ? buf : buf.narrow(1, 0, C);
  const Tensor g = grad.to(at::kFloat).contiguous();
  check(abi.gc_distill_backward(Z.const_data_ptr(), type_of(Z), ld_of(Z), top.const_data_ptr(), type_of(top), ld_of(top),
                                index.const_data_ptr(), bits_of(index), ld_of(index), stats.const_data_ptr<float>(), M, C, top.size(1),
                                float(temperature), float(scale), g.const_data_ptr<float>(), buf.data_ptr(), rows.ld, rows.pad, dz.defined(),
                                stream_of(dev)),
        "gc_distill_backward");
  return dZ;
}

namespace {
// Which capture the current stream takes part in; 0: none.
int64_t recording(const at::Device& dev) {
  cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
  unsigned long long id = 0;
  const cudaError_t e = cudaStreamGetCaptureInfo(static_cast<cudaStream_t>(stream_of(dev)), &status, &id);
  if (e != cudaSuccess) raise(std::string("cudaStreamGetCaptureInfo: ") + cudaGetErrorString(e));
  return status == cudaStreamCaptureStatusActive ? int64_t(id) : 0;
}
struct DistillFunction : torch::autograd::Function<DistillFunction> {
  static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& Z, const Tensor& top, const Tensor& index,
                        const OptTensor& row_mask, double temperature, double scale) {
    const DistillForward f = distill_forward(Z, top, index, row_mask, temperature, scale, true);
    ctx->save_for_backward({f.Z, f.top, f.index, f.stats});
    const int64_t where = f.dz.defined() ? recording(Z.device()) : 0;
    ctx->saved_data["call"] = std::vector<double>{temperature, scale, double(f.pad), double(where)};
    if (f.dz.defined()) ctx->saved_data["dz"] = f.dz;
    return f.loss;
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    once("distill_loss");
    const auto saved = ctx->get_saved_variables();
    const std::vector<double> call = ctx->saved_data["call"].toDoubleVector();
    // Handed out once: whoever differentiates the same graph again may have changed it by then, and gets a buffer of its own.  And only
    // within the recording that has filled it, or outside of all: replayed by itself, a backward pass has to write what it returns.
    Tensor dz;
    const auto made = ctx->saved_data.find("dz");
    if (made != ctx->saved_data.end() && int64_t(call[3]) == recording(saved[0].device())) {
      dz = made->second.toTensor();
      ctx->saved_data.erase(made);
    }
    return {distill_backward(grads[0], saved[0], saved[1], saved[2], saved[3], dz, int64_t(call[2]), call[0], call[1]),
            Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};
}  // namespace

Tensor distill_loss(const Tensor& Z, const Tensor& top, const Tensor& index, const OptTensor& row_mask, double temperature,
                    double scale) {
  if (!recorded({&Z, &top})) return distill_forward(Z, top, index, row_mask, temperature, scale, false).loss;
  return DistillFunction::apply(Z, top, index, row_mask, temperature, scale);
}

// ------------------------------------------------------------------ evaluation
std::pair<Tensor, Tensor> argmax_accuracy(const Tensor& logits, const OptTensor& labels_in,
                                          const std::optional<std::vector<Tensor>>& masks, bool want_pred) {
  require(logits.is_cuda() && logits.dim() == 2 && logits.scalar_type() == at::kFloat,
          "argmax_accuracy: float32 CUDA matrix expected");
  const Tensor Z = (logits.stride(1) == 1 || logits.size(1) == 1) ? logits : logits.contiguous();
  const int64_t M = Z.size(0), C = Z.size(1);
  const at::Device dev = Z.device();
  const c10::cuda::CUDAGuard guard(dev);
  const bool labelled = labels_in && labels_in->defined();
  Tensor labels;
  std::vector<Tensor> rows;
  const uint8_t* list[8] = {};
  if (masks) {
    require(labelled, "argmax_accuracy: masks need labels");
    require(masks->size() >= 1 && masks->size() <= 8, "argmax_accuracy: between 1 and 8 row selections");
    for (const Tensor& m : *masks) {
      require(m.numel() == M && m.device() == dev,
              "argmax_accuracy: every selection needs one entry per row, on the logits' device");
      const bool bytes = m.scalar_type() == at::kBool || m.scalar_type() == at::kByte;
      rows.push_back((bytes ? m : m.ne(0)).contiguous());
      list[rows.size() - 1] = static_cast<const uint8_t*>(rows.back().data_ptr());
    }
  }
  const int n_masks = int(rows.size());
  if (labelled) {
    require(labels_in->scalar_type() == at::kLong && labels_in->numel() == M && labels_in->device() == dev,
            "argmax_accuracy: labels must be int64 [M] on the logits' device");
    labels = labels_in->contiguous();
  }
  Tensor pred, counts;
  const auto i64 = at::TensorOptions().dtype(at::kLong).device(dev);
  if (want_pred) pred = at::empty({M}, i64);
  if (labelled) counts = at::empty({std::max(n_masks, 1), 2}, i64);
  check(abi.gc_argmax_accuracy_masks_f32(Z.const_data_ptr<float>(), M > 1 ? Z.stride(0) : std::max<int64_t>(C, 1), M, C,
                                   labelled ? labels.const_data_ptr<int64_t>() : nullptr,
                                   list, n_masks,
                                   want_pred ? pred.data_ptr<int64_t>() : nullptr,
                                   labelled ? counts.data_ptr<int64_t>() : nullptr, stream_of(dev)),
        "gc_argmax_accuracy_f32");
  return {pred, counts};
}

// ------------------------------------------------------------------ optimizers
namespace {
struct Lists {
  std::vector<float*> p, m, v;
  std::vector<const float*> g;
  std::vector<int64_t> n;
  std::vector<Tensor> keep;
};
Lists lists(const std::vector<Tensor>& p, const std::vector<Tensor>& g) {
  Lists l;
  for (size_t i = 0; i < p.size(); ++i) {
    require(p[i].is_cuda() && p[i].scalar_type() == at::kFloat && p[i].is_contiguous(),
            "fused optimizers need contiguous float32 CUDA parameters");
    require(!g[i].is_sparse() && f32_on(g[i], p[i].device()) && g[i].numel() == p[i].numel(),
            "fused optimizers need dense float32 gradients on the parameter's device");
    require(p[i].device() == p[0].device(), "fused optimizers take the parameters of one device at a time");
    l.keep.push_back(g[i].contiguous());
    l.p.push_back(static_cast<float*>(p[i].data_ptr()));
    l.g.push_back(l.keep.back().const_data_ptr<float>());
    l.n.push_back(p[i].numel());
  }
  return l;
}
}  // namespace

void adam_step(const std::vector<Tensor>& p, const std::vector<Tensor>& g, const std::vector<Tensor>& m,
               const std::vector<Tensor>& v, double lr, double b1, double b2, double eps, double wd,
               const Tensor& state) {
  Lists l = lists(p, g);
  const auto moment = [](const Tensor& t, const Tensor& p) {
    return f32_on(t, p.device()) && t.is_contiguous() && t.numel() == p.numel();
  };
  require(p.empty() || p[0].device() == state.device(), "the optimizer state must be on the parameters' device");
  for (size_t i = 0; i < p.size(); ++i) {
    require(moment(m[i], p[i]) && moment(v[i], p[i]),
            "FusedAdam: exp_avg and exp_avg_sq must be contiguous float32 tensors of the parameter's size on its device");
    l.m.push_back(static_cast<float*>(m[i].data_ptr()));
    l.v.push_back(static_cast<float*>(v[i].data_ptr()));
  }
  const at::Device dev = state.device();
  const c10::cuda::CUDAGuard guard(dev);
  check(abi.gc_adam_step_f32(int(p.size()), l.p.data(), l.g.data(), l.m.data(), l.v.data(), l.n.data(), lr, b1, b2,
                             eps, wd, state.data_ptr(), stream_of(dev)),
        "gc_adam_step_f32");
  for (const auto* list : {&p, &m, &v}) written(*list);
  written(state);
}

void sgd_step(const std::vector<Tensor>& p, const std::vector<Tensor>& g, double lr, double wd) {
  if (p.empty()) return;
  Lists l = lists(p, g);
  const at::Device dev = p[0].device();
  const c10::cuda::CUDAGuard guard(dev);
  check(abi.gc_sgd_step_f32(int(p.size()), l.p.data(), l.g.data(), l.n.data(), lr, wd, stream_of(dev)),
        "gc_sgd_step_f32");
  written(p);
}

}  // namespace gch
