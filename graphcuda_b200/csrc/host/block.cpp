// What stands between the graph layers of a deep model: the norm of the residual stream and the gated feed-forward block, each with its
// autograd node and its 8-bit form, and AdamW over the model's tensors.
#include <torch/csrc/autograd/custom_function.h>

#include <vector>

#include "host.h"

namespace gch {

namespace {
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// GC_TYPE_* of a tensor
int type_of(const Tensor& t) {
  return t.scalar_type() == at::kFloat ? GC_TYPE_F32 : t.scalar_type() == at::kBFloat16 ? GC_TYPE_BF16 : GC_TYPE_E4M3;
}
bool f32_or_bf16(const Tensor& t) { return t.scalar_type() == at::kFloat || t.scalar_type() == at::kBFloat16; }
bool dual(const Tensor& t) { return t._fw_grad(0).defined(); }
Tensor empty_like_rows(int64_t rows, int64_t cols, at::ScalarType type, const at::Device& dev) {
  return at::empty({rows, cols}, at::TensorOptions().dtype(type).device(dev));
}
}  // namespace

bool recorded(std::initializer_list<const Tensor*> inputs) {
  for (const Tensor* t : inputs)
    if (t && t->defined() && ((c10::GradMode::is_enabled() && t->requires_grad()) || dual(*t))) return true;
  return false;
}
void once(const char* what) {
  if (c10::GradMode::is_enabled()) raise(std::string(what) + " has no second derivative (create_graph)");
}

// ------------------------------------------------------------------ norm
NormForward rms_norm_forward(const Tensor& xin, const Tensor& weight, const OptTensor& residual, double eps, int y_type,
                             bool want_rstd) {
  const bool add = residual && residual->defined();
  require(xin.dim() == 2 && xin.is_cuda() && f32_or_bf16(xin), "rms_norm: x must be a float32 or bfloat16 CUDA matrix");
  const at::Device dev = xin.device();
  const int64_t M = xin.size(0), N = xin.size(1);
  require(f32_on(weight, dev) && weight.dim() == 1 && weight.size(0) == N,
          "rms_norm: weight must be a float32 vector of x's width on x's device");
  require(!add || (residual->device() == dev && residual->sizes() == xin.sizes() && f32_or_bf16(*residual)),
          "rms_norm: residual must be a float32 or bfloat16 matrix of x's shape on x's device");
  require(!add || residual->scalar_type() == xin.scalar_type() || residual->scalar_type() == at::kFloat,
          "rms_norm: a bfloat16 residual takes a bfloat16 x");
  require(eps >= 0, "rms_norm: eps must not be negative");
  require(y_type >= GC_TYPE_F32 && y_type <= GC_TYPE_E4M3, "rms_norm: the output is float32, bfloat16 or 8 bits");
  const c10::cuda::CUDAGuard guard(dev);
  NormForward f;
  f.x = row_major(xin);
  f.weight = weight.contiguous();
  if (add) f.residual = row_major(*residual);
  const at::ScalarType stream_type = add ? f.residual.scalar_type() : f.x.scalar_type();
  f.y = empty_like_rows(M, N, y_type == GC_TYPE_F32 ? at::kFloat : y_type == GC_TYPE_BF16 ? at::kBFloat16 : at::kFloat8_e4m3fn, dev);
  if (add) f.stream = empty_like_rows(M, N, stream_type, dev);
  const auto f32 = at::TensorOptions().dtype(at::kFloat).device(dev);
  if (want_rstd) f.rstd = at::empty({M}, f32);
  if (y_type == GC_TYPE_E4M3) f.scale = N ? at::empty({M}, f32) : at::zeros({M}, f32);
  const int64_t ld = std::max<int64_t>(N, 1);
  check(abi.gc_rms_norm_forward(f.x.const_data_ptr(), type_of(f.x), ld_of(f.x), add ? f.residual.const_data_ptr() : nullptr,
                                add ? ld_of(f.residual) : ld, stream_type == at::kFloat ? GC_TYPE_F32 : GC_TYPE_BF16,
                                f.weight.const_data_ptr<float>(), M, N, eps, f.y.data_ptr(), y_type, ld,
                                add ? f.stream.data_ptr() : nullptr, ld, want_rstd ? f.rstd.data_ptr<float>() : nullptr,
                                y_type == GC_TYPE_E4M3 ? f.scale.data_ptr<float>() : nullptr, stream_of(dev)),
        "gc_rms_norm_forward");
  return f;
}

// What the backward pass reads: an fp32 stream is h itself; a bf16 stream is h rounded, and x and the residual are added
// again instead.
variable_list norm_saved(const NormForward& f) {
  if (f.stream.defined() && f.stream.scalar_type() == at::kFloat) return {f.stream, Tensor(), f.weight, f.rstd};
  return {f.x, f.residual, f.weight, f.rstd};
}

NormGrads rms_norm_backward(const OptTensor& dy_in, const OptTensor& dstream_in, const Tensor& h, const OptTensor& residual,
                            const Tensor& weight, const Tensor& rstd, int y_type, int x_type, bool had_residual,
                            bool need_dx, bool need_dw) {
  const at::Device dev = h.device();
  const c10::cuda::CUDAGuard guard(dev);
  const int64_t M = h.size(0), N = h.size(1), ld = std::max<int64_t>(N, 1);
  const at::ScalarType stream_type = h.scalar_type();
  const at::ScalarType dx_type = x_type == GC_TYPE_F32 ? at::kFloat : at::kBFloat16;
  const Tensor dy = dy_in && dy_in->defined()
                        ? row_major(*dy_in)
                        : at::zeros({M, N}, h.options().dtype(y_type == GC_TYPE_F32 ? at::kFloat : at::kBFloat16));
  Tensor dstream;
  if (dstream_in && dstream_in->defined()) dstream = row_major(*dstream_in);
  const bool again = residual && residual->defined();
  NormGrads g;
  const bool other = had_residual && stream_type != dx_type;  // the residual's gradient has a type of its own
  if (need_dx) {
    g.dx = empty_like_rows(M, N, dx_type, dev);
    if (other) g.dresidual = empty_like_rows(M, N, stream_type, dev);
    else if (had_residual) g.dresidual = g.dx;
  }
  if (need_dw) g.dweight = at::empty({N}, at::TensorOptions().dtype(at::kFloat).device(dev));
  const Scratch ws = scratch(kSpmm, need_dw ? abi.gc_rms_norm_backward_workspace_bytes(M, N) : 0, dev);
  check(abi.gc_rms_norm_backward(
            dy.const_data_ptr(), type_of(dy), ld_of(dy), dstream.defined() ? dstream.const_data_ptr() : nullptr,
            dstream.defined() ? ld_of(dstream) : ld, h.const_data_ptr(), ld_of(h),
            again ? residual->const_data_ptr() : nullptr, again ? ld_of(*residual) : ld,
            stream_type == at::kFloat ? GC_TYPE_F32 : GC_TYPE_BF16, weight.const_data_ptr<float>(),
            rstd.const_data_ptr<float>(), M, N, need_dx ? g.dx.data_ptr() : nullptr, x_type, ld,
            need_dx && other ? g.dresidual.data_ptr() : nullptr, ld, need_dw ? g.dweight.data_ptr<float>() : nullptr,
            ws.ptr, ws.bytes, stream_of(dev)),
        "gc_rms_norm_backward");
  return g;
}

namespace {
struct NormFunction : torch::autograd::Function<NormFunction> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const OptTensor& residual,
                               double eps, int64_t y_type) {
    const NormForward f = rms_norm_forward(x, weight, residual, eps, int(y_type), true);
    ctx->save_for_backward(norm_saved(f));
    ctx->set_materialize_grads(false);  // an output that nobody uses has no gradient, not one of zeros
    ctx->saved_data["types"] = y_type | int64_t(type_of(x)) << 2 | int64_t(f.stream.defined()) << 4;
    if (!f.stream.defined()) return {f.y};
    return {f.y, f.stream};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once("rms_norm");
    const auto saved = ctx->get_saved_variables();
    const int64_t types = ctx->saved_data["types"].toInt();
    const bool add = types & 16, res = add && ctx->needs_input_grad(2);
    const bool need_dx = ctx->needs_input_grad(0) || res;
    const NormGrads g = rms_norm_backward(grads[0], add ? OptTensor(grads[1]) : OptTensor(), saved[0], saved[1], saved[2],
                                          saved[3], types & 3, (types >> 2) & 3, add, need_dx, ctx->needs_input_grad(1));
    return {ctx->needs_input_grad(0) ? g.dx : Tensor(), g.dweight, res ? g.dresidual : Tensor(), Tensor(), Tensor()};
  }
};
}  // namespace

std::pair<Tensor, Tensor> rms_norm(const Tensor& x, const Tensor& weight, const OptTensor& residual, double eps,
                                   int64_t y_type) {
  if (!recorded({&x, &weight, residual ? &*residual : nullptr})) {
    const NormForward f = rms_norm_forward(x, weight, residual, eps, int(y_type), false);
    return {f.y, f.stream};
  }
  const variable_list out = NormFunction::apply(x, weight, residual, eps, y_type);
  return {out[0], out.size() > 1 ? out[1] : Tensor()};
}

std::tuple<Tensor, Tensor, Tensor> rms_norm_fp8(const Tensor& x, const Tensor& weight, const OptTensor& residual, double eps) {
  const NormForward f = rms_norm_forward(x, weight, residual, eps, GC_TYPE_E4M3, false);
  return {f.y, f.scale, f.stream};
}

void refuse_norm_fp8_gradient(const Tensor& x, const Tensor& weight, const OptTensor& residual) {
  if (recorded({&x, &weight, residual ? &*residual : nullptr}))
    raise("rms_norm_fp8 has no gradient: call it under torch.no_grad(), or rms_norm for training");
}

// ------------------------------------------------------------------ gated feed-forward block
// Beyond a few megabytes the workspace holds matrices of the size of activations (700 MB at 169,343 rows of 1024): the call's own
// memory then, which the next layer can have when the call has ended.
Scratch product_workspace(size_t bytes, const at::Device& dev) {
  constexpr size_t kKept = size_t(32) << 20;
  if (bytes <= kKept) return scratch(kGemm, bytes, dev);
  Scratch s;
  s.keep = at::empty({int64_t(bytes)}, at::TensorOptions().dtype(at::kByte).device(dev));
  s.ptr = s.keep.data_ptr();
  s.bytes = bytes;
  return s;
}

namespace {
struct FfnSizes {
  int64_t M, D, H, O;
};
const uint16_t* bits(const Tensor& t) { return static_cast<const uint16_t*>(t.const_data_ptr()); }
uint16_t* bits_mut(const Tensor& t) { return static_cast<uint16_t*>(t.data_ptr()); }
bool bf16_matrix(const Tensor& t, const at::Device& dev) {
  return t.dim() == 2 && t.device() == dev && t.scalar_type() == at::kBFloat16;
}
FfnSizes ffn_sizes(const Tensor& x, const Tensor& w_in, const Tensor& w_out) {
  require(x.is_cuda() && bf16_matrix(x, x.device()), "gated_ffn: x must be a bfloat16 CUDA matrix");
  require(bf16_matrix(w_in, x.device()) && w_in.size(0) == x.size(1) && w_in.size(1) % 2 == 0,
          "gated_ffn: w_in must be bfloat16 [in, 2 * hidden] on x's device");
  require(bf16_matrix(w_out, x.device()) && w_out.size(0) == w_in.size(1) / 2,
          "gated_ffn: w_out must be bfloat16 [hidden, out] on x's device");
  return {x.size(0), x.size(1), w_out.size(0), w_out.size(1)};
}
}  // namespace

FfnForward gated_ffn_forward(const Tensor& xin, const Tensor& w_in, const Tensor& w_out, int act, bool save) {
  const FfnSizes n = ffn_sizes(xin, w_in, w_out);
  const at::Device dev = xin.device();
  const c10::cuda::CUDAGuard guard(dev);
  FfnForward f;
  f.x = row_major(xin);
  f.w_in = row_major(w_in);
  f.w_out = row_major(w_out);
  f.y = empty_like_rows(n.M, n.O, at::kBFloat16, dev);
  if (save)
    f.saved = at::empty({int64_t(abi.gc_gated_ffn_saved_bytes(n.M, n.H))}, at::TensorOptions().dtype(at::kByte).device(dev));
  const Scratch ws = product_workspace(abi.gc_gated_ffn_workspace_bytes(n.M, n.D, n.H, n.O, 0), dev);
  check(abi.gc_gated_ffn_forward_bf16(bits(f.x), ld_of(f.x), bits(f.w_in), ld_of(f.w_in), bits(f.w_out), ld_of(f.w_out),
                                      n.M, n.D, n.H, n.O, act, bits_mut(f.y), std::max<int64_t>(n.O, 1),
                                      save ? f.saved.data_ptr() : nullptr, ws.ptr, ws.bytes, stream_of(dev)),
        "gc_gated_ffn_forward_bf16");
  return f;
}

FfnGrads gated_ffn_backward(const Tensor& dy_in, const Tensor& x, const Tensor& w_in, const Tensor& w_out,
                            const Tensor& saved, int act, bool need_dx, bool need_dw_in, bool need_dw_out) {
  const FfnSizes n = ffn_sizes(x, w_in, w_out);
  const at::Device dev = x.device();
  const c10::cuda::CUDAGuard guard(dev);
  const Tensor dy = row_major(dy_in);
  FfnGrads g;
  if (need_dx) g.dx = empty_like_rows(n.M, n.D, at::kBFloat16, dev);
  if (need_dw_in) g.dw_in = empty_like_rows(n.D, 2 * n.H, at::kBFloat16, dev);
  if (need_dw_out) g.dw_out = empty_like_rows(n.H, n.O, at::kBFloat16, dev);
  const Scratch ws = product_workspace(abi.gc_gated_ffn_workspace_bytes(n.M, n.D, n.H, n.O, 1), dev);
  check(abi.gc_gated_ffn_backward_bf16(
            bits(dy), ld_of(dy), bits(x), ld_of(x), bits(w_in), ld_of(w_in), bits(w_out), ld_of(w_out),
            saved.const_data_ptr(), n.M, n.D, n.H, n.O, act, need_dx ? bits_mut(g.dx) : nullptr, std::max<int64_t>(n.D, 1),
            need_dw_in ? bits_mut(g.dw_in) : nullptr, std::max<int64_t>(2 * n.H, 1),
            need_dw_out ? bits_mut(g.dw_out) : nullptr, std::max<int64_t>(n.O, 1), ws.ptr, ws.bytes, stream_of(dev)),
        "gc_gated_ffn_backward_bf16");
  return g;
}

namespace {
struct FfnFunction : torch::autograd::Function<FfnFunction> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w_in, const Tensor& w_out, int64_t act) {
    const FfnForward f = gated_ffn_forward(x, w_in, w_out, int(act), true);
    ctx->save_for_backward({f.x, f.w_in, f.w_out, f.saved});
    ctx->saved_data["act"] = act;
    return f.y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once("gated_ffn");
    if (!grads[0].defined()) return {Tensor(), Tensor(), Tensor(), Tensor()};
    const auto saved = ctx->get_saved_variables();
    const FfnGrads g = gated_ffn_backward(grads[0], saved[0], saved[1], saved[2], saved[3],
                                          int(ctx->saved_data["act"].toInt()), ctx->needs_input_grad(0),
                                          ctx->needs_input_grad(1), ctx->needs_input_grad(2));
    return {g.dx, g.dw_in, g.dw_out, Tensor()};
  }
};
}  // namespace

Tensor gated_ffn(const Tensor& x, const Tensor& w_in, const Tensor& w_out, int64_t act) {
  if (!recorded({&x, &w_in, &w_out})) return gated_ffn_forward(x, w_in, w_out, int(act), false).y;
  return FfnFunction::apply(x, w_in, w_out, act);
}

Tensor gated_ffn_fp8(const Tensor& x8, const Tensor& x_scale, const Tensor& w8, const Tensor& w_scale, const Tensor& w_out,
                     int64_t act) {
  require(x8.is_cuda() && x8.dim() == 2 && x8.scalar_type() == at::kFloat8_e4m3fn,
          "gated_ffn_fp8: x8 must be a float8_e4m3fn CUDA matrix");
  const at::Device dev = x8.device();
  const int64_t M = x8.size(0), D = x8.size(1);
  require(w8.dim() == 2 && w8.device() == dev && w8.scalar_type() == at::kFloat8_e4m3fn && w8.size(1) == D &&
              w8.size(0) % 2 == 0,
          "gated_ffn_fp8: w8 must be float8_e4m3fn [2 * hidden, in] on x8's device");
  const int64_t H = w8.size(0) / 2;
  require(f32_on(x_scale, dev) && x_scale.dim() == 1 && x_scale.size(0) == M && f32_on(w_scale, dev) &&
              w_scale.dim() == 1 && w_scale.size(0) == 2 * H,
          "gated_ffn_fp8: float32 scales expected, one per row of x8 and of w8, on their device");
  require(bf16_matrix(w_out, dev) && w_out.size(0) == H, "gated_ffn_fp8: w_out must be bfloat16 [hidden, out] on x8's device");
  const int64_t O = w_out.size(1);
  const c10::cuda::CUDAGuard guard(dev);
  const Tensor x = row_major(x8), w = row_major(w8), wo = row_major(w_out);
  const Tensor sx = x_scale.contiguous(), sw = w_scale.contiguous();
  Tensor y = empty_like_rows(M, O, at::kBFloat16, dev);
  const Scratch ws = product_workspace(abi.gc_gated_ffn_e4m3_workspace_bytes(M, D, H, O), dev);
  check(abi.gc_gated_ffn_forward_e4m3(static_cast<const uint8_t*>(x.const_data_ptr()), ld_of(x), sx.const_data_ptr<float>(),
                                      static_cast<const uint8_t*>(w.const_data_ptr()), ld_of(w), sw.const_data_ptr<float>(),
                                      bits(wo), ld_of(wo), M, D, H, O, int(act), bits_mut(y), std::max<int64_t>(O, 1),
                                      ws.ptr, ws.bytes, stream_of(dev)),
        "gc_gated_ffn_forward_e4m3");
  return y;
}

void refuse_ffn_fp8_gradient(std::initializer_list<const Tensor*> inputs) {
  if (recorded(inputs))
    raise("gated_ffn_fp8 has no gradient: call it under torch.no_grad(), or gated_ffn for training");
}

// ------------------------------------------------------------------ AdamW
namespace {
bool part(const Tensor& t, at::ScalarType type, const at::Device& dev, int64_t n) {
  return t.scalar_type() == type && t.device() == dev && t.is_contiguous() && t.numel() == n;
}
int64_t blocks_of(int64_t n) { return (n + GC_ADAMW_BLOCK - 1) / GC_ADAMW_BLOCK; }
}  // namespace

void adamw_step(const std::vector<Tensor>& p, const std::vector<Tensor>& g, const std::vector<Tensor>& m,
                const std::vector<Tensor>& v, const Tensor& state, const std::vector<Tensor>& masters,
                const std::vector<Tensor>& ms, const std::vector<Tensor>& vs, double lr, double b1, double b2, double eps,
                double wd, int64_t seed, bool follow) {
  const size_t count = p.size();
  require(state.is_cuda() && state.scalar_type() == at::kLong && state.is_contiguous() && state.numel() >= 2,
          "adamw_step: step must be a CUDA int64 tensor of two elements, zeros before the first step");
  require(g.size() == count && m.size() == count && v.size() == count, "adamw_step: the lists must have one length");
  const at::Device dev = state.device();
  const bool mixed = count && p[0].scalar_type() == at::kBFloat16, eight = count && m[0].scalar_type() == at::kByte;
  require(masters.size() == (mixed ? count : 0), "adamw_step: bfloat16 parameters need float32 masters, float32 ones take none");
  require(!follow || !count || mixed, "adamw_step: float32 parameters have no masters that could follow them");
  require(ms.size() == (eight ? count : 0) && vs.size() == ms.size(),
          "adamw_step: moments in 8 bits need their scales, moments in 32 bits have none");
  require(lr >= 0 && eps >= 0 && wd >= 0 && b1 >= 0 && b1 < 1 && b2 >= 0 && b2 < 1, "adamw_step: invalid hyper-parameter");
  const at::ScalarType pt = mixed ? at::kBFloat16 : at::kFloat, mt = eight ? at::kByte : at::kFloat;
  std::vector<void*> pp(count), mm(count), vv(count);
  std::vector<const void*> gg(count);
  std::vector<float*> mas(masters.size()), mss(ms.size()), vss(vs.size());
  std::vector<int64_t> n(count);
  std::vector<Tensor> keep;
  for (size_t i = 0; i < count; ++i) {
    n[i] = p[i].numel();
    require(part(p[i], pt, dev, n[i]), "adamw_step: parameters must be contiguous, all float32 or all bfloat16, on the step's device");
    require(!g[i].is_sparse() && g[i].scalar_type() == pt && g[i].device() == dev && g[i].numel() == n[i],
            "adamw_step: gradients must be dense tensors of the parameter's type and size on its device");
    require(part(m[i], mt, dev, n[i]) && part(v[i], mt, dev, n[i]),
            "adamw_step: exp_avg and exp_avg_sq must be contiguous tensors of the parameter's size, all float32 or all uint8");
    pp[i] = p[i].data_ptr();
    if (g[i].is_contiguous()) {
      gg[i] = g[i].const_data_ptr();
    } else {
      const c10::cuda::CUDAGuard guard(dev);
      keep.push_back(g[i].contiguous());
      gg[i] = keep.back().const_data_ptr();
    }
    mm[i] = m[i].data_ptr();
    vv[i] = v[i].data_ptr();
    if (mixed) {
      require(part(masters[i], at::kFloat, dev, n[i]), "adamw_step: masters must be contiguous float32 tensors of the parameter's size");
      mas[i] = static_cast<float*>(masters[i].data_ptr());
    }
    if (eight) {
      require(part(ms[i], at::kFloat, dev, blocks_of(n[i])) && part(vs[i], at::kFloat, dev, blocks_of(n[i])),
              "adamw_step: scales must be contiguous float32 tensors with one element per 256 of the parameter");
      mss[i] = static_cast<float*>(ms[i].data_ptr());
      vss[i] = static_cast<float*>(vs[i].data_ptr());
    }
  }
  const c10::cuda::CUDAGuard guard(dev);
  check(abi.gc_adamw_step(int(count), pp.data(), !mixed ? GC_TYPE_F32 : follow ? GC_TYPE_BF16 | GC_ADAMW_FOLLOW : GC_TYPE_BF16, gg.data(), mas.data(), mm.data(),
                          vv.data(), mss.data(), vss.data(), n.data(), eight ? 8 : 32, lr, b1, b2, eps, wd, uint32_t(seed),
                          state.data_ptr(), stream_of(dev)),
        "gc_adamw_step");
  for (const auto* list : {&p, &m, &v, &masters, &ms, &vs}) written(*list);
  written(state);
}

void adamw_moments(const std::vector<Tensor>& m, const std::vector<Tensor>& v, const std::vector<Tensor>& ms,
                   const std::vector<Tensor>& vs, const std::vector<Tensor>& m_out, const std::vector<Tensor>& v_out) {
  const size_t count = m.size();
  require(v.size() == count && ms.size() == count && vs.size() == count && m_out.size() == count && v_out.size() == count,
          "adamw_moments: the lists must have one length");
  if (count == 0) return;
  require(m[0].is_cuda(), "adamw_moments: CUDA tensors expected");
  const at::Device dev = m[0].device();
  std::vector<const uint8_t*> mm(count), vv(count);
  std::vector<const float*> mss(count), vss(count);
  std::vector<float*> mo(count), vo(count);
  std::vector<int64_t> n(count);
  for (size_t i = 0; i < count; ++i) {
    n[i] = m[i].numel();
    require(part(m[i], at::kByte, dev, n[i]) && part(v[i], at::kByte, dev, n[i]) &&
                part(ms[i], at::kFloat, dev, blocks_of(n[i])) && part(vs[i], at::kFloat, dev, blocks_of(n[i])),
            "adamw_moments: uint8 moments with a float32 scale per 256 elements expected, on one device");
    require(part(m_out[i], at::kFloat, dev, n[i]) && part(v_out[i], at::kFloat, dev, n[i]),
            "adamw_moments: outputs must be contiguous float32 tensors of the moments' size on their device");
    mm[i] = m[i].const_data_ptr<uint8_t>();
    vv[i] = v[i].const_data_ptr<uint8_t>();
    mss[i] = ms[i].const_data_ptr<float>();
    vss[i] = vs[i].const_data_ptr<float>();
    mo[i] = static_cast<float*>(m_out[i].data_ptr());
    vo[i] = static_cast<float*>(v_out[i].data_ptr());
  }
  const c10::cuda::CUDAGuard guard(dev);
  check(abi.gc_adamw_moments_f32(int(count), mm.data(), vv.data(), mss.data(), vss.data(), n.data(), mo.data(), vo.data(),
                                 stream_of(dev)),
        "gc_adamw_moments_f32");
  written(m_out);
  written(v_out);
}

}  // namespace gch
