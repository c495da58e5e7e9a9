// Rows sorted by group times a weight per group, with its autograd node.
#include <torch/csrc/autograd/custom_function.h>

#include "host.h"

namespace gch {

namespace {
const uint16_t* bits(const Tensor& t) { return static_cast<const uint16_t*>(t.const_data_ptr()); }
uint16_t* bits_mut(const Tensor& t) { return static_cast<uint16_t*>(t.data_ptr()); }
// The weights of all groups one below the other: any pitch of their rows, and no gap between groups.
Tensor stacked(const Tensor& w) {
  const bool rows = w.stride(2) == 1 && w.stride(1) >= std::max<int64_t>(1, w.size(2)) &&
                    (w.size(0) <= 1 || w.stride(0) == w.size(1) * w.stride(1));
  return rows ? w : w.contiguous();
}
}  // namespace

GroupedForward grouped_linear_forward(const Tensor& x, const Tensor& w, const Tensor& offsets) {
  require(x.dim() == 2 && x.is_cuda() && x.scalar_type() == at::kBFloat16, "grouped_linear: x must be a bfloat16 CUDA matrix");
  const at::Device dev = x.device();
  require(w.dim() == 3 && w.device() == dev && w.scalar_type() == at::kBFloat16 && w.size(1) == x.size(1),
          "grouped_linear: w must be bfloat16 [groups, in, out] on x's device");
  require(offsets.dim() == 1 && offsets.device() == dev && offsets.scalar_type() == at::kInt && offsets.size(0) == w.size(0) + 1,
          "grouped_linear: offsets must be int32 [groups + 1] on x's device");
  const c10::cuda::CUDAGuard guard(dev);
  GroupedForward f;
  f.x = row_major(x);
  f.w = stacked(w);
  f.offsets = offsets.contiguous();
  const int64_t M = x.size(0), K = x.size(1), G = w.size(0), N = w.size(2);
  f.y = at::empty({M, N}, x.options());
  const Scratch ws = product_workspace(abi.gc_grouped_linear_workspace_bytes_for(nullptr, 0, bits(f.x), ld_of(f.x), bits(f.w),
                                                                                     std::max<int64_t>(f.w.stride(1), N), M, K, N, G, 0, 0), dev);
  check(abi.gc_grouped_linear_forward_bf16(bits(f.x), ld_of(f.x), bits(f.w), std::max<int64_t>(f.w.stride(1), N),
                                           f.offsets.const_data_ptr<int32_t>(), M, K, N, G, bits_mut(f.y), std::max<int64_t>(N, 1),
                                           ws.ptr, ws.bytes, stream_of(dev)),
        "gc_grouped_linear_forward_bf16");
  return f;
}

std::pair<Tensor, Tensor> grouped_linear_backward(const Tensor& dy_in, const Tensor& x, const Tensor& w, const Tensor& offsets,
                                                  bool need_dx, bool need_dw) {
  const at::Device dev = x.device();
  const c10::cuda::CUDAGuard guard(dev);
  const int64_t M = x.size(0), K = x.size(1), G = w.size(0), N = w.size(2);
  const Tensor dy = row_major(dy_in);
  Tensor dx, dw;
  if (need_dx) dx = at::empty({M, K}, x.options());
  if (need_dw) dw = at::empty({G, K, N}, x.options());
  const Scratch ws = product_workspace(abi.gc_grouped_linear_workspace_bytes_for(bits(dy), ld_of(dy), bits(x), ld_of(x), bits(w),
                                                                                     std::max<int64_t>(w.stride(1), N), M, K, N, G, need_dx,
                                                                                     need_dw), dev);
  check(abi.gc_grouped_linear_backward_bf16(bits(dy), ld_of(dy), bits(x), ld_of(x), bits(w), std::max<int64_t>(w.stride(1), N),
                                            offsets.const_data_ptr<int32_t>(), M, K, N, G, need_dx ? bits_mut(dx) : nullptr,
                                            std::max<int64_t>(K, 1), need_dw ? bits_mut(dw) : nullptr, ws.ptr, ws.bytes, stream_of(dev)),
        "gc_grouped_linear_backward_bf16");
  return {dx, dw};
}

namespace {
struct GroupedFunction : torch::autograd::Function<GroupedFunction> {
  static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const Tensor& w, const Tensor& offsets) {
    const GroupedForward f = grouped_linear_forward(x, w, offsets);
    ctx->save_for_backward({f.x, f.w, f.offsets});
    return f.y;
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    once("grouped_linear");
    if (!grads[0].defined()) return {Tensor(), Tensor(), Tensor()};
    const auto saved = ctx->get_saved_variables();
    const auto [dx, dw] = grouped_linear_backward(grads[0], saved[0], saved[1], saved[2], ctx->needs_input_grad(0), ctx->needs_input_grad(1));
    return {dx, dw, Tensor()};
  }
};
}  // namespace

Tensor grouped_linear(const Tensor& x, const Tensor& w, const Tensor& offsets) {
  if (!recorded({&x, &w})) return grouped_linear_forward(x, w, offsets).y;
  return GroupedFunction::apply(x, w, offsets);
}

}  // namespace gch
