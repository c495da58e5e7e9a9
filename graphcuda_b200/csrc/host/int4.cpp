// Serving with weights of 4 bits: a product, and the gated feed-forward block.
#include "host.h"

namespace gch {

namespace {
const uint16_t* bits(const Tensor& t) { return static_cast<const uint16_t*>(t.const_data_ptr()); }
const uint8_t* records(const Int4& w) { return static_cast<const uint8_t*>(w.records.const_data_ptr()); }
// The buffer is what the kernels read, up to its end: its size has to be the weight's.
void check_weight(const Int4& w, const at::Device& dev) {
  require(w.k >= 0 && w.n >= 0 && (w.group == 32 || w.group == 64 || w.group == 128), "Int4Weight: a group is 32, 64 or 128 inputs");
  const int64_t groups = 16 * (128 / w.group), record = 1024 + groups * (w.zeros ? 3 : 2);
  require(w.records.device() == dev && w.records.scalar_type() == at::kByte && w.records.is_contiguous() &&
              w.records.numel() == (w.n + 15) / 16 * ((w.k + 127) / 128) * record,
          "Int4Weight: records must be what Int4Weight.from_codes lays out, on x's device");
}
}  // namespace

Tensor linear_int4(const Tensor& xin, const Int4& w) {
  require(xin.dim() == 2 && xin.is_cuda() && xin.scalar_type() == at::kBFloat16, "linear_int4: x must be a bfloat16 CUDA matrix");
  require(xin.size(1) == w.k, "linear_int4: x must have a column per input of the weight");
  const at::Device dev = xin.device();
  check_weight(w, dev);
  const c10::cuda::CUDAGuard guard(dev);
  const Tensor x = row_major(xin);
  const int64_t M = x.size(0);
  Tensor y = at::empty({M, w.n}, x.options());
  const Scratch ws = product_workspace(abi.gc_linear_int4_workspace_bytes(M, w.k, w.n), dev);
  check(abi.gc_linear_int4_bf16(bits(x), ld_of(x), records(w), int(w.group), w.zeros, M, w.k, w.n,
                                static_cast<uint16_t*>(y.data_ptr()), std::max<int64_t>(w.n, 1), ws.ptr, ws.bytes, stream_of(dev)),
        "gc_linear_int4_bf16");
  return y;
}

Tensor gated_ffn_int4(const Tensor& xin, const Int4& w_in, const Int4& w_out, int64_t act) {
  require(xin.dim() == 2 && xin.is_cuda() && xin.scalar_type() == at::kBFloat16, "gated_ffn_int4: x must be a bfloat16 CUDA matrix");
  require(xin.size(1) == w_in.k, "gated_ffn_int4: x must have a column per input of w_in");
  require(w_in.n % 2 == 0 && w_out.k == w_in.n / 2, "gated_ffn_int4: w_in must have two outputs for every input of w_out");
  const at::Device dev = xin.device();
  check_weight(w_in, dev);
  check_weight(w_out, dev);
  const c10::cuda::CUDAGuard guard(dev);
  const Tensor x = row_major(xin);
  const int64_t M = x.size(0), O = w_out.n;
  Tensor y = at::empty({M, O}, x.options());
  const Scratch ws = product_workspace(abi.gc_gated_ffn_int4_workspace_bytes(M, w_in.k, w_out.k, O), dev);
  check(abi.gc_gated_ffn_int4_bf16(bits(x), ld_of(x), records(w_in), int(w_in.group), w_in.zeros, records(w_out), int(w_out.group),
                                   w_out.zeros, M, w_in.k, w_out.k, O,
                                   int(act), static_cast<uint16_t*>(y.data_ptr()), std::max<int64_t>(O, 1), ws.ptr, ws.bytes,
                                   stream_of(dev)),
        "gc_gated_ffn_int4_bf16");
  return y;
}

}  // namespace gch
