// C ABI of the per-head norm and rotation kernels.
#include "norm_rope_series.h"

namespace {

int check(const char* what, const pt::NormRopeArgs& a, int dtype, bool backward) {
  const std::string name(what);
  PT_REQUIRE(a.degree >= 0 && a.degree <= PT_MAX_DEGREE, PT_UNSUPPORTED, name + ": degree must be in 0..8");
  PT_REQUIRE(dtype >= PT_FLOAT32 && dtype <= PT_FLOAT16, PT_UNSUPPORTED, name + ": unknown dtype code");
  PT_REQUIRE((a.n_ops == 1 || a.n_ops == 2) && a.ops != nullptr, PT_INVALID_ARGUMENT, name + ": one or two operands");
  PT_REQUIRE(a.batch >= 0 && a.length >= 0, PT_INVALID_ARGUMENT, name + ": need batch >= 0 and length >= 0");
  PT_REQUIRE(a.head_dim >= 1 && a.head_dim <= PT_NORM_ROPE_MAX_HEAD, PT_UNSUPPORTED, name + ": head_dim must be in 1..256");
  PT_REQUIRE(a.rotary >= 0 && a.rotary <= a.head_dim && a.rotary % 2 == 0, PT_INVALID_ARGUMENT,
             name + ": rotary must be even and at most head_dim");
  PT_REQUIRE(a.table_rows >= 0 && (a.rotary == 0 || a.table_rows == 0 || (a.cos != nullptr && a.sin != nullptr)),
             PT_INVALID_ARGUMENT, name + ": cos and sin tables are required");
  PT_REQUIRE(a.position_batch_stride >= 0, PT_INVALID_ARGUMENT, name + ": need position_batch_stride >= 0");
  PT_REQUIRE(a.eps >= 0.0, PT_INVALID_ARGUMENT, name + ": need eps >= 0");
  for (int o = 0; o < a.n_ops; ++o) {
    const pt_norm_rope_operand& op = a.ops[o];
    PT_REQUIRE(op.heads >= 1, PT_INVALID_ARGUMENT, name + ": need heads >= 1");
    PT_REQUIRE(a.batch == 0 || a.length == 0 ||
                   (a.length <= INT32_MAX && a.batch <= INT32_MAX / a.length && op.heads <= INT32_MAX / (a.batch * a.length)),
               PT_UNSUPPORTED, name + ": batch x length x heads beyond 2^31-1");
    PT_REQUIRE(op.stride_b >= 0 && op.stride_l >= 0 && op.stride_h >= 0, PT_INVALID_ARGUMENT, name + ": negative stride");
    PT_REQUIRE(op.x != nullptr && (backward ? op.grad != nullptr && op.dx != nullptr : op.y != nullptr), PT_INVALID_ARGUMENT,
               name + (backward ? ": x, grad and dx pointer arrays are required" : ": x and y pointer arrays are required"));
    PT_REQUIRE(op.weight_orders == 0 || ((op.weight_orders == 1 || op.weight_orders == a.degree + 1) && op.weight != nullptr),
               PT_INVALID_ARGUMENT, name + ": weight_orders must be 0, 1 or degree + 1");
    for (int k = 0; k < op.weight_orders; ++k)
      PT_REQUIRE(op.weight[k] != nullptr, PT_INVALID_ARGUMENT, name + ": null weight pointer");
    for (int k = 0; k <= a.degree; ++k)
      PT_REQUIRE(op.x[k] != nullptr && (backward ? op.grad[k] != nullptr && op.dx[k] != nullptr : op.y[k] != nullptr),
                 PT_INVALID_ARGUMENT, name + ": null coefficient pointer");
    if (backward) {
      PT_REQUIRE(op.dweight_orders == 0 ||
                     ((op.dweight_orders == 1 || op.dweight_orders == a.degree + 1) && op.dweight != nullptr),
                 PT_INVALID_ARGUMENT, name + ": dweight_orders must be 0, 1 or degree + 1");
      for (int k = 0; k < op.dweight_orders; ++k)
        PT_REQUIRE(op.dweight[k] != nullptr, PT_INVALID_ARGUMENT, name + ": null dweight pointer");
      PT_REQUIRE(op.dweight_orders == 0 || a.batch == 0 || a.length == 0 || a.workspace != nullptr, PT_INVALID_ARGUMENT,
                 name + ": weight gradients need the workspace");
      PT_REQUIRE(op.dweight_orders == 0 || (a.batch > 0 && a.length > 0), PT_UNSUPPORTED,
                 name + ": a weight gradient over no rows");
    }
  }
  return PT_OK;
}

}  // namespace

extern "C" {

size_t pt_norm_rope_series_bwd_workspace_size(int dtype, int degree, int64_t rows, int64_t head_dim) {
  if (degree < 0 || degree > PT_MAX_DEGREE || rows <= 0 || head_dim <= 0 || head_dim > PT_NORM_ROPE_MAX_HEAD) return 0;
  return static_cast<size_t>(pt::norm_rope_partials(rows)) * (degree + 1) * head_dim *
         (dtype == PT_FLOAT64 ? sizeof(double) : sizeof(float));
}

int pt_norm_rope_series_fwd(int dtype, int degree, int n_operands, const pt_norm_rope_operand* operands, int64_t batch,
                            int64_t length, int64_t head_dim, int64_t rotary, int interleaved, const void* cos,
                            const void* sin, int64_t table_rows, const int64_t* positions, int64_t position_batch_stride,
                            double eps, void* stream) {
  pt_host::clear_error();
  pt::NormRopeArgs a{degree, n_operands, operands, batch, length, head_dim, rotary, interleaved, cos, sin, table_rows,
                     positions, position_batch_stride, eps, nullptr, static_cast<hipStream_t>(stream)};
  const int status = check("norm and rotation series", a, dtype, false);
  if (status != PT_OK || batch == 0 || length == 0) return status;
  switch (dtype) {
    case PT_FLOAT32: return pt::launch_norm_rope<float>(a);
    case PT_FLOAT64: return pt::launch_norm_rope<double>(a);
    case PT_BFLOAT16: return pt::launch_norm_rope<pt::bf16>(a);
    default: return pt::launch_norm_rope<_Float16>(a);
  }
}

int pt_norm_rope_series_bwd(int dtype, int degree, int n_operands, const pt_norm_rope_operand* operands, int64_t batch,
                            int64_t length, int64_t head_dim, int64_t rotary, int interleaved, const void* cos,
                            const void* sin, int64_t table_rows, const int64_t* positions, int64_t position_batch_stride,
                            double eps, void* workspace, void* stream) {
  pt_host::clear_error();
  pt::NormRopeArgs a{degree, n_operands, operands, batch, length, head_dim, rotary, interleaved, cos, sin, table_rows,
                     positions, position_batch_stride, eps, workspace, static_cast<hipStream_t>(stream)};
  const int status = check("norm and rotation series backward", a, dtype, true);
  if (status != PT_OK || batch == 0 || length == 0) return status;
  switch (dtype) {
    case PT_FLOAT32: return pt::launch_norm_rope_bwd<float>(a);
    case PT_FLOAT64: return pt::launch_norm_rope_bwd<double>(a);
    case PT_BFLOAT16: return pt::launch_norm_rope_bwd<pt::bf16>(a);
    default: return pt::launch_norm_rope_bwd<_Float16>(a);
  }
}

}  // extern "C"
