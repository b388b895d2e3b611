// C ABI of the dropout kernels, and their instances of every type.
#include "dropout_series.inl"

namespace pt {
template int launch_dropout<float>(const DropoutArgs&);
template int launch_dropout<double>(const DropoutArgs&);
template int launch_dropout<bf16>(const DropoutArgs&);
template int launch_dropout<_Float16>(const DropoutArgs&);
}  // namespace pt

extern "C" {

int pt_dropout_series(int dtype, int orders, const void* const* x, void* const* y, int64_t numel, double p,
                      const int64_t* seed, void* stream) {
  pt_host::clear_error();
  PT_REQUIRE(orders >= 1 && orders <= PT_MAX_ELEMENTWISE_DEGREE + 1, PT_UNSUPPORTED,
             "dropout series: orders must be in 1..17");
  PT_REQUIRE(dtype >= PT_FLOAT32 && dtype <= PT_FLOAT16, PT_UNSUPPORTED, "dropout series: unknown dtype code");
  PT_REQUIRE(p >= 0.0 && p <= 1.0, PT_INVALID_ARGUMENT, "dropout series: p must be in [0, 1]");
  PT_REQUIRE(numel >= 0, PT_INVALID_ARGUMENT, "dropout series: need numel >= 0");
  PT_REQUIRE(x != nullptr && y != nullptr && seed != nullptr, PT_INVALID_ARGUMENT,
             "dropout series: x and y pointer arrays and the seed are required");
  for (int k = 0; k < orders; ++k)
    PT_REQUIRE(numel == 0 || (x[k] != nullptr && y[k] != nullptr), PT_INVALID_ARGUMENT,
               "dropout series: null coefficient pointer");
  if (numel == 0) return PT_OK;
  pt::DropoutArgs a{orders, x, y, numel, p, seed, static_cast<hipStream_t>(stream)};
  switch (dtype) {
    case PT_FLOAT32: return pt::launch_dropout<float>(a);
    case PT_FLOAT64: return pt::launch_dropout<double>(a);
    case PT_BFLOAT16: return pt::launch_dropout<pt::bf16>(a);
    default: return pt::launch_dropout<_Float16>(a);
  }
}

}  // extern "C"
