// C ABI of the token log-probability kernels.
#include <algorithm>

#include "token_log_probs_series.h"

namespace pt {

// Four blocks a compute unit, each with a 16-byte vector of every order a thread at least. Backward, where nothing has to be
// joined, sixteen blocks where that leaves a thread as many vectors, so that the last round of blocks is short (1100 x
// 128256 bfloat16, degree 2: 359 us with four, 328 so; forward 142 and 136, but 1500 x 50257 float32, degree 1, 98 and 114).
int64_t log_prob_splits(int64_t rows, int64_t classes, int elem_size, bool backward) {
  const int64_t round = 256 * (16 / elem_size);   // classes a block takes at a time
  auto pieces = [&](int64_t blocks, int64_t least) { return std::min((blocks + rows - 1) / rows, classes / (round * least)); };
  int64_t splits = pieces(1024, 1);
  if (backward) splits = std::max(splits, pieces(4096, 16));
  return std::max<int64_t>(1, std::min<int64_t>(64, splits));
}

size_t log_prob_workspace(int degree, int64_t rows, int64_t classes, int top, int elem_size) {
  const int64_t splits = log_prob_splits(rows, classes, elem_size, false);
  if (splits == 1) return 0;
  const size_t acc = elem_size == 8 ? 8 : 4;
  return static_cast<size_t>(rows * splits) * (acc * (top + 3 * degree + 3) + sizeof(uint32_t) * top);
}

}  // namespace pt

namespace {

int elem_size(int dtype) { return dtype == PT_FLOAT64 ? 8 : dtype == PT_FLOAT32 ? 4 : 2; }

int check(const std::string& name, int dtype, int degree, const void* const* logits, int64_t rows, int64_t classes,
          int64_t row_stride, const int64_t* tokens, double softcap, int top) {
  PT_REQUIRE(degree >= 0 && degree <= PT_MAX_DEGREE, PT_UNSUPPORTED, name + ": degree must be in 0..8");
  PT_REQUIRE(dtype >= PT_FLOAT32 && dtype <= PT_FLOAT16, PT_UNSUPPORTED, name + ": unknown dtype code");
  PT_REQUIRE(logits != nullptr, PT_INVALID_ARGUMENT, name + ": logits pointer array is required");
  PT_REQUIRE(rows >= 0 && classes >= 1 && row_stride >= classes, PT_INVALID_ARGUMENT,
             name + ": need rows >= 0, classes >= 1, row_stride >= classes");
  PT_REQUIRE(classes <= INT32_MAX, PT_UNSUPPORTED, name + ": classes beyond 2^31-1");
  PT_REQUIRE(rows <= INT32_MAX, PT_UNSUPPORTED, name + ": rows beyond 2^31-1");
  PT_REQUIRE(softcap >= 0.0 && softcap <= 1e300, PT_INVALID_ARGUMENT,
             name + ": softcap must be 0 (none) or a positive finite cap");
  PT_REQUIRE(top >= 0 && top <= PT_LOG_PROBS_MAX_TOP && top <= classes, PT_INVALID_ARGUMENT,
             name + ": top must be in 0..32 and at most classes");
  PT_REQUIRE(rows == 0 || tokens != nullptr, PT_INVALID_ARGUMENT, name + ": tokens are required");
  return PT_OK;
}

int check_orders(const std::string& name, const void* const* p, int degree, bool optional) {
  PT_REQUIRE(optional || p != nullptr, PT_INVALID_ARGUMENT, name + " pointer array is required");
  for (int k = 0; p != nullptr && k <= degree; ++k)
    PT_REQUIRE(p[k] != nullptr, PT_INVALID_ARGUMENT, name + ": null coefficient pointer");
  return PT_OK;
}

}  // namespace

#define PT_LP_CHECK(call)                      \
  do {                                         \
    const int status__ = (call);               \
    if (status__ != PT_OK) return status__;    \
  } while (0)

extern "C" {

size_t pt_token_log_probs_series_workspace_size(int dtype, int degree, int64_t rows, int64_t classes, int top) {
  if (degree < 0 || degree > PT_MAX_DEGREE || rows <= 0 || classes <= 0 || top < 0 || top > PT_LOG_PROBS_MAX_TOP) return 0;
  return pt::log_prob_workspace(degree, rows, classes, top, elem_size(dtype));
}

int pt_token_log_probs_series_fwd(int dtype, int degree, const void* const* logits, int64_t rows, int64_t classes,
                                  int64_t row_stride, const int64_t* tokens, int64_t ignore_index, double softcap, int top,
                                  void* const* log_probs, void* const* entropy, int64_t* top_tokens,
                                  void* const* top_log_probs, void* const* lse, void* workspace, void* stream) {
  pt_host::clear_error();
  const std::string name("token log-prob series");
  PT_LP_CHECK(check(name, dtype, degree, logits, rows, classes, row_stride, tokens, softcap, top));
  if (rows == 0) return PT_OK;
  PT_LP_CHECK(check_orders(name + ": logits", logits, degree, false));
  PT_LP_CHECK(check_orders(name + ": log_probs", log_probs, degree, false));
  PT_LP_CHECK(check_orders(name + ": entropy", entropy, degree, false));
  PT_LP_CHECK(check_orders(name + ": lse", lse, degree, false));
  PT_LP_CHECK(check_orders(name + ": top_log_probs", top > 0 ? top_log_probs : nullptr, degree, top == 0));
  PT_REQUIRE(top == 0 || top_tokens != nullptr, PT_INVALID_ARGUMENT, name + ": top_tokens is required");
  PT_REQUIRE(workspace != nullptr || pt::log_prob_workspace(degree, rows, classes, top, elem_size(dtype)) == 0,
             PT_INVALID_ARGUMENT, name + ": rows in pieces need the workspace");
  pt::LogProbArgs a{degree, logits, rows, classes, row_stride, tokens, ignore_index, softcap, top, log_probs,
                    entropy, top_tokens, top_log_probs, lse, workspace, static_cast<hipStream_t>(stream)};
  switch (dtype) {
    case PT_FLOAT32: return pt::launch_log_probs<float>(a);
    case PT_FLOAT64: return pt::launch_log_probs<double>(a);
    case PT_BFLOAT16: return pt::launch_log_probs<pt::bf16>(a);
    default: return pt::launch_log_probs<_Float16>(a);
  }
}

int pt_token_log_probs_series_bwd(int dtype, int degree, const void* const* logits, int64_t rows, int64_t classes,
                                  int64_t row_stride, const int64_t* tokens, int64_t ignore_index, double softcap, int top,
                                  const int64_t* top_tokens, const void* const* lse, const void* const* entropy,
                                  const void* const* cot_log_probs, const void* const* cot_entropy,
                                  const void* const* cot_top_log_probs, void* const* dz, void* stream) {
  pt_host::clear_error();
  const std::string name("token log-prob series backward");
  PT_LP_CHECK(check(name, dtype, degree, logits, rows, classes, row_stride, tokens, softcap, top));
  if (rows == 0) return PT_OK;
  PT_LP_CHECK(check_orders(name + ": logits", logits, degree, false));
  PT_LP_CHECK(check_orders(name + ": lse", lse, degree, false));
  PT_LP_CHECK(check_orders(name + ": entropy", entropy, degree, false));
  PT_LP_CHECK(check_orders(name + ": dz", dz, degree, false));
  PT_LP_CHECK(check_orders(name + ": cot_log_probs", cot_log_probs, degree, true));
  PT_LP_CHECK(check_orders(name + ": cot_entropy", cot_entropy, degree, true));
  PT_LP_CHECK(check_orders(name + ": cot_top_log_probs", cot_top_log_probs, degree, true));
  PT_REQUIRE(cot_top_log_probs == nullptr || (top > 0 && top_tokens != nullptr), PT_INVALID_ARGUMENT,
             name + ": cot_top_log_probs needs top_tokens");
  pt::LogProbBwdArgs a{degree, logits, rows, classes, row_stride, tokens, ignore_index, softcap, top, top_tokens, lse,
                       entropy, cot_log_probs, cot_entropy, cot_top_log_probs, dz, static_cast<hipStream_t>(stream)};
  switch (dtype) {
    case PT_FLOAT32: return pt::launch_log_probs_bwd<float>(a);
    case PT_FLOAT64: return pt::launch_log_probs_bwd<double>(a);
    case PT_BFLOAT16: return pt::launch_log_probs_bwd<pt::bf16>(a);
    default: return pt::launch_log_probs_bwd<_Float16>(a);
  }
}

}  // extern "C"
