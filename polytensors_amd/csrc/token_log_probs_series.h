// Launch interface of the token log-probability kernels (definitions in token_log_probs_series.inl).
#pragma once

#include "pt_common.h"

namespace pt {

struct LogProbArgs {
  int degree;
  const void* const* z;
  int64_t rows, classes, row_stride;
  const int64_t* tokens;
  int64_t ignore_index;
  double softcap;   // 0: none
  int top;
  void* const* log_probs;
  void* const* entropy;
  int64_t* top_tokens;
  void* const* top_log_probs;
  void* const* lse;
  void* workspace;
  hipStream_t stream;
};

template <typename T>
int launch_log_probs(const LogProbArgs& a);

// Gradient series: dz = -p (*) (c + c_H (*) (log p + H)) + the cotangents at their tokens.
struct LogProbBwdArgs {
  int degree;
  const void* const* z;
  int64_t rows, classes, row_stride;
  const int64_t* tokens;
  int64_t ignore_index;
  double softcap;
  int top;
  const int64_t* top_tokens;
  const void* const* lse;       // [rows] an order, arithmetic type
  const void* const* entropy;   // [rows] an order
  const void* const* cot_log_probs;       // [rows] an order, or null
  const void* const* cot_entropy;         // [rows] an order, or null
  const void* const* cot_top_log_probs;   // [rows, top] an order, or null
  void* const* dz;              // [rows, classes] contiguous
  hipStream_t stream;
};

template <typename T>
int launch_log_probs_bwd(const LogProbBwdArgs& a);

// Pieces that a row is cut into so that few rows fill the device, and the bytes of their partial results.
int64_t log_prob_splits(int64_t rows, int64_t classes, int elem_size, bool backward);
size_t log_prob_workspace(int degree, int64_t rows, int64_t classes, int top, int elem_size);

}  // namespace pt
