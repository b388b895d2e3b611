// Launch interface of the dropout kernels (definitions in dropout_series.inl).
#pragma once

#include "pt_common.h"

namespace pt {

struct DropoutArgs {
  int orders;
  const void* const* x;
  void* const* y;
  int64_t numel;
  double p;
  const int64_t* seed;   // device
  hipStream_t stream;
};

template <typename T>
int launch_dropout(const DropoutArgs& a);

}  // namespace pt
