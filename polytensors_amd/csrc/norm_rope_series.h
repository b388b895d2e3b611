// Launch interface of the per-head norm and rotation kernels (definitions in norm_rope_series.inl).
#pragma once

#include "pt_common.h"

namespace pt {

struct NormRopeArgs {
  int degree;
  int n_ops;
  const pt_norm_rope_operand* ops;
  int64_t batch, length, head_dim, rotary;
  int interleaved;
  const void* cos;
  const void* sin;
  int64_t table_rows;
  const int64_t* positions;       // null: 0, 1, .. along the length
  int64_t position_batch_stride;  // 0: the same positions for every batch entry
  double eps;
  void* workspace;                // backward with weight gradients
  hipStream_t stream;
};

template <typename T>
int launch_norm_rope(const NormRopeArgs& a);

template <typename T>
int launch_norm_rope_bwd(const NormRopeArgs& a);

// Rows of partial weight gradients (one a block, four blocks a compute unit) of an operand of `rows` heads. More blocks take the
// reduction longer than they save, fewer leave the device idle (degree 3 as in norm_rope_series.inl: 109 us with 1024, 116 with 4096).
constexpr int64_t kRopeMaxPartials = 1024;
inline int64_t norm_rope_partials(int64_t rows) { return rows < kRopeMaxPartials ? rows : kRopeMaxPartials; }

}  // namespace pt
