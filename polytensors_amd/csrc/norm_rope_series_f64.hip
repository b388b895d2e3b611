// Instantiates the per-head norm and rotation kernels for one storage type.
#include "norm_rope_series.inl"

namespace pt {
template int launch_norm_rope<double>(const NormRopeArgs&);
template int launch_norm_rope_bwd<double>(const NormRopeArgs&);
}  // namespace pt
