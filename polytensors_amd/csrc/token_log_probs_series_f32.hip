// Instantiates the token log-probability kernels for one storage type.
#include "token_log_probs_series.inl"

namespace pt {
template int launch_log_probs<float>(const LogProbArgs&);
template int launch_log_probs_bwd<float>(const LogProbBwdArgs&);
}  // namespace pt
