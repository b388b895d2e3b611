// Instantiates the token log-probability kernels for one storage type.
#include "token_log_probs_series.inl"

namespace pt {
template int launch_log_probs<bf16>(const LogProbArgs&);
template int launch_log_probs_bwd<bf16>(const LogProbBwdArgs&);
}  // namespace pt
