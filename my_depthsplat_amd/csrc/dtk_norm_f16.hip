// The layer norm's kernels for f16 rows.
#include "dtk_norm.h"

namespace dtk {
template void run_fwd<f16>(const FwdArgs&, const Shape&, hipStream_t);
template void run_bwd<f16>(const BwdArgs&, int, const Shape&, bool, hipStream_t);
}  // namespace dtk
