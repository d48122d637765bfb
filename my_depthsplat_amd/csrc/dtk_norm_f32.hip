// The layer norm's kernels for f32 rows.
#include "dtk_norm.h"

namespace dtk {
template void run_fwd<float>(const FwdArgs&, const Shape&, hipStream_t);
template void run_bwd<float>(const BwdArgs&, int, const Shape&, bool, hipStream_t);
}  // namespace dtk
