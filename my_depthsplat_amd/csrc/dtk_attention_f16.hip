// The attention's kernels for f16 rows.
#include "dtk_attention.h"

namespace dtk {
DTK_ATTEND(, f16)
}  // namespace dtk
