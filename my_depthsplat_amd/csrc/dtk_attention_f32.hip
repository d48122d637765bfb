// The attention's kernels for f32 rows.
#include "dtk_attention.h"

namespace dtk {
DTK_ATTEND(, float)
}  // namespace dtk
