// The attention's kernels for bf16 rows.
#include "dtk_attention.h"

namespace dtk {
DTK_ATTEND(, bf16)
}  // namespace dtk
