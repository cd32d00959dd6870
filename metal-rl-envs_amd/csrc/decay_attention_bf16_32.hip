// The chunked walk's kernels for bfloat16 rows and states of up to 32 rows (decay_attention.h).
#define HIPENVS_DA_DEFINE
#include "decay_attention.h"

namespace hipenvs {
namespace da {
HIPENVS_DA_ROWS(, __bf16, 32)
}  // namespace da
}  // namespace hipenvs
