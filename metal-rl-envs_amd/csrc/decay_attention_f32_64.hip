// The chunked walk's kernels for float32 rows and states of up to 64 rows (decay_attention.h).
#define HIPENVS_DA_DEFINE
#include "decay_attention.h"

namespace hipenvs {
namespace da {
HIPENVS_DA_ROWS(, float, 64)
}  // namespace da
}  // namespace hipenvs
