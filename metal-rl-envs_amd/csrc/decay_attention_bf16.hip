// The chunked walk's kernels for bfloat16 rows (decay_attention.h).
#include "decay_attention.h"

namespace hipenvs {
namespace da {
template int launch_chunks<__bf16>(const Walks&, bool, hipStream_t);
}  // namespace da
}  // namespace hipenvs
