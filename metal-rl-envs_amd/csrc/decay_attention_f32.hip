// The chunked walk's kernels for float32 rows (decay_attention.h).
#include "decay_attention.h"

namespace hipenvs {
namespace da {
template int launch_chunks<float>(const Walks&, bool, hipStream_t);
}  // namespace da
}  // namespace hipenvs
