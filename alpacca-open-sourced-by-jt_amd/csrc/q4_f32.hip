// The attention over 4-bit pools for float32 queries (q4_kernel.h).
#include "q4_kernel.h"

namespace alpx {

Q4Kernel q4_kernel_f32(int head_dim, int cols) { return pick<float>(head_dim, cols); }

}  // namespace alpx
