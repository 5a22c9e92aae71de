// The attention over 4-bit pools for float16 queries (q4_kernel.h).
#include "q4_kernel.h"

namespace alpx {

Q4Kernel q4_kernel_f16(int head_dim, int cols) { return pick<f16_t>(head_dim, cols); }

}  // namespace alpx
