// The attention over 4-bit pools for bfloat16 queries (q4_kernel.h).
#include "q4_kernel.h"

namespace alpx {

Q4Kernel q4_kernel_bf16(int head_dim, int cols) { return pick<bf16_t>(head_dim, cols); }

}  // namespace alpx
