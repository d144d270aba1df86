// Debug build of kernels/token_logprobs.hip: same source with the device bounds checks compiled in (kernels/common.h).
#define ACC_DEBUG_BOUNDS 1
#include "../kernels/token_logprobs.hip"
