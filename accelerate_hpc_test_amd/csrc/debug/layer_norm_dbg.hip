// Debug build of kernels/layer_norm.hip: same source with the device bounds checks compiled in (kernels/common.h).
#define ACC_DEBUG_BOUNDS 1
#include "../kernels/layer_norm.hip"
