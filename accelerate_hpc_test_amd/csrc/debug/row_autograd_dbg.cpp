// Debug build of runtime/row_autograd.cpp (module accelerate_hpc_test_amd._C_debug).
#define ACC_DEBUG_BOUNDS 1
#include "../runtime/row_autograd.cpp"
