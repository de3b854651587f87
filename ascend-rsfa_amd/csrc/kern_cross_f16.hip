// Instantiations of the forward kernel for cross attention, float16.
#include "kern_cross.hpp"

using namespace rsfa;

RSFA_DEFINE_CROSS_LIST(kernels_cross_f16, TypeF16, 0)
