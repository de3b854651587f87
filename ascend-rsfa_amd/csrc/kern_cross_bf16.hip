// Instantiations of the forward kernel for cross attention, bfloat16.
#include "kern_cross.hpp"

using namespace rsfa;

RSFA_DEFINE_CROSS_LIST(kernels_cross_bf16, TypeBF16, 1)
