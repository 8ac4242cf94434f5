// The products of linear.hip on fp32 tensors.
#include "linear_kernels.h"

ODIE_LINEAR_FOR(float)
