// The products of linear.hip on fp16 tensors.
#include "linear_kernels.h"

ODIE_LINEAR_FOR(_Float16)
