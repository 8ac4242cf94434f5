// The products of linear.hip on bf16 tensors.
#include "linear_kernels.h"

ODIE_LINEAR_FOR(__bf16)
