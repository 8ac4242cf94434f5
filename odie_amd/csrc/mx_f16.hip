// The products of mx_linear.hip with fp16 outside the 4 bits.
#include "mx_kernels.h"

ODIE_MX_FOR(_Float16)
