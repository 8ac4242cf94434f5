// The products of mx_linear.hip with fp32 outside the 4 bits.
#include "mx_kernels.h"

ODIE_MX_FOR(float)
