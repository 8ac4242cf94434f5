// The row gradients of mx_linear.hip in bf16.
#include "mx_input.h"

namespace odie {
template int launch_mx_input<__bf16>(const MxInputArgs&, hipStream_t);
}
