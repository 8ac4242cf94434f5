// The row gradients of mx_linear.hip in fp16.
#include "mx_input.h"

namespace odie {
template int launch_mx_input<_Float16>(const MxInputArgs&, hipStream_t);
}
