// The linear layers' kernels for bf16 operands.
#include "linear_kernels.h"

namespace tch {

int launch_linear_bf16(Context* ctx, int mode, LinearArgs& a) { return launch_linear_typed<bf16>(ctx, mode, a); }

}  // namespace tch
