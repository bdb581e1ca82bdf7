// The linear layers' kernels for fp32 operands.
#include "linear_kernels.h"

namespace tch {

int launch_linear_f32(Context* ctx, int mode, LinearArgs& a) { return launch_linear_typed<float>(ctx, mode, a); }

}  // namespace tch
