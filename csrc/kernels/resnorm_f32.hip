// The residual-norm kernels (grace_resnorm.h) for blocks of type f32.
#include "grace_resnorm.h"

namespace grace {
namespace resnorm {
GRACE_RESNORM_DECLARE(, float, float)
}  // namespace resnorm
}  // namespace grace
