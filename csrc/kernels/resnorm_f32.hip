// The residual-norm kernels (grace_resnorm.h) for a residual of type float and a block of type float.
#include "grace_resnorm.h"

namespace grace {
namespace resnorm {
GRACE_RESNORM_DECLARE(, float, float)
}  // namespace resnorm
}  // namespace grace
