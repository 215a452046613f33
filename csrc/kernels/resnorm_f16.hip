// The residual-norm kernels (grace_resnorm.h) for blocks of type f16.
#include "grace_resnorm.h"

namespace grace {
namespace resnorm {
GRACE_RESNORM_DECLARE(, half_t, half_t)
GRACE_RESNORM_DECLARE(, float, half_t)
}  // namespace resnorm
}  // namespace grace
