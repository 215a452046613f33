// The residual-norm kernels (grace_resnorm.h) for a residual of type half_t and a block of type half_t.
#include "grace_resnorm.h"

namespace grace {
namespace resnorm {
GRACE_RESNORM_DECLARE(, half_t, half_t)
}  // namespace resnorm
}  // namespace grace
