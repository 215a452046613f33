// The residual-norm kernels (grace_resnorm.h) for a residual of type float and a block of type bf16_t.
#include "grace_resnorm.h"

namespace grace {
namespace resnorm {
GRACE_RESNORM_DECLARE(, float, bf16_t)
}  // namespace resnorm
}  // namespace grace
