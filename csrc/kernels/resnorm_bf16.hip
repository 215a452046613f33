// The residual-norm kernels (grace_resnorm.h) for blocks of type bf16.
#include "grace_resnorm.h"

namespace grace {
namespace resnorm {
GRACE_RESNORM_DECLARE(, bf16_t, bf16_t)
GRACE_RESNORM_DECLARE(, float, bf16_t)
}  // namespace resnorm
}  // namespace grace
