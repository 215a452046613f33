// The residual-norm kernels (grace_resnorm.h) for a residual of type bf16_t and a block of type bf16_t.
#include "grace_resnorm.h"

namespace grace {
namespace resnorm {
GRACE_RESNORM_DECLARE(, bf16_t, bf16_t)
}  // namespace resnorm
}  // namespace grace
