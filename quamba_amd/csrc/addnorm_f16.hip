// The residual sum with its norms, of fp16 rows (addnorm.hpp).
#include "addnorm.hpp"

namespace qa {
namespace lm {
int add_rmsnorm_f16(const QaAddNormParams& p, const AddNormShape& s, bool wide, hipStream_t stream) { return add_rmsnorm_of_type<_Float16>(p, s, wide, stream); }
}  // namespace lm
}  // namespace qa
