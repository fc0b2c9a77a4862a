// The residual norms for rows of bfloat16 (a source of its own, so that the three types compile side by side).
#include "residual_norm.hpp"

namespace cfh {
template void residual_norm_forward<bf16>(const ResidualNorm&, bf16*, bf16*, float*, hipStream_t);
template void residual_norm_backward<bf16>(const ResidualNorm&, NormGrads, int64_t, float*, hipStream_t);
}  // namespace cfh
