// The residual norms for rows of float32 (a source of its own, so that the three types compile side by side).
#include "residual_norm.hpp"

namespace cfh {
template void residual_norm_forward<float>(const ResidualNorm&, float*, float*, float*, hipStream_t);
template void residual_norm_backward<float>(const ResidualNorm&, NormGrads, int64_t, float*, hipStream_t);
}  // namespace cfh
