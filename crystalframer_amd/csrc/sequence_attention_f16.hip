// Attention between sequences of float16 (a source of its own, so that the three types compile side by side).
#include "sequence_attention.hpp"

namespace cfh {
template void sequence_attention_forward<f16>(const SequenceAttention&, const AttentionPlan&, f16*, f16*, float*, float*, hipStream_t);
template void sequence_attention_backward<f16>(const SequenceAttention&, const AttentionGradPlan&, AttentionGrads, void*, float*, hipStream_t);
}  // namespace cfh
