// Attention between sequences of float32 (a source of its own, so that the three types compile side by side).
#include "sequence_attention.hpp"

namespace cfh {
template void sequence_attention_forward<float>(const SequenceAttention&, const AttentionPlan&, float*, float*, float*, float*, hipStream_t);
template void sequence_attention_backward<float>(const SequenceAttention&, const AttentionGradPlan&, AttentionGrads, void*, float*, hipStream_t);
}  // namespace cfh
