// Attention between sequences of bfloat16 (a source of its own, so that the three types compile side by side).
#include "sequence_attention.hpp"

namespace cfh {
template void sequence_attention_forward<bf16>(const SequenceAttention&, const AttentionPlan&, bf16*, bf16*, float*, float*, hipStream_t);
template void sequence_attention_backward<bf16>(const SequenceAttention&, const AttentionGradPlan&, AttentionGrads, void*, float*, hipStream_t);
}  // namespace cfh
