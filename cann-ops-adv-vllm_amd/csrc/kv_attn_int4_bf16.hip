// Attention over the 4-bit cache, bfloat16 queries (kv_attn_int4.inc).
#include "kv_attn_int4.inc"

namespace spfa {

hipError_t int4_attention_bf16(const Int4AttnParams& p, hipStream_t s, int* resident) { return int4_attention_tu<true>(p, s, resident); }

}  // namespace spfa
