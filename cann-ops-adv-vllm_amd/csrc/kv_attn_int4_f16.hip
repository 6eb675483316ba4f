// Attention over the 4-bit cache, float16 queries (kv_attn_int4.inc), and the choice between the two translation units.
#include "kv_attn_int4.inc"

namespace spfa {

hipError_t int4_attention_f16(const Int4AttnParams& p, hipStream_t s, int* resident) { return int4_attention_tu<false>(p, s, resident); }
hipError_t int4_attention_bf16(const Int4AttnParams& p, hipStream_t s, int* resident);
static hipError_t any(const Int4AttnParams& p, hipStream_t s, int* resident) {
    return p.q_dtype == kBF16 ? int4_attention_bf16(p, s, resident) : int4_attention_f16(p, s, resident);
}

hipError_t launch_int4_attention(const Int4AttnParams& p, hipStream_t s) { return any(p, s, nullptr); }
int int4_attention_resident(const Int4AttnParams& p) {
    int n = 0;
    if (device_cu_count() <= 0 || any(p, nullptr, &n) != hipSuccess) { (void)hipGetLastError(); return 0; }
    return n;
}
long long int4_attention_part_bytes(const Int4AttnParams& p) { return (long long)(p.rows_tile / 16) * (p.D / 16 * 2 + 1) * 128 * 4; }

}  // namespace spfa
