/*
 * PagedAttentionInt4: attention over a paged cache held in 4 bits, as AppendKvCache writes it (layouts there).
 *
 * K_t = scale_t code_t + zero_t, V likewise with parameters of its own;
 * attentionOut[row] = softmax(scaleValue * query[row] . K^T over the tokens the row sees) V, fp32 accumulation.
 *
 * query [T, Hq, D] f16 | bf16, D in {32, 64, 128, 256}, channels contiguous, any token and head stride; groups of up to
 * 64 heads.  Rows belong to sequences as in AppendKvCache (queryStart NULL: decode, one row per sequence); the i-th of n
 * rows of sequence b stands at position seqLen[b] - n + i.  causal: it sees the tokens up to its own; otherwise all
 * seqLen[b] tokens (a cache of another sequence: an encoder's states).  Tokens behind the table and pages whose table entry
 * lies outside the pool are not there.  A row that sees no token (length 0, more rows than tokens) gets zeros.
 * maxQueryLen (with queryStart): most rows of a sequence.  It decides how rows and tokens are shared out, so the exact number
 * is the quickest; with any other one from 1 on the results are the same up to rounding (order of the sums; weights in one
 * float16 part or two).
 *
 * Parameters may be of any sign and size.  Beyond rounding a row depends neither on other rows nor on tokens that it does not
 * see.  What is rounded besides the output: a weight times its token's value scale, to float16 (2^-11 of it; at least 2^-31 of the largest
 * such product that its tokens' scales and probabilities allow), or to two float16 parts where a sequence's rows of a kv head
 * are at most eight.  A bfloat16 row whose largest element times scaleValue reaches 2^117 comes out NaN.
 *
 * blockPosition [B, Hq | Hkv, P] i32 (or NULL): logical pages of one row per sequence, as CentSelect yields them, a row
 * ending at its first entry outside the table (0x7fffffff among them); tokens from seqLen[b] on are not seen.  P <= 4096.
 *
 * attentionOut: query's shape, contiguous; query's dtype or float32; query itself or memory of its own.  softmaxLse (or
 * NULL): float32 [T, Hq], the natural logarithm of every row's sum of exponentials, -3.4e38 for a row without tokens.
 * zeroRest: rows in no sequence are set to zero (log-sum-exp -3.4e38); 0 leaves them as they are.
 *
 * Results are bit-reproducible for the same shapes and lengths on the same device.  The workspace holds arrival counters and
 * the partial states of work that several workgroups share; its contents do not matter.
 */
#ifndef SPFA_ACLNN_PAGED_ATTENTION_INT4_H_
#define SPFA_ACLNN_PAGED_ATTENTION_INT4_H_
#include "acl_shim.h"
#ifdef __cplusplus
extern "C" {
#endif
SPFA_API aclnnStatus aclnnPagedAttentionInt4GetWorkspaceSize(
    const aclTensor* query, const aclTensor* keyCache, const aclTensor* valueCache, const aclTensor* keyParams,
    const aclTensor* valueParams, const aclTensor* blockTable, const aclTensor* seqLen, const aclTensor* queryStart,
    const aclTensor* blockPosition, double scaleValue, int64_t numKeyValueHeads, int64_t blockSize, int64_t maxQueryLen,
    int64_t causal, int64_t zeroRest, const aclTensor* attentionOut, const aclTensor* softmaxLse, uint64_t* workspaceSize,
    aclOpExecutor** executor);
SPFA_API aclnnStatus aclnnPagedAttentionInt4(void* workspace, uint64_t workspaceSize, aclOpExecutor* executor, aclrtStream stream);
#ifdef __cplusplus
}
#endif
#endif
