/*
 * GatherKvCache: rows of a paged cache back in 16 bits — the inverse of AppendKvCache (aclnn_append_kv_cache.h): the same
 * cache types and the same naming of tokens by blockTable, seqLen and queryStart (the last n tokens of every sequence).
 *
 * keyOut, valueOut [T, Hkv, D] f16 | bf16, contiguous, not overlapping: x = code * scale + zero (4 bits), (code + offset) * scale (int8)
 * or the element itself, rounded once to the output's dtype.  A 16-bit cache has the output's dtype; int8 parameters have it too.
 * Tokens of a sequence without a place in the cache (see there) come out as zeros.  zeroRest: the same for rows in no
 * sequence; 0 leaves those as they are.  Workspace size is 0.
 */
#ifndef SPFA_ACLNN_GATHER_KV_CACHE_H_
#define SPFA_ACLNN_GATHER_KV_CACHE_H_
#include "acl_shim.h"
#ifdef __cplusplus
extern "C" {
#endif
SPFA_API aclnnStatus aclnnGatherKvCacheGetWorkspaceSize(
    const aclTensor* keyCache, const aclTensor* valueCache, const aclTensor* keyParams, const aclTensor* valueParams,
    const aclTensor* blockTable, const aclTensor* seqLen, const aclTensor* queryStart, const aclTensor* antiquantScale,
    const aclTensor* antiquantOffset, int64_t blockSize, int64_t antiquantMode, int64_t zeroRest, const aclTensor* keyOut,
    const aclTensor* valueOut, uint64_t* workspaceSize, aclOpExecutor** executor);
SPFA_API aclnnStatus aclnnGatherKvCache(void* workspace, uint64_t workspaceSize, aclOpExecutor* executor, aclrtStream stream);
#ifdef __cplusplus
}
#endif
#endif
