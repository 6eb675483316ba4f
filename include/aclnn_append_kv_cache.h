/*
 * AppendKvCache: the new rows of a step into the paged cache, with the position rotation applied on the way.
 *
 * No counterpart in the reference, whose ops only read the cache.  One launch rotates q and K, quantises where the cache
 * asks for it and writes every row to its place.
 *
 * Tokens: rows queryStart[b] .. queryStart[b + 1] of key / value / query belong to sequence b (queryStart [B + 1] i32;
 * NULL: row b, one per sequence, T = B).  The i-th of n rows stands at position seqLen[b] - n + i — seqLen counts the
 * sequence with its new rows — and is stored in row pos % blockSize of page blockTable[b][pos / blockSize].  Nothing is
 * stored for a position outside [0, table columns * blockSize) or a table entry outside the pool (the usual -1); two
 * sequences that name the same page and row leave one of their tokens there, unspecified which.
 *
 * key, value [T, Hkv, D], query [T, Hq, D] (or NULL): f16 | bf16, channels contiguous, any token and head stride (views
 * of one projection's output).  queryOut: query's shape; it may be query itself and
 * overlaps nothing else.
 *
 * cosSin [positions, R] float32 or the rows' dtype, R even <= D: R / 2 cosines, then R / 2 sines (NULL: no rotation).
 * Channel pairs (i, i + R / 2), or (2 i, 2 i + 1) with interleaved, turn by the angles of the row's position —
 * positions[t] where given ([T] i32), else the position in the sequence; channels from R on pass through.  Computed in
 * fp32, rounded once.  A row whose table row does not exist is not stored and its queryOut row is zero.
 *
 * Cache types (keyCacheInout / valueCacheInout), head dims 32, 64, 128, 256, 512:
 *   rows' dtype  [blocks, bs, Hkv * D], [blocks, bs, Hkv, D] or [blocks, Hkv, bs, D], as the attention ops take them
 *   int8         the same shapes; code = clamp(round_to_even(x / scale - offset)) with antiquantScale / antiquantOffset
 *                [2, Hkv, D] | [2] (antiquantMode 0) or [2, Hkv] (2) in the rows' dtype, keys first — the inverse of the
 *                attention ops' (code + offset) * scale.  NaN and scale 0: code 0
 *   uint8        4 bits (D <= 256): K codes [blocks, Hkv, bs, D / 2] (byte i: channel 2 i in the low bits, 2 i + 1 in the
 *                high bits), V codes [blocks, Hkv, bs / 4, D / 2, 4] (the same bytes, those of four consecutive tokens
 *                side by side), keyParamsInout / valueParamsInout float16 [blocks, Hkv, bs, 2]: scale and zero of every
 *                token.  With lo / hi the row's least and largest value: scale = f16(min((hi - lo) / 15, 65504)),
 *                zero = f16(lo), code = clamp(round_to_even((x - zero) / scale), 0, 15); a value outside float16 saturates.
 *                A row that holds a NaN or an infinity gets scale 0 and a NaN zero.
 *
 * zeroRest: queryOut rows that are in no sequence (behind queryStart[B]) are set to zero; 0 leaves them as they are.
 * Workspace size is 0.
 */
#ifndef SPFA_ACLNN_APPEND_KV_CACHE_H_
#define SPFA_ACLNN_APPEND_KV_CACHE_H_
#include "acl_shim.h"
#ifdef __cplusplus
extern "C" {
#endif
SPFA_API aclnnStatus aclnnAppendKvCacheGetWorkspaceSize(
    const aclTensor* key, const aclTensor* value, const aclTensor* query, const aclTensor* cosSin, const aclTensor* positions,
    const aclTensor* blockTable, const aclTensor* seqLen, const aclTensor* queryStart, const aclTensor* antiquantScale,
    const aclTensor* antiquantOffset, int64_t blockSize, int64_t interleaved, int64_t antiquantMode, int64_t zeroRest,
    const aclTensor* keyCacheInout, const aclTensor* valueCacheInout, const aclTensor* keyParamsInout,
    const aclTensor* valueParamsInout, const aclTensor* queryOut, uint64_t* workspaceSize, aclOpExecutor** executor);
SPFA_API aclnnStatus aclnnAppendKvCache(void* workspace, uint64_t workspaceSize, aclOpExecutor* executor, aclrtStream stream);
#ifdef __cplusplus
}
#endif
#endif
