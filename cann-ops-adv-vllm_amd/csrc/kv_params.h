// Launch descriptors of the KV-cache operators (append, read back, attention over a 4-bit cache), shared by the host
// planner (aclnn_kv_ops.inc) and the kernels (kv_cache.hip, kv_assign_int4.hip, kv_attn_int4.inc).
//
// The 4-bit cache.  A token of a kv head is D codes 0 .. 15 and a pair (scale, zero) of float16: x = scale * code + zero.
//   K codes  uint8 [blocks, Hkv, bs, D / 2]         byte i of a token: channel 2 i (low bits), channel 2 i + 1 (high bits)
//   V codes  uint8 [blocks, Hkv, bs / 4, D / 2, 4]  the same bytes with those of four consecutive tokens side by side, so
//            that a 32-bit word is four tokens x two channels: what the matrix cores want as operand of P.V (a run of
//            tokens for one channel) comes out of memory by masking, without a transposition
//   params   float16 [blocks, Hkv, bs, 2]           (scale, zero) of every token, one tensor for K, one for V
#pragma once
#include <hip/hip_runtime_api.h>
#include <stdint.h>

#include "spfa_params.h"

namespace spfa {

// The tokens of a call.  Rows query_start[b] .. query_start[b + 1] belong to sequence b (null: row b, one per sequence);
// the i-th of n rows stands at position seq_len[b] - n + i and lives in row pos % block_size of page
// block_table[b][pos / block_size].  A position outside [0, max_page * block_size) and a table entry outside the pool
// name no place.
struct TokenMap {
    const int32_t* query_start;   // [B + 1] or null
    const int32_t* seq_len;       // [B]
    const int32_t* block_table;   // [>= B, max_page]
    int T, B, max_page, block_size, n_blocks;
};

// A paged cache of any type.  16-bit and int8: [blocks, bs, Hkv, D] or [blocks, Hkv, bs, D]; 4 bits as above.
struct CacheView {
    void* k;
    void* v;
    long long blk_stride, tok_stride, head_stride;   // bytes (4-bit V: tok_stride per token within whole quads)
    int dtype;                    // kF16 | kBF16 | kI8 | kI4
    uint32_t* k_params;           // 4 bits: [blocks, Hkv, bs] (scale, zero) pairs of float16
    uint32_t* v_params;
    const void* antiq_scale;      // int8: key parameters first; x = (code + offset) * scale
    const void* antiq_offset;     // or null
    int antiq_layout;             // 0 [2, Hkv, D], 1 [2], 2 [2, Hkv]
    int antiq_dtype;              // kF16 | kBF16
};

struct AppendParams {
    TokenMap map;
    CacheView cache;
    const void* q;                // [T, Hq, D] or null
    void* q_out;
    const void* k;                // [T, Hkv, D]
    const void* v;
    long long q_tok, q_head, qo_tok, qo_head, k_tok, k_head, v_tok, v_head;   // elements
    int dtype;                    // kF16 | kBF16
    int Hq, Hkv, D;
    const void* cos_sin;          // [cs_rows, rot]: rot / 2 cosines, then rot / 2 sines; null: no rotation
    int cs_dtype;                 // kF32 | kF16 | kBF16
    int cs_rows, rot, interleaved;
    const int32_t* positions;     // [T] rows of cos_sin, or null: the position in the sequence
    int wide;                     // every row, table row and chunk of 8 channels starts at a multiple of 16 bytes
    int zero_rest;                // rows that are in no sequence: 1 zeros, 0 left as they are
    int tokens_per_wg, head_split;
};

struct GatherParams {
    TokenMap map;
    CacheView cache;
    void* k_out;                  // [T, Hkv, D]
    void* v_out;
    int dtype;                    // kF16 | kBF16
    int Hkv, D;
    int zero_rest;
    int tokens_per_wg, head_split;
};

struct Int4AttnParams {
    TokenMap map;
    const void* q;                // [T, Hq, D]
    long long q_tok, q_head;      // elements
    int q_wide;                   // rows start at multiples of 16 bytes
    void* out;                    // [T, Hq, D]
    int q_dtype, out_dtype;       // kF16 | kBF16; out: the same or kF32
    const uint8_t* kcache;
    const uint8_t* vcache;
    const uint32_t* k_params;
    const uint32_t* v_params;
    int Hq, Hkv, G, D;
    float scale;
    int causal;
    int zero_rest;
    float* lse;                   // [T, Hq] or null
    // page lists (one row of a sequence each): [B, list_rows, P], list_rows = Hq or Hkv; null: all tokens
    const int32_t* lists;
    int list_rows, P;
    // plan
    int nt;                       // 16-row tiles a wave keeps
    int row_waves;                // 1, 2, 4: groups of rows among the four waves of a workgroup; the rest shares the tokens
    int rows_tile;                // rows of a work item: 16 * nt * row_waves
    int wide_line;                // the steps of all items may exceed 31 bits
    int most_tiles;               // work items of one (sequence, kv head), at most
    int workers;                  // workgroups (all tokens) / workgroups per list (n_split)
    int min_steps;                // fewest 32-token steps worth a workgroup of their own
    int item_steps;               // what an item costs besides its steps, in steps
    unsigned g_magic;             // ceil(2^32 / G), 0 for a group of one
    int paired;                   // 32 tokens never cross a page (block_size a multiple of 32)
    unsigned page_magic;          // ceil(2^32 / (block_size / 16)), 0 for a block size of 16
    unsigned* counters;           // arrivals per split item, zeroed before and left zeroed
    float* parts;                 // partial states
};

hipError_t launch_append(const AppendParams& p, hipStream_t s);
hipError_t launch_gather(const GatherParams& p, hipStream_t s);
hipError_t launch_int4_attention(const Int4AttnParams& p, hipStream_t s);
// Workgroups of the planned kernel that the current device holds at once (0: no device).
int int4_attention_resident(const Int4AttnParams& p);
// Bytes of one partial state (two per workgroup; with page lists one per workgroup).
long long int4_attention_part_bytes(const Int4AttnParams& p);
constexpr int kInt4StepTokens = 32;
constexpr int kInt4MaxList = 4096;     // entries of a page list (8 bytes of LDS each)

}  // namespace spfa
