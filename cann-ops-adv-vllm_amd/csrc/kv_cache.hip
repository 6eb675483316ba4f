// Writing and reading a paged KV cache (gfx950): append (rotation, quantisation and placement in one pass over the new
// rows) and read-back (rows in 16 bits).  Both move bytes and little else, so what matters is that every row is read
// once in whole 16-byte pieces and that small calls are one short launch.
#include "kv_params.h"

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace spfa {
namespace {

#include "spfa_common.inc"

constexpr int kTokMax = 16;        // tokens a workgroup deals with

// Where a token of the call lives.
struct Place {
    int seq;        // sequence, or -1: the row is in none
    int page;       // physical page, or -1: nothing is stored for it
    int row;        // row in the page
    int pos;        // position in the sequence (-1: none)
};

// The places of tokens [t0, t0 + n), n <= kTokMax, computed by one wave: the sequence of a token is the number of
// sequences that end at or before it, counted 64 at a time by a ballot (one load latency for 64 sequences; a binary
// search per token is a chain of them).
__device__ __forceinline__ void find_places(const TokenMap& m, int t0, int n, Place* out, int lane) {
    int mine = t0 + lane, b = mine;
    if (m.query_start) {
        b = 0;
        for (int base = 0; base < m.B; base += 64) {
            const int end = base + lane < m.B ? m.query_start[base + lane + 1] : 0x7fffffff;
            for (int j = 0; j < n; ++j) {
                const int c = __popcll(__ballot(end <= t0 + j));
                if (lane == j) b += c;
            }
        }
    }
    if (lane < n) {
        Place pl{-1, -1, 0, -1};
        if (mine < m.T && b < m.B) {
            const int first = m.query_start ? m.query_start[b] : b;
            const int end = m.query_start ? m.query_start[b + 1] : b + 1;
            if (mine >= first && mine < end) {
                pl.seq = b;
                const long long pos = (long long)m.seq_len[b] - ((long long)end - mine);
                if (pos >= 0 && pos < (long long)m.max_page * m.block_size) {
                    const int lp = (int)pos / m.block_size;
                    pl.pos = (int)pos;
                    pl.row = (int)pos - lp * m.block_size;
                    const int phys = m.block_table[(long long)b * m.max_page + lp];
                    pl.page = (phys >= 0 && phys < m.n_blocks) ? phys : -1;
                }
            }
        }
        out[lane] = pl;
    }
}

// Runs of stored tokens inside a quad of four (the unit of the 4-bit V layout): first token (index in the workgroup's
// range) and how many.  Returns their number.  One wave; n <= kTokMax.
__device__ __forceinline__ int find_quads(const Place* pl, int n, uint8_t* first, uint8_t* count, int lane) {
    bool lead = false;
    int len = 0;
    if (lane < n && pl[lane].page >= 0) {
        const Place me = pl[lane];
        lead = (me.row & 3) == 0 || lane == 0 || pl[lane - 1].page < 0 || pl[lane - 1].seq != me.seq;
        if (lead) {
            len = 1;
            while (len < 4 - (me.row & 3) && lane + len < n && pl[lane + len].page >= 0 && pl[lane + len].seq == me.seq) ++len;
        }
    }
    const unsigned long long leads = __ballot(lead);
    if (lead) {
        const int at = __popcll(leads & lanes_below(lane));
        first[at] = (uint8_t)lane;
        count[at] = (uint8_t)len;
    }
    return __popcll(leads);
}

__device__ __forceinline__ float load_elem(const void* p, int dtype, long long i) {
    return dtype == kF32 ? ((const float*)p)[i] : load_qk_elem(p, dtype, i);
}

// Eight consecutive channels of a 16-bit row.
__device__ __forceinline__ void load8(const void* base, long long off, int dtype, bool wide, float* f) {
    const uint16_t* p = (const uint16_t*)base + off;
    uint32_t w[4];
    if (wide) {
        const uint4 v = *(const uint4*)p;
        w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = (uint32_t)p[2 * i] | ((uint32_t)p[2 * i + 1] << 16);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[2 * i] = dtype == kBF16 ? bf16_lo(w[i]) : f16_bits((uint16_t)(w[i] & 0xffffu));
        f[2 * i + 1] = dtype == kBF16 ? bf16_hi(w[i]) : f16_bits((uint16_t)(w[i] >> 16));
    }
}
__device__ __forceinline__ uint32_t pack2(float a, float b, int dtype) {
    if (dtype == kBF16)
        return (uint32_t)__builtin_bit_cast(uint16_t, (__bf16)a) | ((uint32_t)__builtin_bit_cast(uint16_t, (__bf16)b) << 16);
    return (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)a) | ((uint32_t)__builtin_bit_cast(uint16_t, (_Float16)b) << 16);
}
__device__ __forceinline__ void store8(void* base, long long off, int dtype, bool wide, const float* f) {
    uint16_t* p = (uint16_t*)base + off;
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = pack2(f[2 * i], f[2 * i + 1], dtype);
    if (wide) {
        *(uint4*)p = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) { p[2 * i] = (uint16_t)w[i]; p[2 * i + 1] = (uint16_t)(w[i] >> 16); }
    }
}

// Rotation of the eight channels c0 .. c0 + 7 of a row: channel c < rot turns with its partner by the angle of its pair.
// The partner's value is read from the row again (a cache hit); all loads of a row come before its stores and one wave
// holds the whole row, so the output may be the input itself.
__device__ __forceinline__ void load_rotated(const AppendParams& p, const void* row, long long off, int c0, int cs_row, float* x) {
#pragma clang fp contract(off)   // two rounded products and a rounded sum: the same value whichever of the paths below takes the row
    load8(row, off + c0, p.dtype, p.wide != 0, x);
    if (!p.cos_sin || c0 >= p.rot) return;
    const long long cs = (long long)cs_row * p.rot;
    const int half = p.rot >> 1;
    if (p.interleaved) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int pair = (c0 >> 1) + i;
            if (pair < half) {
                const float c = load_elem(p.cos_sin, p.cs_dtype, cs + pair), s = load_elem(p.cos_sin, p.cs_dtype, cs + half + pair);
                const float a = x[2 * i], b = x[2 * i + 1];
                x[2 * i] = a * c - b * s;
                x[2 * i + 1] = b * c + a * s;
            }
        }
    } else if (p.wide && (half & 7) == 0) {
        const bool low = c0 < half;
        const int pair = low ? c0 : c0 - half;
        float y[8];
        load8(row, off + (low ? c0 + half : c0 - half), p.dtype, true, y);
        float cv[8], sv[8];
        if (p.cs_dtype == kF32) {
            const float4* cp = (const float4*)((const float*)p.cos_sin + cs + pair);
            const float4* sp = (const float4*)((const float*)p.cos_sin + cs + half + pair);
            const float4 c_0 = cp[0], c_1 = cp[1], s_0 = sp[0], s_1 = sp[1];
            cv[0] = c_0.x; cv[1] = c_0.y; cv[2] = c_0.z; cv[3] = c_0.w; cv[4] = c_1.x; cv[5] = c_1.y; cv[6] = c_1.z; cv[7] = c_1.w;
            sv[0] = s_0.x; sv[1] = s_0.y; sv[2] = s_0.z; sv[3] = s_0.w; sv[4] = s_1.x; sv[5] = s_1.y; sv[6] = s_1.z; sv[7] = s_1.w;
        } else {
            load8(p.cos_sin, cs + pair, p.cs_dtype, true, cv);
            load8(p.cos_sin, cs + half + pair, p.cs_dtype, true, sv);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = low ? x[i] * cv[i] - y[i] * sv[i] : x[i] * cv[i] + y[i] * sv[i];
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int c = c0 + i;
            if (c >= p.rot) break;
            const bool low = c < half;
            const int pair = low ? c : c - half;
            const float cc = load_elem(p.cos_sin, p.cs_dtype, cs + pair), ss = load_elem(p.cos_sin, p.cs_dtype, cs + half + pair);
            const float y = load_qk_elem(row, p.dtype, off + (low ? c + half : c - half));
            x[i] = low ? x[i] * cc - y * ss : x[i] * cc + y * ss;
        }
    }
}

// Scale, zero and codes of a row whose channels lie in `lanes` consecutive lanes, eight each.  The parameters are rounded
// to float16 first and the codes are taken against the rounded ones, so a value inside the representable range is off by
// at most half a step.  A NaN or infinity has no code: the zero becomes NaN and with it everything the row stands for.
__device__ __forceinline__ uint32_t quantise8(const float* x, int lanes, int lane, uint32_t* param) {
    float lo = fminf(fminf(fminf(x[0], x[1]), fminf(x[2], x[3])), fminf(fminf(x[4], x[5]), fminf(x[6], x[7])));
    float hi = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
    float nan = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) nan += x[i] * 0.f;   // NaN if any channel is not finite
    const unsigned long long bad = __ballot(nan != 0.f);
    const unsigned long long mine = lanes >= 64 ? ~0ull : ((1ull << lanes) - 1ull) << (lane & ~(lanes - 1));
    for (int step = 1; step < lanes; step <<= 1) {
        lo = fminf(lo, __shfl_xor(lo, step));
        hi = fmaxf(hi, __shfl_xor(hi, step));
    }
    const _Float16 s = (_Float16)fminf((hi - lo) * (1.f / 15.f), 65504.f);
    _Float16 z = (_Float16)fminf(fmaxf(lo, -65504.f), 65504.f);
    // the division proper: 16-bit inputs meet exact halves often, and a reciprocal's rounding would decide those
    const float zf = (float)z, sf = (float)s;
    uint32_t codes = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float c = sf > 0.f ? fminf(fmaxf(rintf((x[i] - zf) / sf), 0.f), 15.f) : 0.f;
        codes |= (uint32_t)(int)c << (4 * i);
    }
    uint16_t zb = __builtin_bit_cast(uint16_t, z), sb = __builtin_bit_cast(uint16_t, s);
    if (bad & mine) { zb = 0x7e00u; sb = 0; }
    *param = (uint32_t)sb | ((uint32_t)zb << 16);
    return codes;
}

// (x / scale - offset) rounded to the nearest even code, saturating; NaN becomes code 0, a scale of 0 code 0 as well.
__device__ __forceinline__ uint2 quantise8_int8(const CacheView& c, int which, int n2, int c0, int Hkv, int D, const float* x) {
    uint32_t w[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const long long at = which == 0 ? antiq_key_index(c.antiq_layout, n2, c0 + i, D)
                                        : antiq_value_index(c.antiq_layout, n2, c0 + i, D, Hkv);
        const float s = load_qk_elem(c.antiq_scale, c.antiq_dtype, at);
        const float o = c.antiq_offset ? load_qk_elem(c.antiq_offset, c.antiq_dtype, at) : 0.f;
        float y = s != 0.f ? x[i] / s - o : 0.f;
        if (!(y == y)) y = 0.f;
        const int code = (int)rintf(fminf(fmaxf(y, -128.f), 127.f));
        w[i / 4] |= (uint32_t)(code & 255) << (8 * (i % 4));
    }
    return make_uint2(w[0], w[1]);
}

// Address of eight channels of a 16-bit or int8 row, or of a 4-bit K row.
__device__ __forceinline__ char* cache_at(const CacheView& c, void* base, const Place& pl, int n2, int c0) {
    const long long off = (long long)pl.page * c.blk_stride + (long long)pl.row * c.tok_stride + (long long)n2 * c.head_stride;
    return (char*)base + off + (c.dtype == kI4 ? c0 / 2 : (c.dtype == kI8 ? c0 : 2 * c0));
}
// 4-bit V: the four 32-bit words (channel pairs) of eight channels in the quad that holds the token.
__device__ __forceinline__ char* quad_at(const CacheView& c, const Place& pl, int n2, int c0) {
    return (char*)c.v + (long long)pl.page * c.blk_stride + (long long)n2 * c.head_stride + (long long)(pl.row >> 2) * 4 * c.tok_stride +
           c0 / 2 * 4;
}
__device__ __forceinline__ long long param_at(const CacheView& c, const TokenMap& m, const Place& pl, int Hkv, int n2) {
    return ((long long)pl.page * Hkv + n2) * m.block_size + pl.row;
}
// codes of four tokens (8 channels each) -> the quad's words: word p holds byte (channel pair p) of token j at byte j
__device__ __forceinline__ uint4 transpose_codes(const uint32_t* c) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        w[i] = ((c[0] >> (8 * i)) & 255u) | (((c[1] >> (8 * i)) & 255u) << 8) | (((c[2] >> (8 * i)) & 255u) << 16) |
               (((c[3] >> (8 * i)) & 255u) << 24);
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// One workgroup: tokens_per_wg tokens (their places found once, by the first wave), all heads or a share of them
// (head_split workgroups).  D / 8 consecutive lanes hold a row, eight channels each.  The rows are dealt in the order
// q rows, K rows, V rows; 4-bit V rows go by quads of tokens, so that a whole quad is one 16-byte store per lane.
__global__ __launch_bounds__(256) void append_kernel(const AppendParams p) {
    __shared__ Place places[kTokMax];
    __shared__ uint8_t q_first[kTokMax], q_count[kTokMax];
    __shared__ int n_quads;
    const int lane = lane_id(), wave = wave_id();
    const int t0 = blockIdx.x * p.tokens_per_wg;
    const int n = min(p.tokens_per_wg, p.map.T - t0);
    if (wave == 0) {
        find_places(p.map, t0, n, places, lane);
        wave_lds_sync();
        if (p.cache.dtype == kI4) {
            const int k = find_quads(places, n, q_first, q_count, lane);
            if (lane == 0) n_quads = k;
        }
    }
    __syncthreads();
    const int lanes = p.D >> 3;                     // 4 .. 64
    const int sub = threadIdx.x & (lanes - 1);
    const int per_wg = 256 / lanes;
    const int c0 = sub * 8;
    const bool quads = p.cache.dtype == kI4;
    const int nq = p.q ? n * p.Hq : 0, nk = n * p.Hkv, nv = (quads ? n_quads : n) * p.Hkv;
    const int total = nq + nk + nv;
    // (whole waves stay in the loop: the reductions of a row cross its lanes)
    for (int i0 = blockIdx.y * per_wg; i0 < total; i0 += per_wg * gridDim.y) {
        const int i = i0 + (int)threadIdx.x / lanes;
        float x[8];
        if (i < nq) {
            const int j = i / p.Hq, h = i - j * p.Hq;
            const Place pl = places[j];
            const int t = t0 + j;
            const long long dst = (long long)t * p.qo_tok + (long long)h * p.qo_head + c0;
            const int cs = p.positions && pl.seq >= 0 ? p.positions[t] : pl.pos;
            const bool turn = pl.pos >= 0 && (!p.cos_sin || (cs >= 0 && cs < p.cs_rows));
            if (turn) load_rotated(p, p.q, (long long)t * p.q_tok + (long long)h * p.q_head, c0, cs, x);
            else
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = 0.f;
            if (pl.seq >= 0 || p.zero_rest) store8(p.q_out, dst, p.dtype, p.wide != 0, x);
        } else if (i < nq + nk || !quads) {
            const bool is_k = i < nq + nk;
            const int r = i - nq - (is_k ? 0 : nk);
            if (r >= nk) continue;                  // past the end (not with 4-bit V: no reductions here)
            const int j = r / p.Hkv, h = r - j * p.Hkv;
            const Place pl = places[j];
            const int t = t0 + j;
            const int cs = p.positions && pl.seq >= 0 ? p.positions[t] : pl.pos;
            const bool ok = pl.page >= 0 && (!p.cos_sin || (cs >= 0 && cs < p.cs_rows));
            if (!ok) continue;
            if (is_k) load_rotated(p, p.k, (long long)t * p.k_tok + (long long)h * p.k_head, c0, cs, x);
            else load8(p.v, (long long)t * p.v_tok + (long long)h * p.v_head + c0, p.dtype, p.wide != 0, x);
            char* dst = cache_at(p.cache, is_k ? p.cache.k : p.cache.v, pl, h, c0);
            if (p.cache.dtype == kI4) {
                uint32_t par;
                const uint32_t codes = quantise8(x, lanes, lane, &par);
                *(uint32_t*)dst = codes;
                if (sub == 0) p.cache.k_params[param_at(p.cache, p.map, pl, p.Hkv, h)] = par;
            } else if (p.cache.dtype == kI8) {
                *(uint2*)dst = quantise8_int8(p.cache, is_k ? 0 : 1, h, c0, p.Hkv, p.D, x);
            } else {
                store8(dst, 0, p.dtype, true, x);
            }
        } else {
            const int r = i - nq - nk;
            if (r >= nv) continue;
            const int u = r / p.Hkv, h = r - u * p.Hkv;
            const int j0 = q_first[u], cnt = q_count[u];
            const Place pl = places[j0];
            uint32_t codes[4] = {0, 0, 0, 0}, par[4];
            unsigned ok = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (e >= cnt) break;
                const int t = t0 + j0 + e;
                const int cs = p.positions ? p.positions[t] : places[j0 + e].pos;
                if (p.cos_sin && (cs < 0 || cs >= p.cs_rows)) continue;
                load8(p.v, (long long)t * p.v_tok + (long long)h * p.v_head + c0, p.dtype, p.wide != 0, x);
                codes[e] = quantise8(x, lanes, lane, &par[e]);
                ok |= 1u << e;
                if (sub == 0) p.cache.v_params[param_at(p.cache, p.map, pl, p.Hkv, h) + e] = par[e];
            }
            char* dst = quad_at(p.cache, pl, h, c0);
            if (ok == 15u) {
                *(uint4*)dst = transpose_codes(codes);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (ok >> e & 1u)
#pragma unroll
                        for (int b = 0; b < 4; ++b) dst[4 * b + (pl.row & 3) + e] = (char)(codes[e] >> (8 * b));
            }
        }
    }
}

__device__ __forceinline__ void dequantise8(uint32_t codes, uint32_t par, float* x) {
    const float s = f16_bits((uint16_t)(par & 0xffffu)), z = f16_bits((uint16_t)(par >> 16));
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = s * (float)((codes >> (4 * i)) & 15u) + z;
}

// Rows back in 16 bits; the work is dealt as in append_kernel.
__global__ __launch_bounds__(256) void gather_kernel(const GatherParams p) {
    __shared__ Place places[kTokMax];
    __shared__ uint8_t q_first[kTokMax], q_count[kTokMax];
    __shared__ int n_quads;
    const int lane = lane_id(), wave = wave_id();
    const int t0 = blockIdx.x * p.tokens_per_wg;
    const int n = min(p.tokens_per_wg, p.map.T - t0);
    if (wave == 0) {
        find_places(p.map, t0, n, places, lane);
        wave_lds_sync();
        if (p.cache.dtype == kI4) {
            const int k = find_quads(places, n, q_first, q_count, lane);
            if (lane == 0) n_quads = k;
        }
    }
    __syncthreads();
    const int lanes = p.D >> 3;
    const int sub = threadIdx.x & (lanes - 1);
    const int per_wg = 256 / lanes;
    const int c0 = sub * 8;
    const bool quads = p.cache.dtype == kI4;
    const int rows = n * p.Hkv, nv = quads ? n_quads * p.Hkv : 0;
    // K rows, V rows (4 bits: those without a place only, the others come by quads), V quads
    const int total = 2 * rows + nv;
    const long long row_elems = (long long)p.Hkv * p.D;
    for (int i0 = blockIdx.y * per_wg; i0 < total; i0 += per_wg * gridDim.y) {
        const int i = i0 + (int)threadIdx.x / lanes;
        float x[8];
        if (i < 2 * rows) {
            const bool is_k = i < rows;
            const int r = is_k ? i : i - rows;
            const int j = r / p.Hkv, h = r - j * p.Hkv;
            const Place pl = places[j];
            const long long dst = (long long)(t0 + j) * row_elems + (long long)h * p.D + c0;
            if (pl.page < 0) {
                if (pl.seq < 0 && !p.zero_rest) continue;
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = 0.f;
            } else {
                if (quads && !is_k) continue;
                const char* src = cache_at(p.cache, is_k ? p.cache.k : p.cache.v, pl, h, c0);
                if (p.cache.dtype == kI4) {
                    dequantise8(*(const uint32_t*)src, p.cache.k_params[param_at(p.cache, p.map, pl, p.Hkv, h)], x);
                } else if (p.cache.dtype == kI8) {
                    const uint2 w = *(const uint2*)src;
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const int code = (int)(int8_t)((e < 4 ? w.x : w.y) >> (8 * (e & 3)));
                        const long long at = is_k ? antiq_key_index(p.cache.antiq_layout, h, c0 + e, p.D)
                                                  : antiq_value_index(p.cache.antiq_layout, h, c0 + e, p.D, p.Hkv);
                        const float o = p.cache.antiq_offset ? load_qk_elem(p.cache.antiq_offset, p.cache.antiq_dtype, at) : 0.f;
                        x[e] = ((float)code + o) * load_qk_elem(p.cache.antiq_scale, p.cache.antiq_dtype, at);
                    }
                } else {
                    load8(src, 0, p.cache.dtype, true, x);
                }
            }
            store8(is_k ? p.k_out : p.v_out, dst, p.dtype, true, x);
        } else {
            const int r = i - 2 * rows;
            if (r >= nv) continue;
            const int u = r / p.Hkv, h = r - u * p.Hkv;
            const int j0 = q_first[u], cnt = q_count[u];
            const Place pl = places[j0];
            const uint4 w = *(const uint4*)quad_at(p.cache, pl, h, c0);
            const uint32_t* par = p.cache.v_params + param_at(p.cache, p.map, pl, p.Hkv, h);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (e >= cnt) break;
                const int sh = 8 * ((pl.row & 3) + e);
                const uint32_t codes = ((w.x >> sh) & 255u) | (((w.y >> sh) & 255u) << 8) | (((w.z >> sh) & 255u) << 16) |
                                       (((w.w >> sh) & 255u) << 24);
                dequantise8(codes, par[e], x);
                store8(p.v_out, (long long)(t0 + j0 + e) * row_elems + (long long)h * p.D + c0, p.dtype, true, x);
            }
        }
    }
}

}  // namespace

hipError_t launch_append(const AppendParams& p, hipStream_t s) {
    if (p.map.T <= 0) return hipSuccess;
    const dim3 grid((unsigned)((p.map.T + p.tokens_per_wg - 1) / p.tokens_per_wg), (unsigned)p.head_split);
    count_launch();
    hipLaunchKernelGGL(append_kernel, grid, dim3(256), 0, s, p);
    return hipGetLastError();
}
hipError_t launch_gather(const GatherParams& p, hipStream_t s) {
    if (p.map.T <= 0) return hipSuccess;
    const dim3 grid((unsigned)((p.map.T + p.tokens_per_wg - 1) / p.tokens_per_wg), (unsigned)p.head_split);
    count_launch();
    hipLaunchKernelGGL(gather_kernel, grid, dim3(256), 0, s, p);
    return hipGetLastError();
}

}  // namespace spfa
