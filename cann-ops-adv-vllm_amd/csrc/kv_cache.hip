// Writing and reading a paged KV cache (gfx950): append (rotation, quantisation and placement in one pass over the new
// rows) and read-back (rows in 16 bits).  Both move bytes and little else, so what matters is that every row is read
// once in whole 16-byte pieces and that small calls are one short launch.
#include "kv_params.h"

#include <hip/hip_runtime.h>
#include <stdint.h>
#include <type_traits>

namespace spfa {
namespace {

#include "spfa_common.inc"

constexpr int kTokMax = 8;        // most tokens a workgroup deals with
// rows whose loads are under way at once: 11485 tokens into a 4-bit cache and back 85 us with two, 83 with four, 78 with six,
// 81 with eight; into a 16-bit cache 48 us with two, 55 with six; int8 rows need registers for their parameters (1813 rows of
// 256 channels 22 us with two, 24 with six)
template <int KIND> constexpr int batch() { return KIND == kI4 ? 6 : 2; }

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
__device__ __forceinline__ uint4 raw8(const void* base, long long off, bool wide) {
    const uint16_t* p = (const uint16_t*)base + off;
    if (wide) return *(const uint4*)p;
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = (uint32_t)p[2 * i] | ((uint32_t)p[2 * i + 1] << 16);
    return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ void floats8(uint4 v, int dtype, float* f) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[2 * i] = dtype == kBF16 ? bf16_lo(w[i]) : f16_bits((uint16_t)(w[i] & 0xffffu));
        f[2 * i + 1] = dtype == kBF16 ? bf16_hi(w[i]) : f16_bits((uint16_t)(w[i] >> 16));
    }
}
__device__ __forceinline__ void load8(const void* base, long long off, int dtype, bool wide, float* f) {
    floats8(raw8(base, off, wide), dtype, f);
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

// The same into rows that nothing reads again soon (aligned): past the caches.
__device__ __forceinline__ void stream8(void* base, long long off, int dtype, const float* f) {
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
    __builtin_nontemporal_store(u32x4{pack2(f[0], f[1], dtype), pack2(f[2], f[3], dtype), pack2(f[4], f[5], dtype), pack2(f[6], f[7], dtype)},
                                (u32x4*)((uint16_t*)base + off));
}

// Rotation of the eight channels c0 .. c0 + 7 of a row: channel c < rot turns with its partner by the angle of its pair.
// Two rounded products and a rounded sum, contraction off: the same value whichever of the two functions takes the row.
//
// Turn: the angles of a lane's channels, loaded once per token; the rows of all its heads turn by them.  The partners'
// values come from the lane that holds them.
struct Turn {
    float c[8], s[8];     // pairs side by side: four of each; low half: s is the sine's negative
    int mode;             // 0 nothing turns, 1 low half, 2 high half, 3 pairs side by side
    int partner;          // 4 x the lane that holds the partners (modes 1 and 2), or the lane itself
    bool halves;          // the call turns channels with those half a rotation away
};
__device__ __forceinline__ void load_turn(const AppendParams& p, int c0, int cs_row, Turn* t) {
    t->mode = 0;
    t->partner = 4 * lane_id();
    t->halves = p.cos_sin && !p.interleaved;
#pragma unroll
    for (int i = 0; i < 8; ++i) { t->c[i] = 1.f; t->s[i] = 0.f; }
    if (!p.cos_sin || c0 >= p.rot) return;
    const int half = p.rot >> 1, n = p.interleaved ? 4 : 8;
    t->mode = p.interleaved ? 3 : (c0 < half ? 1 : 2);
    if (!p.interleaved) t->partner += c0 < half ? half / 2 : -(half / 2);       // (eight channels a lane)
    const long long at = (long long)cs_row * p.rot + (p.interleaved ? c0 >> 1 : (c0 < half ? c0 : c0 - half));
#pragma unroll
    for (int i = 0; i < 8; i += 4) {
        if (i >= n) break;
        if (p.cs_dtype == kF32) {
            const float4 c = *(const float4*)((const float*)p.cos_sin + at + i), s = *(const float4*)((const float*)p.cos_sin + at + half + i);
            t->c[i] = c.x; t->c[i + 1] = c.y; t->c[i + 2] = c.z; t->c[i + 3] = c.w;
            t->s[i] = s.x; t->s[i + 1] = s.y; t->s[i + 2] = s.z; t->s[i + 3] = s.w;
        } else {
            const uint2 c = *(const uint2*)((const uint16_t*)p.cos_sin + at + i), s = *(const uint2*)((const uint16_t*)p.cos_sin + at + half + i);
            const uint32_t w[4] = {c.x, c.y, s.x, s.y};
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                t->c[i + 2 * j] = p.cs_dtype == kBF16 ? bf16_lo(w[j]) : f16_bits((uint16_t)(w[j] & 0xffffu));
                t->c[i + 2 * j + 1] = p.cs_dtype == kBF16 ? bf16_hi(w[j]) : f16_bits((uint16_t)(w[j] >> 16));
                t->s[i + 2 * j] = p.cs_dtype == kBF16 ? bf16_lo(w[2 + j]) : f16_bits((uint16_t)(w[2 + j] & 0xffffu));
                t->s[i + 2 * j + 1] = p.cs_dtype == kBF16 ? bf16_hi(w[2 + j]) : f16_bits((uint16_t)(w[2 + j] >> 16));
            }
        }
    }
    if (t->mode == 1)
#pragma unroll
        for (int i = 0; i < 8; ++i) t->s[i] = -t->s[i];
}
__device__ __forceinline__ void apply_turn(const Turn& t, uint4 own, int dtype, float* x) {
#pragma clang fp contract(off)
    uint4 other = own;
    if (t.halves)         // (of the call: all lanes of a row take part, those that do not turn with themselves)
        other = make_uint4(__builtin_amdgcn_ds_bpermute(t.partner, own.x), __builtin_amdgcn_ds_bpermute(t.partner, own.y),
                           __builtin_amdgcn_ds_bpermute(t.partner, own.z), __builtin_amdgcn_ds_bpermute(t.partner, own.w));
    if (t.mode == 0) return;
    if (t.mode == 3) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float a = x[2 * i], b = x[2 * i + 1];
            x[2 * i] = a * t.c[i] - b * t.s[i];
            x[2 * i + 1] = b * t.c[i] + a * t.s[i];
        }
    } else {
        float y[8];
        floats8(other, dtype, y);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = x[i] * t.c[i] + y[i] * t.s[i];
    }
}

// A row element by element, for strides, starts and rotations that are not in whole 16 bytes.  All loads of a row come
// before its stores and one wave holds the whole row, so the output may be the input itself.
__device__ __forceinline__ void load_rotated(const AppendParams& p, const void* row, long long off, int c0, int cs_row, float* x) {
#pragma clang fp contract(off)
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
    for (int i = 0; i < 8; ++i) nan = fmaf(x[i], 0.f, nan);   // NaN if any channel is not finite
    const unsigned long long bad = __ballot(nan != 0.f);
    const unsigned long long mine = lanes >= 64 ? ~0ull : ((1ull << lanes) - 1ull) << (lane & ~(lanes - 1));
    for (int step = 1; step < lanes; step <<= 1) {
        lo = fminf(lo, __shfl_xor(lo, step));
        hi = fmaxf(hi, __shfl_xor(hi, step));
    }
    // (the corrected quotient by 15, see below, equal to the division for every mantissa: the product with 1 / 15 alone misses
    // half-way cases between two scales.  An infinite difference makes it NaN, which fminf leaves for the bound.)
    const float span = hi - lo, s0 = span * (1.f / 15.f);
    const _Float16 s = (_Float16)fminf(fmaf(fmaf(-s0, 15.f, span), 1.f / 15.f, s0), 65504.f);
    _Float16 z = (_Float16)fminf(fmaxf(lo, -65504.f), 65504.f);
    // 16-bit inputs meet exact halves often, so the quotient has to be the correctly rounded one; the divisor is the same
    // for the row, so this takes three instructions a channel: with r the rounded reciprocal (one Newton step from within
    // one unit makes it that, the divisor's 11 bits being no all-ones mantissa) the corrected quotient is the rounded
    // quotient (Markstein, "Computation of elementary functions on the IBM RISC System/6000 processor", 1990).
    const float zf = (float)z, sf = (float)s;
    float r = __builtin_amdgcn_rcpf(sf);
    r = fmaf(fmaf(-sf, r, 1.f), r, r);
    uint32_t codes = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float a = x[i] - zf, q0 = a * r, q = fmaf(fmaf(-q0, sf, a), r, q0);
        codes |= (uint32_t)(int)fminf(fmaxf(rintf(q), 0.f), 15.f) << (4 * i);
    }
    if (!(sf > 0.f)) codes = 0;
    uint16_t zb = __builtin_bit_cast(uint16_t, z), sb = __builtin_bit_cast(uint16_t, s);
    if (bad & mine) { zb = 0x7e00u; sb = 0; }
    *param = (uint32_t)sb | ((uint32_t)zb << 16);
    return codes;
}

// Parameters of eight channels of an int8 row: side by side, or one of the head or of the tensor.
__device__ __forceinline__ void int8_params(const CacheView& c, int which, int n2, int c0, int Hkv, int D, float* s, float* o) {
    const long long at = which == 0 ? antiq_key_index(c.antiq_layout, n2, c0, D) : antiq_value_index(c.antiq_layout, n2, c0, D, Hkv);
    if (c.antiq_layout == 0) {
        load8(c.antiq_scale, at, c.antiq_dtype, ((uintptr_t)c.antiq_scale & 15) == 0, s);
        if (c.antiq_offset) load8(c.antiq_offset, at, c.antiq_dtype, ((uintptr_t)c.antiq_offset & 15) == 0, o);
    } else {
        s[0] = load_qk_elem(c.antiq_scale, c.antiq_dtype, at);
        if (c.antiq_offset) o[0] = load_qk_elem(c.antiq_offset, c.antiq_dtype, at);
#pragma unroll
        for (int i = 1; i < 8; ++i) { s[i] = s[0]; o[i] = o[0]; }
    }
    if (!c.antiq_offset)
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = 0.f;
}

// (x / scale - offset) rounded to the nearest even code, saturating; NaN becomes code 0, a scale of 0 code 0 as well.
__device__ __forceinline__ uint2 quantise8_int8(const CacheView& c, int which, int n2, int c0, int Hkv, int D, const float* x) {
    float s[8], o[8];
    int8_params(c, which, n2, c0, Hkv, D, s, o);
    float y[8];
    float low = fabsf(s[0]), high = low, top = fabsf(x[0]);
#pragma unroll
    for (int i = 1; i < 8; ++i) {
        low = fminf(low, fabsf(s[i]));
        high = fmaxf(high, fabsf(s[i]));
        top = fmaxf(top, fabsf(x[i]));
    }
    if (low >= 0x1p-60f && high <= 0x1p60f && top <= 0x1p60f) {
        // the corrected quotient of quantise8: nothing leaves the normal range here, scales have 11 bits at most (11485 tokens
        // into an int8 cache and back 104 us, 108 with divisions)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            float r = __builtin_amdgcn_rcpf(s[i]);
            r = fmaf(fmaf(-s[i], r, 1.f), r, r);
            const float q0 = x[i] * r;
            y[i] = fmaf(fmaf(-q0, s[i], x[i]), r, q0) - o[i];
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = s[i] != 0.f ? x[i] / s[i] - o[i] : 0.f;
    }
    uint32_t w[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float known = y[i] == y[i] ? y[i] : 0.f;
        const int code = (int)rintf(fminf(fmaxf(known, -128.f), 127.f));
        w[i / 4] |= (uint32_t)(code & 255) << (8 * (i % 4));
    }
    return make_uint2(w[0], w[1]);
}

// Address of eight channels of a 16-bit or int8 row, or of a 4-bit K row.
template <int KIND>
__device__ __forceinline__ char* cache_at(const CacheView& c, void* base, const Place& pl, int n2, int c0) {
    const long long off = (long long)pl.page * c.blk_stride + (long long)pl.row * c.tok_stride + (long long)n2 * c.head_stride;
    return (char*)base + off + (KIND == kI4 ? c0 / 2 : (KIND == kI8 ? c0 : 2 * c0));
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

// (unit, head) pairs of a workgroup, head fastest, dealt to its groups of lanes (and to the workgroups that share its
// tokens): the division by the number of heads is done once.
struct Deal {
    int u, h, du, dh, heads;
    __device__ __forceinline__ Deal(int first, int step, int n_heads) : u(first / n_heads), h(first % n_heads), du(step / n_heads), dh(step % n_heads), heads(n_heads) {}
    __device__ __forceinline__ void next() {
        u += du;
        h += dh;
        if (h >= heads) { h -= heads; ++u; }
    }
};

// One workgroup: up to tokens_per_wg tokens (their places found once, by the first wave), all heads or a share of them
// (head_split workgroups).  D / 8 consecutive lanes hold a row, eight channels each.
//
// What bounds it: the bytes of the rows, read and written once.  A group of lanes keeps to a token and goes through the
// token's q and K rows (16 bits and int8: V rows too), the loads of several rows under way at once, the angles loaded once
// for all of them; 4-bit V rows go by quads of tokens, so that a whole quad is one 16-byte store per lane.
// VALU work counts next to them, so types are compiled in, addresses step and the quantiser divides by its one divisor in
// three instructions.  A prompt of 11485 tokens (32 q heads, 8 kv heads, D = 128, 4-bit cache; 248 MB): 56 us, 4.4 TB/s, with
// 19 M instructions of a wave; 74 us and 27 M with types and addresses at run time, 120 us a row at a time.
// KIND: dtype of the cache, 16 bits as kF16.  TYPE: dtype of the rows where all of them are in whole 16-byte pieces, -1: of
// any dtype, element by element.
enum { kRowQ, kRowK, kRowV };

// Rows r, r + step, ... below `end` (counted over q, K and V rows) of a token.  Returns the first one that it left.
template <int WHAT, int KIND, int TYPE>
__device__ __forceinline__ int token_rows(const AppendParams& p, const Place& pl, const Turn& angles, bool turn, bool store, int t, int cs, int r, int begin,
                                          int end, int step, int lanes, int sub, int lane) {
    constexpr int AT_ONCE = TYPE >= 0 ? batch<KIND>() : 1;
    const int dtype = TYPE >= 0 ? TYPE : p.dtype, c0 = sub * 8;
    const long long head = WHAT == kRowQ ? p.q_head : (WHAT == kRowK ? p.k_head : p.v_head);
    const long long start = (long long)t * (WHAT == kRowQ ? p.q_tok : (WHAT == kRowK ? p.k_tok : p.v_tok));
    const uint16_t* base = (const uint16_t*)(WHAT == kRowQ ? p.q : (WHAT == kRowK ? p.k : p.v)) + start;
    const bool any = WHAT == kRowQ || store;
    for (; r < end; r += AT_ONCE * step) {
        const int h0 = r - begin;
        uint4 own[AT_ONCE];
        if (TYPE >= 0 && turn && any) {
            const uint16_t* row = base + h0 * head + c0;
#pragma unroll
            for (int b = 0; b < AT_ONCE; ++b) {
                own[b] = *(const uint4*)row;
                if (r + (b + 1) * step < end) row += step * head;        // (past the end: the last row again)
            }
        }
        if (any)
#pragma unroll
            for (int b = 0; b < AT_ONCE; ++b) {
                if (r + b * step >= end) break;
                const int h = h0 + b * step;
                float x[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = 0.f;
                if (turn) {
                    if (TYPE >= 0) {
                        floats8(own[b], dtype, x);
                        if (WHAT != kRowV) apply_turn(angles, own[b], dtype, x);
                    } else if (WHAT == kRowV) {
                        load8(p.v, start + h * head + c0, dtype, p.wide != 0, x);
                    } else {
                        load_rotated(p, WHAT == kRowQ ? p.q : p.k, start + h * head, c0, cs, x);
                    }
                }
                if (WHAT == kRowQ) {
                    store8(p.q_out, (long long)t * p.qo_tok + h * p.qo_head + c0, dtype, TYPE >= 0 || p.wide != 0, x);
                    continue;
                }
                char* dst = cache_at<KIND>(p.cache, WHAT == kRowV ? p.cache.v : p.cache.k, pl, h, c0);
                if (KIND == kI4) {
                    uint32_t par;
                    const uint32_t codes = quantise8(x, lanes, lane, &par);
                    *(uint32_t*)dst = codes;
                    if (sub == 0) p.cache.k_params[param_at(p.cache, p.map, pl, p.Hkv, h)] = par;
                } else if (KIND == kI8) {
                    *(uint2*)dst = quantise8_int8(p.cache, WHAT == kRowV ? 1 : 0, h, c0, p.Hkv, p.D, x);
                } else {
                    store8(dst, 0, dtype, true, x);
                }
            }
    }
    while (r - step >= end) r -= step;
    return r;
}

template <int KIND, int TYPE>
__global__ __launch_bounds__(256) void append_kernel(const AppendParams p) {
    __shared__ Place places[kTokMax];
    __shared__ uint8_t q_first[kTokMax], q_count[kTokMax];
    __shared__ int n_quads;
    constexpr bool QUADS = KIND == kI4, FAST = TYPE >= 0;
    const int dtype = FAST ? TYPE : p.dtype;
    const int lane = lane_id(), wave = wave_id();
    const int t0 = blockIdx.x * p.tokens_per_wg;
    const int n = min(p.tokens_per_wg, p.map.T - t0);
    if (wave == 0) {
        find_places(p.map, t0, n, places, lane);
        wave_lds_sync();
        if (QUADS) {
            const int k = find_quads(places, n, q_first, q_count, lane);
            if (lane == 0) n_quads = k;
        }
    }
    __syncthreads();
    const int lanes = p.D >> 3;                     // 4 .. 64
    const int sub = threadIdx.x & (lanes - 1), c0 = sub * 8;
    const int group = (int)threadIdx.x / lanes, groups = 256 / lanes;
    // groups of a token (1, or several when the tokens are fewer than the groups), and the tokens of a group
    const int per_token = max(1, groups / p.tokens_per_wg), tokens_at_once = min(groups, p.tokens_per_wg);
    const int nq = p.q ? p.Hq : 0, step = per_token * gridDim.y;
    const int first = group / tokens_at_once + blockIdx.y * per_token;
    for (int j = group % tokens_at_once; j < n; j += tokens_at_once) {
        const Place pl = places[j];
        const int t = t0 + j;
        const int cs = p.positions && pl.seq >= 0 ? p.positions[t] : pl.pos;
        const bool known = !p.cos_sin || (cs >= 0 && cs < p.cs_rows);
        const bool turn = pl.pos >= 0 && known, store = pl.page >= 0 && known;
        if (!turn && pl.seq < 0 && !p.zero_rest) continue;       // (rows in no sequence are left as they are)
        Turn angles;
        if (FAST && turn) load_turn(p, c0, cs, &angles);
        int r = first;
        r = token_rows<kRowQ, KIND, TYPE>(p, pl, angles, turn, store, t, cs, r, 0, nq, step, lanes, sub, lane);
        r = token_rows<kRowK, KIND, TYPE>(p, pl, angles, turn, store, t, cs, r, nq, nq + p.Hkv, step, lanes, sub, lane);
        if (!QUADS) token_rows<kRowV, KIND, TYPE>(p, pl, angles, turn, store, t, cs, r, nq + p.Hkv, nq + 2 * p.Hkv, step, lanes, sub, lane);
    }
    if constexpr (QUADS) {
        for (Deal d(group + blockIdx.y * groups, groups * gridDim.y, p.Hkv); d.u < n_quads; d.next()) {
            const int j0 = q_first[d.u], cnt = q_count[d.u];
            const Place pl = places[j0];
            uint4 raw[4];
            int cs[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {            // (a run that is shorter reads its last row again)
                const int j = j0 + min(e, cnt - 1);
                raw[e] = raw8(p.v, (long long)(t0 + j) * p.v_tok + (long long)d.h * p.v_head + c0, FAST || p.wide != 0);
                cs[e] = p.cos_sin && p.positions ? p.positions[t0 + j] : places[j].pos;
            }
            uint32_t codes[4] = {0, 0, 0, 0};
            unsigned ok = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (e >= cnt) break;
                if (p.cos_sin && (cs[e] < 0 || cs[e] >= p.cs_rows)) continue;
                float x[8];
                uint32_t par;
                floats8(raw[e], dtype, x);
                codes[e] = quantise8(x, lanes, lane, &par);
                ok |= 1u << e;
                if (sub == 0) p.cache.v_params[param_at(p.cache, p.map, pl, p.Hkv, d.h) + e] = par;
            }
            char* dst = quad_at(p.cache, pl, d.h, c0);
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

// Rows back in 16 bits.  A unit of work is a quad of tokens of a head (4 bits: a 16-byte piece of V per lane, four rows of
// K) or a row of K and its V row; all loads of a unit come first.  Rows without a place become zeros in a loop of their own.
// Bound by the bytes that it writes: 88 k tokens of 8 heads, D = 128, 4-bit cache (456 MB) 79 us, 5.8 TB/s; 106 us with
// stores that stay in the caches, 137 us a row at a time.
template <int KIND>
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
        if (KIND == kI4) {
            const int k = find_quads(places, n, q_first, q_count, lane);
            if (lane == 0) n_quads = k;
        }
    }
    __syncthreads();
    const int lanes = p.D >> 3;
    const int sub = threadIdx.x & (lanes - 1), c0 = sub * 8;
    const int group = (int)threadIdx.x / lanes, groups = 256 / lanes;
    const int first = group + blockIdx.y * groups, step = groups * gridDim.y;
    const long long row_elems = (long long)p.Hkv * p.D;
    if constexpr (KIND == kI4) {
        for (Deal d(first, step, p.Hkv); d.u < n_quads; d.next()) {
            const int j0 = q_first[d.u], cnt = q_count[d.u];
            const Place pl = places[j0];
            const char* ks = cache_at<KIND>(p.cache, p.cache.k, pl, d.h, c0);
            const uint4 w = *(const uint4*)quad_at(p.cache, pl, d.h, c0);
            const long long at = param_at(p.cache, p.map, pl, p.Hkv, d.h);
            uint32_t kc[4], kp[4], vp[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {            // (a run that is shorter reads its last row again)
                const int i = min(e, cnt - 1);
                kc[e] = *(const uint32_t*)(ks + i * p.cache.tok_stride);
                kp[e] = p.cache.k_params[at + i];
                vp[e] = p.cache.v_params[at + i];
            }
            const long long out = (long long)(t0 + j0) * row_elems + (long long)d.h * p.D + c0;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (e >= cnt) break;
                float x[8];
                dequantise8(kc[e], kp[e], x);
                stream8(p.k_out, out + e * row_elems, p.dtype, x);
                const int sh = 8 * ((pl.row & 3) + e);
                const uint32_t codes = ((w.x >> sh) & 255u) | (((w.y >> sh) & 255u) << 8) | (((w.z >> sh) & 255u) << 16) |
                                       (((w.w >> sh) & 255u) << 24);
                dequantise8(codes, vp[e], x);
                stream8(p.v_out, out + e * row_elems, p.dtype, x);
            }
        }
    }
    for (Deal d(first, step, p.Hkv); d.u < n; d.next()) {
        const Place pl = places[d.u];
        if (pl.page >= 0 ? KIND == kI4 : (pl.seq < 0 && !p.zero_rest)) continue;
        float x[8], y[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) { x[e] = 0.f; y[e] = 0.f; }
        if (KIND != kI4 && pl.page >= 0) {
            const char* ks = cache_at<KIND>(p.cache, p.cache.k, pl, d.h, c0);
            const char* vs = cache_at<KIND>(p.cache, p.cache.v, pl, d.h, c0);
            if (KIND == kI8) {
                const uint2 kw = *(const uint2*)ks, vw = *(const uint2*)vs;
                float s[8], o[8];
                int8_params(p.cache, 0, d.h, c0, p.Hkv, p.D, s, o);
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = ((float)(int)(int8_t)((e < 4 ? kw.x : kw.y) >> (8 * (e & 3))) + o[e]) * s[e];
                int8_params(p.cache, 1, d.h, c0, p.Hkv, p.D, s, o);
#pragma unroll
                for (int e = 0; e < 8; ++e) y[e] = ((float)(int)(int8_t)((e < 4 ? vw.x : vw.y) >> (8 * (e & 3))) + o[e]) * s[e];
            } else {
                const uint4 kw = *(const uint4*)ks, vw = *(const uint4*)vs;
                floats8(kw, p.cache.dtype, x);
                floats8(vw, p.cache.dtype, y);
            }
        }
        const long long dst = (long long)(t0 + d.u) * row_elems + (long long)d.h * p.D + c0;
        stream8(p.k_out, dst, p.dtype, x);
        stream8(p.v_out, dst, p.dtype, y);
    }
}

}  // namespace

hipError_t launch_append(const AppendParams& p, hipStream_t s) {
    if (p.map.T <= 0) return hipSuccess;
    if (p.tokens_per_wg < 1 || p.tokens_per_wg > kTokMax) return hipErrorInvalidValue;
    const dim3 grid((unsigned)((p.map.T + p.tokens_per_wg - 1) / p.tokens_per_wg), (unsigned)p.head_split);
    // whole pieces of 16 bytes, and all eight channels of a lane turn or none does
    const bool fast = p.wide && (!p.cos_sin || (p.interleaved ? p.rot % 8 == 0 : p.rot % 16 == 0));
    count_launch();
    auto go = [&](auto kind) {
        constexpr int K = decltype(kind)::value;
        if (fast && p.dtype == kF16) hipLaunchKernelGGL((append_kernel<K, kF16>), grid, dim3(256), 0, s, p);
        else if (fast) hipLaunchKernelGGL((append_kernel<K, kBF16>), grid, dim3(256), 0, s, p);
        else hipLaunchKernelGGL((append_kernel<K, -1>), grid, dim3(256), 0, s, p);
    };
    if (p.cache.dtype == kI4) go(std::integral_constant<int, kI4>{});
    else if (p.cache.dtype == kI8) go(std::integral_constant<int, kI8>{});
    else go(std::integral_constant<int, kF16>{});
    return hipGetLastError();
}
hipError_t launch_gather(const GatherParams& p, hipStream_t s) {
    if (p.map.T <= 0) return hipSuccess;
    if (p.tokens_per_wg < 1 || p.tokens_per_wg > kTokMax) return hipErrorInvalidValue;
    const dim3 grid((unsigned)((p.map.T + p.tokens_per_wg - 1) / p.tokens_per_wg), (unsigned)p.head_split);
    count_launch();
    if (p.cache.dtype == kI4) hipLaunchKernelGGL((gather_kernel<kI4>), grid, dim3(256), 0, s, p);
    else if (p.cache.dtype == kI8) hipLaunchKernelGGL((gather_kernel<kI8>), grid, dim3(256), 0, s, p);
    else hipLaunchKernelGGL((gather_kernel<kF16>), grid, dim3(256), 0, s, p);
    return hipGetLastError();
}

}  // namespace spfa
