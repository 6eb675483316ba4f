// Attention over a paged cache held in 4 bits (gfx950).
//
//   K_t = s_t c_t + z_t,  V_t = s'_t c'_t + z'_t    (codes c, c' in 0 .. 15; s, z per token and kv head, float16)
//   score(n, t) = scale (s_t (q_n . c_t) + z_t sum(q_n)),
//   O_n = (sum_t (p_t s'_t) (c'_t - 7.5) + sum_t p_t (z'_t + 7.5 s'_t)) / sum_t p_t
//
// so the matrix cores multiply CODES and the parameters are applied to scores and probabilities, one fma each.  A code
// becomes a matrix operand by masking alone: (w & 0x000f000f) are two codes in the bits of float16 denormals c * 2^-24
// (the matrix cores take denormals as they are; the odd codes of a byte come out 16 times larger, which the q elements
// they meet and the final scaling take back).  Five vector instructions unpack eight codes.
//
// Per step of 32 tokens a wave computes, with v_mfma_f32_16x16x32_f16 (A = K codes of 16 tokens, B = 16 q rows):
//   S^T[token, row]: lane l holds row l % 16 and the tokens 4 (l / 16) .. + 3 of each half of the step;
//   O^T[channel, row] += V^T[channel, token] P^T[token, row]: the probabilities are already where operand B wants them
//   (tokens 4 (l / 16) .. + 3 of both halves = its eight k slots), nothing crosses lanes between the two products.
//
// The running maximum is lazy: a row keeps a reference m that is at most 8 (log2) below its true maximum, and a step
// that would exceed that (or whose V scales outgrow the reference scale R that keeps p * s' inside float16) takes the
// slow path, which moves m and R and rescales the sums.  Sums, statistics and O are float32; p * s' is rounded to
// float16 (relative 2^-11, down to 2^-20 of the peak) for the second product.
//
// Work.  An item is (sequence, kv head, tile of q rows); its tokens are cut into steps of 32 tokens.  All items' steps
// form one line that is cut into equal pieces, one per resident workgroup: lengths may be as ragged as they like.  A
// workgroup computes its piece from seq_len alone.  An item that spans several workgroups is merged by the last of them
// to arrive (partial states in the workspace, one arrival counter per split item).
// The four waves of a workgroup are RW groups of rows x 4 / RW shares of the steps: few rows (decode) share the steps and
// merge their states through LDS, prompts hold four times as many rows and walk the same tokens (shared through the L1
// cache), candidate tokens are in between.
// With page lists (one row of q per sequence) an item is (sequence, list) and workers workgroups share each list.
#include "kv_params.h"

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <mutex>

namespace spfa {
namespace {

#include "spfa_common.inc"

typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNoMax = -3.0e38f;          // reference of a row that has seen no token
constexpr float kLazy = 8.f;                // log2 distance a reference may fall behind the true maximum
constexpr int kScaleTop = 6;                // V scales are brought below 2^6 (and may grow to 2^7 before the next slow path)

// A step: for each half of 16 tokens the row of the cache where it begins, the first token's place in the sequence, and
// whether the page is there.
struct Ptrs { long long row[2]; int tok[2]; bool ok[2]; };

template <int W> struct Words { uint32_t w[W]; };
template <int W>
__device__ __forceinline__ Words<W> load_words(const uint8_t* p) {
    Words<W> r;
    if constexpr (W == 1) r.w[0] = *(const uint32_t*)p;
    else if constexpr (W == 2) { const uint2 v = *(const uint2*)p; r.w[0] = v.x; r.w[1] = v.y; }
    else {
        const uint4 v = *(const uint4*)p;
        r.w[0] = v.x; r.w[1] = v.y; r.w[2] = v.z; r.w[3] = v.w;
    }
    return r;
}

__device__ __forceinline__ f32x4 mfma(const u32x4& a, const u32x4& b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c, 0, 0, 0);
}
// eight codes of a word as four operand words: nibbles (0, 4), (1, 5), (2, 6), (3, 7)
__device__ __forceinline__ u32x4 codes_of(uint32_t w) {
    const uint32_t h = w >> 8;
    return u32x4{w & 0x000f000fu, w & 0x00f000f0u, h & 0x000f000fu, h & 0x00f000f0u};
}
__device__ __forceinline__ uint32_t pack_f16(float a, float b) {   // round to nearest even
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, half2v));
}
__device__ __forceinline__ float lo16(uint32_t w) { return f16_bits((uint16_t)(w & 0xffffu)); }
__device__ __forceinline__ float hi16(uint32_t w) { return f16_bits((uint16_t)(w >> 16)); }

// Sums / maxima over the four lane groups that hold the same row.
__device__ __forceinline__ float rows_sum(float x) { x += __shfl_xor(x, 16); return x + __shfl_xor(x, 32); }
__device__ __forceinline__ float rows_max(float x) { x = fmaxf(x, __shfl_xor(x, 16)); return fmaxf(x, __shfl_xor(x, 32)); }

// ---- the line of steps ----------------------------------------------------------------------------------------------
// rows of a sequence: first row of the call, how many; its tokens, and those that its table can hold
struct Seq { int first, n, tokens, len; };
__device__ __forceinline__ Seq seq_of(const TokenMap& m, int b) {
    Seq s;
    s.first = m.query_start ? m.query_start[b] : b;
    const int end = m.query_start ? min(m.query_start[b + 1], m.T) : b + 1;
    s.first = max(s.first, 0);
    s.n = max(end - s.first, 0);
    s.tokens = max(m.seq_len[b], 0);
    s.len = (int)min((long long)s.tokens, (long long)m.max_page * m.block_size);
    return s;
}
// The same values, known to be the same in all lanes (they then live in scalar registers).
__device__ __forceinline__ int uni(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ long long uni(long long x) {
    return (long long)(((unsigned long long)(unsigned)uni((int)((unsigned long long)x >> 32)) << 32) | (unsigned)uni((int)x));
}
__device__ __forceinline__ Seq uniform_seq(const TokenMap& m, int b) {
    const Seq s = seq_of(m, b);
    return Seq{uni(s.first), uni(s.n), uni(s.tokens), uni(s.len)};
}
// Tokens that row i of a sequence sees: its position is seq_len - n + i, and nothing lies behind the table.
__device__ __forceinline__ int seen_by(const Int4AttnParams& p, const Seq& s, int i) {
    return p.causal ? max(0, min(s.len, s.tokens - s.n + i + 1)) : s.len;
}
__device__ __forceinline__ int steps_of(const Int4AttnParams& p, const Seq& s, int rt) {
    const int last = min((rt + 1) * p.rows_tile, s.n * p.G) - 1;
    return max(1, (seen_by(p, s, last / p.G) + kInt4StepTokens - 1) / kInt4StepTokens);
}
__device__ __forceinline__ int row_tiles(const Int4AttnParams& p, const Seq& s) { return (s.n * p.G + p.rows_tile - 1) / p.rows_tile; }

__device__ __forceinline__ long long wave_scan(long long x, int lane) {   // inclusive
    for (int d = 1; d < 64; d <<= 1) {
        const long long up = __shfl_up(x, d);
        if (lane >= d) x += up;
    }
    return x;
}
template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp_add(int x) { return x + __builtin_amdgcn_update_dpp(0, x, CTRL, ROWS, 0xf, false); }
__device__ __forceinline__ int wave_scan(int x, int) {
    x = dpp_add<0x111, 0xf>(x);      // row_shr 1, 2, 4, 8: inclusive within 16 lanes
    x = dpp_add<0x112, 0xf>(x);
    x = dpp_add<0x114, 0xf>(x);
    x = dpp_add<0x118, 0xf>(x);
    x = dpp_add<0x142, 0xa>(x);      // row_bcast 15 into rows 1 and 3, row_bcast 31 into rows 2 and 3
    return dpp_add<0x143, 0xc>(x);
}
__device__ __forceinline__ int lane_of(int x, int lane) { return __builtin_amdgcn_readlane(x, lane); }
__device__ __forceinline__ long long lane_of(long long x, int lane) {
    return (long long)(((unsigned long long)(unsigned)lane_of((int)((unsigned long long)x >> 32), lane) << 32) | (unsigned)lane_of((int)x, lane));
}
// non-negative; the 64-bit division is a long routine and hardly ever needed
__device__ __forceinline__ long long quotient(long long a, long long b) {
    return (((unsigned long long)a | (unsigned long long)b) >> 32) == 0 ? (long long)((unsigned)a / (unsigned)b) : a / b;
}

// steps of one kv head of a sequence (all its row tiles), computed by one lane / by the wave
__device__ __forceinline__ long long head_steps_lane(const Int4AttnParams& p, const Seq& s) {
    const int nt = row_tiles(p, s);
    if (nt <= 0) return 0;
    if (!p.causal) return (long long)nt * steps_of(p, s, 0);
    long long t = 0;
    for (int rt = 0; rt < nt; ++rt) t += steps_of(p, s, rt);
    return t;
}
template <typename I>
__device__ __forceinline__ I head_steps_wave(const Int4AttnParams& p, const Seq& s, int lane) {
    const int nt = row_tiles(p, s);
    if (!p.causal) return nt > 0 ? (I)nt * steps_of(p, s, 0) : 0;
    I t = 0;
    for (int rt = lane; rt < nt; rt += 64) t += steps_of(p, s, rt);
    return lane_of(wave_scan(t, lane), 63);
}

// A workgroup's piece [g, g1) of the line of all steps, and where it begins: step s0 of row tile rt of kv head h of sequence b.
struct Piece { long long g, g1, size; int b, h, rt, s0; };
// I: 32 bits where the line is known to be short enough (64-bit scans and divisions cost microseconds here)
template <typename I>
__device__ __forceinline__ bool find_piece(const Int4AttnParams& p, int w, int lane, Piece& out) {
    const int B = p.map.B;
    const bool lanes_b = B >= 16 || p.most_tiles <= 4;     // a lane per sequence, or the wave over the row tiles of each
    I total = 0, mine = 0, incl = 0;
    for (int b0 = 0; b0 < B; b0 += lanes_b ? 64 : 1) {
        if (lanes_b) {
            mine = b0 + lane < B ? (I)head_steps_lane(p, seq_of(p.map, b0 + lane)) : 0;
            incl = wave_scan(mine, lane);
            total += lane_of(incl, 63);
        } else {
            total += head_steps_wave<I>(p, uniform_seq(p.map, b0), lane);
        }
    }
    total *= p.Hkv;
    out.size = max((long long)p.min_steps, quotient((long long)total + p.workers - 1, p.workers));
    out.g = w * out.size;
    if (out.g >= total) return false;
    out.g1 = min((long long)total, out.g + out.size);
    I off = (I)out.g, heads = 0;
    int b = 0;
    if (lanes_b) {
        for (int b0 = 0; b0 < B; b0 += 64) {
            if (B > 64) {
                mine = b0 + lane < B ? (I)head_steps_lane(p, seq_of(p.map, b0 + lane)) : 0;
                incl = wave_scan(mine, lane);
            }
            const unsigned long long past = __ballot(incl * p.Hkv > off);
            if (past) {
                const int at = __ffsll(past) - 1;
                heads = lane_of(mine, at);
                off -= (lane_of(incl, at) - heads) * p.Hkv;
                b = b0 + at;
                break;
            }
            off -= lane_of(incl, 63) * p.Hkv;
        }
    } else {
        for (;; ++b) {
            heads = head_steps_wave<I>(p, uniform_seq(p.map, b), lane);
            if (off < heads * p.Hkv) break;
            off -= heads * p.Hkv;
        }
    }
    out.b = uni(b);
    const Seq sq = uniform_seq(p.map, out.b);
    out.h = uni((int)quotient(off, heads));
    off -= out.h * heads;
    int rt = 0;
    if (!p.causal) {
        const int n = steps_of(p, sq, 0);
        rt = (int)quotient(off, n);
        off -= (I)rt * n;
    } else if (row_tiles(p, sq) > 1) {
        for (int r0 = 0;; r0 += 64) {
            const I tile = r0 + lane < row_tiles(p, sq) ? steps_of(p, sq, r0 + lane) : 0, upto = wave_scan(tile, lane);
            const unsigned long long past = __ballot(upto > off);
            if (past) {
                const int at = __ffsll(past) - 1;
                off -= lane_of(upto, at) - lane_of(tile, at);
                rt = r0 + at;
                break;
            }
            off -= lane_of(upto, 63);
        }
    }
    out.rt = uni(rt);
    out.s0 = uni((int)off);
    return true;
}

// ---- the state of a wave -------------------------------------------------------------------------------------------
template <int D, int NT>
struct State {
    f32x4 o[NT][D / 16];     // [2 j + parity][i]: channel (4 kg + i) * D / 16 + 2 j + parity, in units of the codes
    f32x4 r[NT];             // sum of w (every element holds it)
    float m[NT], l[NT], z[NT];
    float inv_r;             // power of two: V scales are taken times inv_r
    int seen;                // bit t: the lane's row of tile t has seen a token
    int open;                // wave-uniform, bit 0: some row has seen none, bit 1: no V scale above 0 so far
};
template <int D, int NT>
__device__ __forceinline__ void clear_state(State<D, NT>& S) {
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        S.m[t] = S.l[t] = S.z[t] = 0.f;
        S.r[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int d = 0; d < D / 16; ++d) S.o[t][d] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    S.inv_r = 1.f;
    S.seen = 0;
    S.open = 3;
}

template <int D, int NT>
struct Query {
    u32x4 q[NT][D / 32];     // operand B: k slots in the order of codes_of
    float sum[NT];           // sum(q) * scale * log2(e)
    int lim[NT];             // tokens the lane's row sees
    float ks;                // what a score in code units is multiplied by (besides s_t)
    int lim_min, lim_max;    // fewest / most tokens a live row of the wave sees
};

// What the rows of a work item are: row r is token first + r / G of the sequence, q head head0 + r % G.
struct Rows { int first, head0, G, kvh, n; };

template <int D, int NT>
__device__ __forceinline__ void set_limits(const Int4AttnParams& p, const Seq& s, const Rows& R, int row0, Query<D, NT>& Q, int lane) {
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int r = row0 + 16 * t + (lane & 15);
        Q.lim[t] = r < R.n ? seen_by(p, s, r / R.G) : 0;
    }
    // later rows never see less
    Q.lim_min = row0 < R.n ? uni(seen_by(p, s, row0 / R.G)) : 0x7fffffff;
    Q.lim_max = row0 < R.n ? uni(seen_by(p, s, (min(row0 + 16 * NT, R.n) - 1) / R.G)) : 0;
}
// The lane's channels of q rows [row0, row0 + 16 NT) of an item, as they lie in memory.
template <int D, int NT> struct RawQuery { uint32_t w[NT][D / 8]; };
template <int D, int NT>
__device__ __forceinline__ void load_query(const Int4AttnParams& p, const Rows& R, int row0, RawQuery<D, NT>& q, int lane) {
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int r = row0 + 16 * t + (lane & 15);
        const bool live = r < R.n;
        const int i = live ? r / R.G : 0;
        const uint16_t* src = (const uint16_t*)p.q + (long long)(R.first + i) * p.q_tok + (long long)(R.head0 + (live ? r - i * R.G : 0)) * p.q_head +
                              (lane >> 4) * (D / 4);
#pragma unroll
        for (int j = 0; j < D / 8; ++j) q.w[t][j] = 0u;
        if (live && p.q_wide) {
#pragma unroll
            for (int j = 0; j < D / 32; ++j) {
                const uint4 v = *(const uint4*)(src + 8 * j);
                q.w[t][4 * j] = v.x; q.w[t][4 * j + 1] = v.y; q.w[t][4 * j + 2] = v.z; q.w[t][4 * j + 3] = v.w;
            }
        } else if (live) {
#pragma unroll
            for (int j = 0; j < D / 8; ++j) q.w[t][j] = (uint32_t)src[2 * j] | ((uint32_t)src[2 * j + 1] << 16);
        }
    }
}
// -> operand B.  The rows of a wave are brought to a common power of two with the largest element in [2^10, 2^11): float16
// then holds every element down to 2^-25 of it exactly (bfloat16 rows outside float16's range included), and the even
// slots, 16 times larger, stay below 2^15.
template <int D, int NT>
__device__ __forceinline__ void make_query(const Int4AttnParams& p, const RawQuery<D, NT>& q, Query<D, NT>& Q) {
    const bool bf = p.q_dtype == kBF16;
    auto lo = [&](uint32_t w) { return bf ? bf16_lo(w) : lo16(w); };
    auto hi = [&](uint32_t w) { return bf ? bf16_hi(w) : hi16(w); };
    float top = 0.f;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < D / 8; ++j) {
            const float a = lo(q.w[t][j]), b = hi(q.w[t][j]);
            sum += a + b;
            top = fmaxf(top, fmaxf(fabsf(a), fabsf(b)));
        }
        Q.sum[t] = rows_sum(sum) * (p.scale * kLog2e);
    }
    for (int d = 1; d < 64; d <<= 1) top = fmaxf(top, __shfl_xor(top, d));
    // exponent of the largest element (an infinite query is not scaled: its row comes out NaN)
    const int eb = (int)((__float_as_uint(top) >> 23) & 255u);
    const int up = uni(max(-118, min(118, (top > 0.f && eb < 255) ? 127 + 10 - eb : 0)));
    const float f = __uint_as_float((uint32_t)(127 + up) << 23);
    // codes arrive as c * 2^-24 (even channels) and 16 c * 2^-24 (odd); even slots of q carry 16 f, odd ones f
    Q.ks = p.scale * kLog2e * __uint_as_float((uint32_t)(127 - up) << 23) * 1048576.f;   // 2^24 / 16
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int j = 0; j < D / 32; ++j) {
            float x[8];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                x[2 * e] = lo(q.w[t][4 * j + e]) * (16.f * f);
                x[2 * e + 1] = hi(q.w[t][4 * j + e]) * f;
            }
            Q.q[t][j] = u32x4{pack_f16(x[0], x[4]), pack_f16(x[1], x[5]), pack_f16(x[2], x[6]), pack_f16(x[3], x[7])};
        }
}

// ---- the data of a step ---------------------------------------------------------------------------------------------
// A step's data goes from memory straight into LDS (no registers while it is under way, so several steps can be): the four
// half tiles K0, K1, V0, V1 of 8 D bytes each as 16-byte pieces, then the parameters, K of the 32 tokens and V of them.
// The pieces of a half lie in the order in which the lanes read them back.
template <int D> struct Slot {
    static constexpr int half = 8 * D, params = 32 * D, bytes = 32 * D + 256, loads = D / 32 + 1;
};
// Loads into LDS: lane l's bytes go to dst + l * size.  Written as assembly because the compiler, which knows such a load
// as a write to LDS, waits for all of them before the next read of LDS it cannot tell apart; here the steps are counted
// (wait_loads).  STREAM (nt): bytes that nobody reads again soon.  (A write of m0 needs one wait state before its use.)
__device__ __forceinline__ uint32_t lds_offset(const void* p) { return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)p; }
template <bool STREAM>
__device__ __forceinline__ void pieces_to_lds(const uint8_t* base, unsigned off, void* dst) {   // base uniform
    if constexpr (STREAM)
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2 nt" ::"s"(lds_offset(dst)), "v"(off), "s"(base) : "memory");
    else
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds_offset(dst)), "v"(off), "s"(base) : "memory");
}
template <bool STREAM>
__device__ __forceinline__ void pieces_to_lds(const uint8_t* src, void* dst) {
    if constexpr (STREAM)
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off nt" ::"s"(lds_offset(dst)), "v"(src) : "memory");
    else
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds_offset(dst)), "v"(src) : "memory");
}
__device__ __forceinline__ void word_to_lds(const uint32_t* src, void* dst) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(lds_offset(dst)), "v"(src) : "memory");
}
template <int N>
__device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }

// par: the lane's place in the parameters of the cache's first row (K for lanes 0 .. 31, V behind)
template <int D, bool STREAM>
__device__ __forceinline__ void fetch(const Int4AttnParams& p, const uint32_t* par, const Ptrs& a, uint8_t* slot, int lane) {
    const int n = lane & 15, kg = lane >> 4;
    word_to_lds(par + (p.paired ? a.row[0] : ((lane & 16) ? a.row[1] - 16 : a.row[0])), slot + Slot<D>::params);
    if constexpr (D >= 128) {
        // a lane's own bytes: D / 128 pieces of each half
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int c = 0; c < D / 128; ++c) {
                const unsigned ko = n * (D / 2) + kg * (D / 8) + c * 16, vo = kg * (2 * D) + n * (D / 8) + c * 16;
                pieces_to_lds<STREAM>(p.kcache + a.row[i] * (D / 2), ko, slot + (i * (D / 128) + c) * 1024);
                pieces_to_lds<STREAM>(p.vcache + a.row[i] * (D / 2), vo, slot + 2 * Slot<D>::half + (i * (D / 128) + c) * 1024);
            }
    } else if constexpr (D == 64) {
        // 32 pieces a half: K by (half of a token's row, token), V as it lies in memory
        const long long row = (lane & 32) ? a.row[1] : a.row[0];
        pieces_to_lds<STREAM>(p.kcache + row * (D / 2) + (n * 32 + (kg & 1) * 16), slot);
        pieces_to_lds<STREAM>(p.vcache + row * (D / 2) + (lane & 31) * 16, slot + 2 * Slot<D>::half);
    } else {
        // 16 pieces a half, all four halves in one load
        const long long row = (lane & 16) ? a.row[1] : a.row[0];
        pieces_to_lds<STREAM>((lane < 32 ? p.kcache : p.vcache) + row * (D / 2) + n * 16, slot);
    }
}
template <int D>
__device__ __forceinline__ Words<D / 32> k_words(const uint8_t* slot, int i, int lane) {
    const int n = lane & 15, kg = lane >> 4;
    const uint8_t* at = slot + i * Slot<D>::half;
    if constexpr (D == 256) {
        const Words<4> a = load_words<4>(at + lane * 16), b = load_words<4>(at + 1024 + lane * 16);
        return Words<8>{{a.w[0], a.w[1], a.w[2], a.w[3], b.w[0], b.w[1], b.w[2], b.w[3]}};
    } else if constexpr (D == 128) return load_words<4>(at + lane * 16);
    else if constexpr (D == 64) return load_words<2>(at + ((kg >> 1) * 16 + n) * 16 + (kg & 1) * 8);
    else return load_words<1>(at + n * 16 + kg * 4);
}
template <int D>
__device__ __forceinline__ Words<D / 32> v_words(const uint8_t* slot, int i, int lane) {
    const int n = lane & 15, kg = lane >> 4;
    const uint8_t* at = slot + (2 + i) * Slot<D>::half;
    if constexpr (D >= 128) return k_words<D>(slot, 2 + i, lane);
    else return load_words<D / 32>(at + kg * (2 * D) + n * (D / 8));
}
struct Params { u32x4 k[2], v[2]; };     // of the lane's four tokens in each half
template <int D>
__device__ __forceinline__ Params params_of(const uint8_t* slot, int lane) {
    const u32x4* at = (const u32x4*)(slot + Slot<D>::params) + (lane >> 4);
    return Params{{at[0], at[4]}, {at[8], at[12]}};
}

// A step in three parts.  MASKED: some token of the step is hidden from some row (the end of the sequence, the causal
// border, a page that is not there); a hidden token counts as probability 0 whatever its parameters hold.
template <int D, int NT>
__device__ __forceinline__ void products(const Query<D, NT>& Q, const uint8_t* slot, f32x4 (&s)[2][NT], int lane) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const Words<D / 32> k = k_words<D>(slot, i, lane);
#pragma unroll
        for (int t = 0; t < NT; ++t) s[i][t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < D / 32; ++j) {
            const u32x4 c = codes_of(k.w[j]);
#pragma unroll
            for (int t = 0; t < NT; ++t) s[i][t] = mfma(c, Q.q[t][j], s[i][t]);
        }
    }
}
// scores relative to the rows' references (log2), largest of them
template <int D, int NT, bool MASKED>
__device__ __forceinline__ float scores(const Query<D, NT>& Q, const State<D, NT>& S, const Params& P, const Ptrs& a, int seq_end, int kg,
                                        f32x4 (&s)[2][NT]) {
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float ks = lo16(P.k[i][e]) * Q.ks, kz = hi16(P.k[i][e]);
            const int tok = a.tok[i] + 4 * kg + e;
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                float x = fmaf(s[i][t][e], ks, fmaf(kz, Q.sum[t], -S.m[t]));
                if (MASKED && (!a.ok[i] || tok >= min(seq_end, Q.lim[t]))) x = -__builtin_inff();
                s[i][t][e] = x;
                top = fmaxf(top, x);
            }
        }
    return top;
}
// V scales of the lane's tokens over the scale reference, largest of them
template <int D, int NT, bool MASKED>
__device__ __forceinline__ float value_scales(const State<D, NT>& S, const Params& P, const Ptrs& a, int seq_end, int kg, float (&vs)[2][4]) {
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            vs[i][e] = lo16(P.v[i][e]) * S.inv_r;
            if (MASKED && (!a.ok[i] || a.tok[i] + 4 * kg + e >= seq_end)) vs[i][e] = 0.f;
            top = fmaxf(top, vs[i][e]);
        }
    return top;
}
// The slow path: rows' references to their true maxima, the scale reference where it is free or outgrown.
template <int D, int NT>
__device__ __forceinline__ void move_references(State<D, NT>& S, f32x4 (&s)[2][NT], float (&vs)[2][4], float vs_top) {
    float vmax = fminf(vs_top, 3.0e38f);
    for (int d = 1; d < 64; d <<= 1) vmax = fmaxf(vmax, __shfl_xor(vmax, d));
    float r = 1.f;
    if (vmax > (float)(2 << kScaleTop) || ((S.open & 2) && vmax > 0.f)) {
        const int e = max(-60, min(60, (int)((__float_as_uint(vmax) >> 23) & 255u) - 127 + 1 - kScaleTop));
        r = __uint_as_float((uint32_t)(127 - e) << 23);   // vmax * r in [2^5, 2^6)
        S.open &= 1;
    }
    S.inv_r *= r;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) vs[i][e] *= r;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        float top = -__builtin_inff();
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) top = fmaxf(top, s[i][t][e]);
        top = rows_max(top);
        const bool before = (S.seen >> t) & 1, now = top > -__builtin_inff();
        const float up = before ? fmaxf(top, 0.f) : (now ? top : 0.f);
        const float alpha = before ? fast_exp2(-up) : 1.f;      // (nothing is in the sums before the first token)
        S.m[t] += up;
        S.l[t] *= alpha;
        S.z[t] *= alpha;
        S.r[t] *= alpha * r;
#pragma unroll
        for (int d = 0; d < D / 16; ++d) S.o[t][d] *= alpha * r;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[i][t][e] -= up;
        if (now) S.seen |= 1 << t;
    }
    const int none = __any(S.seen != (1 << NT) - 1) ? 1 : 0;
    S.open = __builtin_amdgcn_readfirstlane((S.open & 2) | none);
}
// probabilities into the sums and into operand B of the second product: tokens (0, 2), (1, 3) of the lane's four, first
// half then second half
template <int D, int NT, bool MASKED>
__device__ __forceinline__ void weights(State<D, NT>& S, const Params& P, const f32x4 (&s)[2][NT], const float (&vs)[2][4], u32x4 (&pb)[NT]) {
    float w[NT][2][4];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float vz = fmaf(7.5f, lo16(P.v[i][e]), hi16(P.v[i][e]));
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const float x = s[i][t][e], pr = fast_exp2(x);
                const bool hidden = MASKED && x == -__builtin_inff();
                S.l[t] += pr;
                S.z[t] = hidden ? S.z[t] : fmaf(pr, vz, S.z[t]);
                w[t][i][e] = hidden ? 0.f : pr * vs[i][e];
            }
        }
#pragma unroll
    for (int t = 0; t < NT; ++t)
        pb[t] = u32x4{pack_f16(w[t][0][0], w[t][0][2]), pack_f16(w[t][0][1], w[t][0][3]), pack_f16(w[t][1][0], w[t][1][2]),
                      pack_f16(w[t][1][1], w[t][1][3])};
}
template <int D, int NT>
__device__ __forceinline__ void accumulate(State<D, NT>& S, const uint8_t* slot, const u32x4 (&pb)[NT], int lane) {
    const Words<D / 32> v0 = v_words<D>(slot, 0, lane), v1 = v_words<D>(slot, 1, lane);
    const u32x4 ones = {0x3c003c00u, 0x3c003c00u, 0x3c003c00u, 0x3c003c00u};
#pragma unroll
    for (int t = 0; t < NT; ++t) S.r[t] = mfma(ones, pb[t], S.r[t]);
#pragma unroll
    for (int j = 0; j < D / 32; ++j) {
        const u32x4 c0 = codes_of(v0.w[j]), c1 = codes_of(v1.w[j]);
        const u32x4 even = {c0[0], c0[2], c1[0], c1[2]}, odd = {c0[1], c0[3], c1[1], c1[3]};
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            S.o[t][2 * j] = mfma(even, pb[t], S.o[t][2 * j]);
            S.o[t][2 * j + 1] = mfma(odd, pb[t], S.o[t][2 * j + 1]);
        }
    }
}

// ---- finished states ------------------------------------------------------------------------------------------------
// Per row: D un-normalised outputs, the reference m (log2) and the sum l, complete in every lane of the row; a row without
// tokens has m = kNoMax, l = 0.
template <int D, int NT>
__device__ __forceinline__ void settle(State<D, NT>& S) {
    const float even = 16777216.f / S.inv_r, odd = even * 0.0625f, mid = 7.5f / S.inv_r;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        S.l[t] = rows_sum(S.l[t]);
        const float z = rows_sum(S.z[t]) - S.r[t][0] * mid;
        if (!((S.seen >> t) & 1) && !(S.l[t] != S.l[t])) S.m[t] = kNoMax;
#pragma unroll
        for (int d = 0; d < D / 16; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) S.o[t][d][i] = S.o[t][d][i] * ((d & 1) ? odd : even) + z;
    }
}
// channel of o[.][d][i] in a lane: kg * D / 4 + i * D / 16 + d
template <int D, int NT>
__device__ __forceinline__ void state_to_lds(const State<D, NT>& S, float* st, int lane) {
    const int n = lane & 15, kg = lane >> 4;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        float* row = st + (16 * t + n) * (D + 2);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int d = 0; d < D / 16; ++d) row[kg * (D / 4) + i * (D / 16) + d] = S.o[t][d][i];
        if (kg == 0) { row[D] = S.m[t]; row[D + 1] = S.l[t]; }
    }
}
template <int D, int NT>
__device__ __forceinline__ void merge_from_lds(State<D, NT>& S, const float* st, int lane) {
    const int n = lane & 15, kg = lane >> 4;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const float* row = st + (16 * t + n) * (D + 2);
        const float mo = row[D], lo = row[D + 1], m = fmaxf(S.m[t], mo);
        const float a = fast_exp2(S.m[t] - m), b = fast_exp2(mo - m);
        S.m[t] = m;
        S.l[t] = S.l[t] * a + lo * b;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int d = 0; d < D / 16; ++d) S.o[t][d][i] = S.o[t][d][i] * a + row[kg * (D / 4) + i * (D / 16) + d] * b;
    }
}

__device__ __forceinline__ void put_out(const Int4AttnParams& p, long long at, float a, float b) {
    if (p.out_dtype == kF32) *(float2*)((float*)p.out + at) = make_float2(a, b);
    else if (p.out_dtype == kBF16)
        *(uint32_t*)((uint16_t*)p.out + at) = (uint32_t)__builtin_bit_cast(uint16_t, (__bf16)a) | ((uint32_t)__builtin_bit_cast(uint16_t, (__bf16)b) << 16);
    else *(uint32_t*)((uint16_t*)p.out + at) = pack_f16(a, b);
}
__device__ __forceinline__ float out_factor(float l) { return l == 0.f ? 0.f : 1.f / l; }
__device__ __forceinline__ float lse_of(float m, float l) { return l == 0.f ? -3.4e38f : (m + __log2f(l)) * 0.6931471805599453f; }

template <int D, int NT>
__device__ __forceinline__ void write_out(const Int4AttnParams& p, const Rows& R, int row0, const State<D, NT>& S, int lane) {
    const int n = lane & 15, kg = lane >> 4;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int r = row0 + 16 * t + n;
        if (r >= R.n) continue;
        const int i0 = r / R.G, head = R.head0 + r - i0 * R.G;
        const long long row = (long long)(R.first + i0) * p.Hq + head;
        const float f = out_factor(S.l[t]);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int d = 0; d < D / 16; d += 2)
                put_out(p, row * D + kg * (D / 4) + i * (D / 16) + d, S.o[t][d][i] * f, S.o[t][d + 1][i] * f);
        if (p.lse && kg == 0) p.lse[row] = lse_of(S.m[t], S.l[t]);
    }
}

union Pair { unsigned long long u; float f[2]; };
__device__ __forceinline__ void st_pair(float* ptr, float a, float b) {
    Pair v;
    v.f[0] = a; v.f[1] = b;
    st_agent((unsigned long long*)ptr, v.u);
}
__device__ __forceinline__ Pair ld_pair(const float* ptr) {
    Pair v;
    v.u = ld_agent((const unsigned long long*)ptr);
    return v;
}
// A partial state in the workspace, tile by tile of 16 rows as the lanes hold it, so that every access is 512 contiguous
// bytes: [tile][d][pair of o's elements][lane] pairs of outputs, then [tile][lane] (m, l).
template <int D> constexpr int part_tile_floats() { return (D / 16 * 2 + 1) * 128; }
template <int D, int NT>
__device__ __forceinline__ void state_to_part(const State<D, NT>& S, float* part, int tile0, int n_rows, int lane) {
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        if ((tile0 + t) * 16 >= n_rows) break;
        float* at = part + (long long)(tile0 + t) * part_tile_floats<D>() + 2 * lane;
#pragma unroll
        for (int d = 0; d < D / 16; ++d) {
            st_pair(at + (2 * d) * 128, S.o[t][d][0], S.o[t][d][1]);
            st_pair(at + (2 * d + 1) * 128, S.o[t][d][2], S.o[t][d][3]);
        }
        st_pair(at + (D / 16 * 2) * 128, S.m[t], S.l[t]);
    }
}

// The last workgroup to arrive at a split item merges its np partial states, which lie `stride` floats apart except for
// the first.  The waves share the tiles, or the channels of a tile where tiles are fewer; the loads of BATCH states are
// under way at once (they come past the caches, about 2 us each).
template <int D, int TILES>
__device__ __forceinline__ void merge_parts(const Int4AttnParams& p, const Rows& R, int row0, int n_rows, const float* first,
                                            const float* rest, long long stride, int np, int wave, int lane) {
    constexpr int WANT = TILES >= 4 ? 1 : 4 / TILES, SHARE = WANT < D / 32 ? WANT : D / 32;   // waves of a tile
    constexpr int DW = D / 16 / SHARE;                         // d's of a wave
    constexpr int BATCH = DW <= 2 ? 8 : (DW <= 8 ? 4 : 2);
    const int n = lane & 15, kg = lane >> 4, d0 = wave % SHARE * DW;
    for (int tile = wave / SHARE; tile * 16 < n_rows; tile += 4 / SHARE) {
        const long long off = (long long)tile * part_tile_floats<D>() + 2 * lane;
        float m = kNoMax, l = 0.f;
        f32x4 o[DW];
#pragma unroll
        for (int d = 0; d < DW; ++d) o[d] = f32x4{0.f, 0.f, 0.f, 0.f};
        for (int p0 = 0; p0 < np; p0 += BATCH) {
            Pair ml[BATCH], a[BATCH][DW], b[BATCH][DW];
#pragma unroll
            for (int u = 0; u < BATCH; ++u) {
                const int j = min(p0 + u, np - 1);
                const float* at = (j == 0 ? first : rest + (long long)(j - 1) * stride) + off;
                ml[u] = ld_pair(at + (D / 16 * 2) * 128);
#pragma unroll
                for (int d = 0; d < DW; ++d) {
                    a[u][d] = ld_pair(at + (2 * (d0 + d)) * 128);
                    b[u][d] = ld_pair(at + (2 * (d0 + d) + 1) * 128);
                }
            }
            float top = m;
#pragma unroll
            for (int u = 0; u < BATCH; ++u) top = fmaxf(top, ml[u].f[0]);
            const float keep = fast_exp2(m - top);
            m = top;
            l *= keep;
#pragma unroll
            for (int d = 0; d < DW; ++d) o[d] *= keep;
#pragma unroll
            for (int u = 0; u < BATCH; ++u)
                if (p0 + u < np) {
                    const float f = fast_exp2(ml[u].f[0] - top);
                    l += ml[u].f[1] * f;
#pragma unroll
                    for (int d = 0; d < DW; ++d)
                        o[d] += f32x4{a[u][d].f[0] * f, a[u][d].f[1] * f, b[u][d].f[0] * f, b[u][d].f[1] * f};
                }
        }
        const int r = tile * 16 + n;
        if (r < n_rows) {
            const int rr = row0 + r, i0 = rr / R.G, head = R.head0 + rr - i0 * R.G;
            const long long row = (long long)(R.first + i0) * p.Hq + head;
            const float f = out_factor(l);
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int d = 0; d < DW; d += 2)
                    put_out(p, row * D + kg * (D / 4) + i * (D / 16) + d0 + d, o[d][i] * f, o[d + 1][i] * f);
            if (p.lse && kg == 0 && d0 == 0) p.lse[row] = lse_of(m, l);
        }
    }
}

// ---- the kernel -----------------------------------------------------------------------------------------------------
// Steps under way per wave: as many as two workgroups per CU have LDS for.
#ifndef KV_DEPTH
#define KV_DEPTH 4
#endif
template <int D> constexpr int depth() { return D >= 256 ? 2 : KV_DEPTH; }
template <int D, int NT, int RW, bool LIST>
struct Lds {
    static constexpr int ring = depth<D>() * Slot<D>::bytes + 512;                      // of a wave: steps, table entries
    static constexpr int merge = RW == 4 ? 0 : 2 * 16 * NT * (D + 2) * 4;               // two states, after the walk
    static constexpr int head = 4 * ring > merge ? 4 * ring : merge;
    static constexpr int fixed = head + 16;                                             // the flag
};

// Steps [s0, s1) of an item for this wave: every (4 / RW)-th one from s0 + wave / RW.  A step's slot is filled again as
// soon as the step is done.  The loads are not conditional (behind the end the last step is loaded again, from the cache),
// so that counting them is enough to know what has arrived.
template <int D, int NT, int RW, bool LIST>
__device__ __forceinline__ void walk(const Int4AttnParams& p, const Seq& sq, int b, const Rows& R, int row0, State<D, NT>& S, int s0, int s1,
                                     const int2* list, int n_list, uint8_t* ring, int wave, int lane) {
    constexpr int stride = 4 / RW, DEPTH = depth<D>(), LOADS = Slot<D>::loads;
    const int seq_end = sq.len, kg = lane >> 4;
    Query<D, NT> Q;
    set_limits<D, NT>(p, sq, R, row0, Q, lane);
    int s = s0 + wave / RW;
    // no row of the wave sees anything from lim_max on (lists are not ordered by position: all of theirs is walked)
    if (!LIST) s1 = min(s1, (min(Q.lim_max, seq_end) + kInt4StepTokens - 1) / kInt4StepTokens);
    if (s >= s1) {
        clear_state(S);
        return;
    }
    RawQuery<D, NT> raw;
    load_query<D, NT>(p, R, row0, raw, lane);
    const int last = s + (s1 - 1 - s) / stride * stride;
    const int32_t* table = p.map.block_table + (long long)b * p.map.max_page;
    const int bs = p.map.block_size;
    // page of 16 tokens: (units of 16) * ceil(2^32 / (bs / 16)) >> 32, exact below 2^22 units
    auto page_of = [&](unsigned u) { return (int)(p.page_magic ? __umulhi(u, p.page_magic) : u); };
    // 64 table entries in a register, so that a lookup is a lane read; the next 64 come through LDS like the steps' data and
    // have long arrived when they are needed (64 pages are at least 8 steps, more than are under way)
    uint32_t* const window = (uint32_t*)(ring + DEPTH * Slot<D>::bytes);
    auto entry = [&](int i) { return (const uint32_t*)table + min(i, p.map.max_page - 1); };
    int base = page_of(2u * (unsigned)s) & ~63, cur = 0;
    if (!LIST) {
        word_to_lds(entry(base + 64 + lane), window + ((base + 64) & 64));
        cur = *(const volatile int*)entry(base + lane);        // (after the load above: both have arrived with it)
    }
    const int page_rows = p.Hkv * bs, first_row = R.kvh * bs;
    auto place = [&](int step, int i, Ptrs& a) {
        const unsigned u = 2u * (unsigned)step + i;
        const int page = page_of(u), in_page = (int)(16u * u) - page * bs;
        int e;
        if (LIST) {
            const int2 le = page < n_list ? list[page] : make_int2(0, -1);
            a.tok[i] = uni(le.x) * bs + in_page;
            e = uni(le.y);
        } else {
            a.tok[i] = (int)(16u * u);
            while (page - base >= 64) {
                base += 64;
                cur = (int)window[(base & 64) + lane];
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                word_to_lds(entry(base + 64 + lane), window + ((base + 64) & 64));
            }
            e = a.tok[i] < seq_end ? __builtin_amdgcn_readlane(cur, page - base) : -1;
        }
        a.ok[i] = (unsigned)e < (unsigned)p.map.n_blocks;
        a.row[i] = (long long)(a.ok[i] ? e : 0) * page_rows + (first_row + in_page);
    };
    auto locate = [&](int step, Ptrs& a) {
        place(step, 0, a);
        if (p.paired) {                     // both halves in one page
            a.row[1] = a.row[0] + 16;
            a.tok[1] = a.tok[0] + 16;
            a.ok[1] = a.ok[0];
        } else {
            place(step, 1, a);
        }
    };
    const uint32_t* par = (lane < 32 ? p.k_params : p.v_params) + (lane & 31);
    const int end = min(seq_end, Q.lim_min);
    auto compute = [&](const uint8_t* slot, const Ptrs& a) {
        f32x4 x[2][NT];
        u32x4 pb[NT];
        const Params P = params_of<D>(slot, lane);
        products<D, NT>(Q, slot, x, lane);
        const bool masked = !a.ok[0] || !a.ok[1] || max(a.tok[0], a.tok[1]) + 16 > end;
        float vs[2][4], top, vs_top;
        if (masked) {
            top = scores<D, NT, true>(Q, S, P, a, seq_end, kg, x);
            vs_top = value_scales<D, NT, true>(S, P, a, seq_end, kg, vs);
        } else {
            top = scores<D, NT, false>(Q, S, P, a, seq_end, kg, x);
            vs_top = value_scales<D, NT, false>(S, P, a, seq_end, kg, vs);
        }
        if (masked || S.open || __any(top > kLazy || vs_top > (float)(2 << kScaleTop))) move_references<D, NT>(S, x, vs, vs_top);
        if (masked) weights<D, NT, true>(S, P, x, vs, pb);
        else weights<D, NT, false>(S, P, x, vs, pb);
        accumulate<D, NT>(S, slot, pb, lane);
    };
    Ptrs a[DEPTH];
#pragma unroll
    for (int u = 0; u < DEPTH; ++u) {
        locate(min(s + u * stride, last), a[u]);
        fetch<D, RW == 1>(p, par, a[u], ring + u * Slot<D>::bytes, lane);
    }
    make_query<D, NT>(p, raw, Q);       // while the first steps' data is on its way
    clear_state(S);
#pragma unroll 1
    while (true) {
#pragma unroll
        for (int u = 0; u < DEPTH; ++u) {
            uint8_t* const slot = ring + u * Slot<D>::bytes;
            wait_loads<(DEPTH - 1) * LOADS>();
            compute(slot, a[u]);
            s += stride;
            if (s >= s1) {
                wait_loads<0>();         // nothing may land in LDS after this
                return;
            }
            locate(min(s + (DEPTH - 1) * stride, last), a[u]);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");     // the slot has been read
            fetch<D, RW == 1>(p, par, a[u], slot, lane);
        }
    }
}

// One item, steps [s0, s1) of n_steps: the whole of it is written out, a part goes to the workspace and the last
// workgroup to arrive merges.  part: where this workgroup's state goes; first / rest / stride / np: where all of them are.
template <int D, int NT, int RW, bool LIST>
__device__ __forceinline__ void run_item(const Int4AttnParams& p, const Seq& sq, int b, const Rows& R, int row0, int s0, int s1, bool whole,
                                         float* part, const float* first, const float* rest, long long stride, int np,
                                         unsigned* counter, const int2* list, int n_list, float* lds, int* flag, int wave, int lane) {
    const int my_row0 = row0 + wave % RW * 16 * NT;
    const int n_rows = min(p.rows_tile, R.n - row0);
    State<D, NT> S;
    if (RW < 4) __syncthreads();                          // the areas may still be read for the item before
    walk<D, NT, RW, LIST>(p, sq, b, R, my_row0, S, s0, s1, list, n_list, (uint8_t*)lds + wave * Lds<D, NT, RW, LIST>::ring, wave, lane);
    settle<D, NT>(S);
    // the waves that hold the same rows merge pairwise
    float* const area[2] = {lds, lds + 16 * NT * (D + 2)};
    if (RW < 4) {
        __syncthreads();                                  // every wave has left its ring
        const int odd = RW == 1 ? wave & 1 : wave >> 1, which = RW == 1 ? wave >> 1 : wave & 1;
        if (odd) state_to_lds<D, NT>(S, area[which], lane);
        __syncthreads();
        if (!odd) merge_from_lds<D, NT>(S, area[which], lane);
    }
    if (RW == 1) {
        __syncthreads();
        if (wave == 2) state_to_lds<D, NT>(S, lds, lane);
        __syncthreads();
        if (wave == 0) merge_from_lds<D, NT>(S, lds, lane);
    }
    const bool mine = wave < RW;
    if (whole) {
        if (mine) write_out<D, NT>(p, R, my_row0, S, lane);
        return;
    }
    if (mine) state_to_part<D, NT>(S, part, wave % RW * NT, n_rows, lane);
    wait_stores();
    __syncthreads();
    if (threadIdx.x == 0)
        *flag = (int)__hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == np - 1;
    __syncthreads();
    const int last = *flag;
    if (last) {
        if (threadIdx.x == 0) st_agent(counter, 0u);      // left as found: the next launch on this workspace counts again
        merge_parts<D, NT * RW>(p, R, row0, n_rows, first, rest, stride, np, wave, lane);
    }
    __syncthreads();
}

template <int D, int NT, int RW, bool LIST>
__global__ __launch_bounds__(256, 2) void int4_attention_kernel(const Int4AttnParams p) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    float* lds = (float*)smem;
    int* flag = (int*)(smem + Lds<D, NT, RW, LIST>::head);
    const int lane = lane_id(), wave = wave_id();
    constexpr long long state = (long long)NT * RW * part_tile_floats<D>();

    if constexpr (LIST) {
        const int item = blockIdx.x / p.workers, share = blockIdx.x - item * p.workers;
        const int b = item / p.list_rows, lr = item - b * p.list_rows;
        const Seq sq = uniform_seq(p.map, b);
        const bool per_head = p.list_rows == p.Hq;
        const Rows R{sq.first, per_head ? lr : lr * p.G, per_head ? 1 : p.G, per_head ? lr / p.G : lr, per_head ? 1 : p.G};
        int2* list = (int2*)(smem + Lds<D, NT, RW, LIST>::fixed);
        // a list ends at its first entry outside the table (the sentinel among them): the shortest over the threads
        if (threadIdx.x == 0) *flag = p.P;
        __syncthreads();
        const int32_t* src = p.lists + ((long long)b * p.list_rows + lr) * p.P;
        int end = p.P;
        for (int j = threadIdx.x; j < p.P; j += 256) {
            const int lp = src[j];
            const bool ok = lp >= 0 && lp < p.map.max_page;
            list[j] = make_int2(ok ? lp : 0, ok ? p.map.block_table[(long long)b * p.map.max_page + lp] : -1);
            if (!ok && j < end) end = j;
        }
        if (end < p.P) atomicMin(flag, end);
        __syncthreads();
        const int n_list = uni(*flag);
        const int n_steps = (int)(((long long)n_list * p.map.block_size + kInt4StepTokens - 1) / kInt4StepTokens);
        const int s0 = (int)((long long)n_steps * share / p.workers), s1 = (int)((long long)n_steps * (share + 1) / p.workers);
        float* base = p.parts + (long long)item * p.workers * state;
        run_item<D, NT, RW, LIST>(p, sq, b, R, 0, s0, s1, p.workers == 1, base + share * state, base, base + state, state, p.workers,
                                    p.counters + item, list, n_list, lds, flag, wave, lane);
    } else {
        if (p.zero_rest && p.map.query_start) {           // rows of no sequence
            const int T = p.map.T, from = max(0, min(p.map.query_start[p.map.B], T)), lead = max(0, min(p.map.query_start[0], T));
            for (long long r = blockIdx.x; r < lead + (long long)(T - from); r += gridDim.x) {
                const long long t = r < lead ? r : from + (r - lead);
                for (int e = threadIdx.x * 2; e < p.Hq * D; e += 512) put_out(p, t * p.Hq * D + e, 0.f, 0.f);
                if (p.lse) for (int e = threadIdx.x; e < p.Hq; e += 256) p.lse[t * p.Hq + e] = -3.4e38f;
            }
        }
        // Consecutive pieces go to workgroups of one XCD (workgroups are dealt to the eight XCDs in turn), so that the row
        // tiles of a kv head meet its tokens in one L2.
        const int per = (p.workers + 7) / 8;
        const int w = (int)(blockIdx.x & 7) * per + (int)(blockIdx.x >> 3);
        if (w >= p.workers) return;
        Piece pc;
        if (!(p.wide_line ? find_piece<long long>(p, w, lane, pc) : find_piece<int>(p, w, lane, pc))) return;
        const long long piece = uni(pc.size), g1 = uni(pc.g1);
        long long g = uni(pc.g);
        int b = pc.b, h = pc.h, rt = pc.rt, s0 = pc.s0;
        Seq sq = uniform_seq(p.map, b);
        while (true) {
            const int n_steps = uni(steps_of(p, sq, rt));
            const int s1 = (int)min((long long)n_steps, s0 + (g1 - g));
            const long long item0 = g - s0;
            const int w0 = uni((int)quotient(item0, piece)), w1 = uni((int)quotient(item0 + n_steps - 1, piece));
            const Rows R{sq.first, h * p.G, p.G, h, sq.n * p.G};
            // slot 2 w + 1: the item begins in w's piece; slot 2 w: it began before
            run_item<D, NT, RW, LIST>(p, sq, b, R, rt * p.rows_tile, s0, s1, w0 == w1, p.parts + (2ll * w + (s0 == 0)) * state,
                                        p.parts + (2ll * w0 + 1) * state, p.parts + 2ll * (w0 + 1) * state, 2 * state, w1 - w0 + 1,
                                        p.counters + w0, nullptr, 0, lds, flag, wave, lane);
            g += s1 - s0;
            if (g >= g1) break;
            s0 = 0;
            if (++rt == row_tiles(p, sq)) {
                rt = 0;
                if (++h == p.Hkv) {
                    h = 0;
                    do sq = uniform_seq(p.map, ++b); while (sq.n == 0);
                }
            }
        }
    }
}

template <int D, int NT, int RW, bool LIST>
hipError_t launch_one(const Int4AttnParams& p, hipStream_t s, int* resident) {
    auto kern = int4_attention_kernel<D, NT, RW, LIST>;
    const size_t lds_bytes = (size_t)Lds<D, NT, RW, LIST>::fixed + (LIST ? (size_t)p.P * sizeof(int2) : 0);
    static int lds_limit[kMaxDevices];
    hipError_t e = ensure_lds_limit((const void*)kern, lds_limit, lds_bytes);
    if (e != hipSuccess) return e;
    if (resident) {
        static int seen[kMaxDevices];     // (the lists' kernels are not resident grids: asked with the smallest list)
        static std::mutex seen_mutex;
        int dev = 0, occ = 0;
        e = hipGetDevice(&dev);
        if (e != hipSuccess) return e;
        if (dev < 0 || dev >= kMaxDevices) return hipErrorInvalidDevice;
        std::lock_guard<std::mutex> lock(seen_mutex);
        if (seen[dev] == 0) {
            e = hipOccupancyMaxActiveBlocksPerMultiprocessor(&occ, kern, 256, (size_t)Lds<D, NT, RW, LIST>::fixed);
            if (e != hipSuccess) return e;
            seen[dev] = (occ < 1 ? 1 : occ) * device_cu_count();
        }
        *resident = seen[dev];
        return hipSuccess;
    }
    const unsigned grid = LIST ? (unsigned)(p.map.B * p.list_rows * p.workers) : (unsigned)((p.workers + 7) / 8 * 8);
    if (grid == 0) return hipSuccess;
    count_launch();
    hipLaunchKernelGGL(kern, dim3(grid), dim3(256), lds_bytes, s, p);
    return hipGetLastError();
}

template <int D, bool LIST>
hipError_t dispatch(const Int4AttnParams& p, hipStream_t s, int* resident) {
    constexpr int N = D <= 128 ? 2 : 1;      // row tiles of a wave (registers)
    if (p.nt == 1 && p.row_waves == 1) return launch_one<D, 1, 1, LIST>(p, s, resident);
    if constexpr (N == 2) if (p.nt == 2 && p.row_waves == 1) return launch_one<D, 2, 1, LIST>(p, s, resident);
    if (p.nt == N && p.row_waves == 2) return launch_one<D, N, 2, LIST>(p, s, resident);
    if (p.nt == N && p.row_waves == 4) return launch_one<D, N, 4, LIST>(p, s, resident);
    return hipErrorInvalidConfiguration;
}
template <int D>
hipError_t dispatch(const Int4AttnParams& p, hipStream_t s, int* resident) {
    return p.lists ? dispatch<D, true>(p, s, resident) : dispatch<D, false>(p, s, resident);
}
hipError_t any_launch(const Int4AttnParams& p, hipStream_t s, int* resident) {
    switch (p.D) {
        case 32: return dispatch<32>(p, s, resident);
        case 64: return dispatch<64>(p, s, resident);
        case 128: return dispatch<128>(p, s, resident);
        case 256: return dispatch<256>(p, s, resident);
    }
    return hipErrorInvalidValue;
}

}  // namespace

hipError_t launch_int4_attention(const Int4AttnParams& p, hipStream_t s) { return any_launch(p, s, nullptr); }
long long int4_attention_part_bytes(const Int4AttnParams& p) { return (long long)(p.rows_tile / 16) * (p.D / 16 * 2 + 1) * 128 * 4; }
int int4_attention_resident(const Int4AttnParams& p) {
    int n = 0;
    if (device_cu_count() <= 0 || any_launch(p, nullptr, &n) != hipSuccess) { (void)hipGetLastError(); return 0; }
    return n;
}

}  // namespace spfa
