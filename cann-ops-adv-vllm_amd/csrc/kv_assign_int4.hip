// Cluster ids of newly filled pages of a 4-bit key cache: assign_block_ids (see spfa_assign.inc for the definition) with
// K_t = scale_t code_t + zero_t, so a page's mean is (sum_t scale_t code_t + sum_t zero_t) / n.
//
// A workgroup takes up to 32 new pages of one kv head and all or a slice of the head's centroids: its sixteen waves form
// the pages' means, then walk the centroids in tiles of 16, pages x centroids on the matrix cores (fp32 accumulation in
// the order of the channels), and keep the best cluster of every page as they go.
//
// What bounds it: the pages come from HBM once, and that is the floor; but each workgroup also reads its centroids from
// L2, half a megabyte for 2048 of them.  So as many pages as possible share a pass over the centroids, and where the pages
// are few (a decode step's) the centroids are sliced over workgroups that each form the means again from L2; their results
// join by an atomic maximum of (score, cluster), which no order of arrival changes.
// Which pages are new is known on the device only: every workgroup counts them and derives the split from their number.
// Measured, D = 128, pages of 128 tokens, 8 heads x 2048 clusters (a call, launch included): 64 pages 18 us, 1024
// pages 23 us, of which reading the pages takes 11 (64 MB, 6 TB/s) and the centroids 8 (18 when the lanes load them as the
// matrix instruction wants them).  With the scores of 16 pages kept in LDS and no slices, as the kernel for the other types
// has it, they took 41 and 103.
#include "spfa_params.h"

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace spfa {
namespace {

#include "spfa_common.inc"
#include "kv_lds.inc"

constexpr int kRows = 32, kFew = 16;                // most pages of a workgroup; pages before slices make way for more pages
constexpr int kSpread = 256;                        // workgroups that fill the card

struct Slot { int b, page, phys, valid; };

__device__ __forceinline__ int new_pages(const AssignParams& p, int b, int* first) {
    const int len = p.seq_len[b], page_len = len > 0 ? min((int)((unsigned)(len - 1) / (unsigned)p.block_size) + 1, p.max_page) : 0;
    *first = max(0, p.first_new[b]);
    return max(0, min(page_len - *first, p.max_new));
}
__device__ __forceinline__ int scan64(int x, int lane) {
#pragma unroll 1
    for (int d = 1; d < 64; d <<= 1) {
        const int up = __shfl_up(x, d);
        if (lane >= d) x += up;
    }
    return x;
}

// Sums of a page on the matrix cores, contraction over 32 tokens at a time: row of A = the tokens' scales (all 16 rows
// alike), column of B = a channel's codes.  A code is a 16-bit pattern 0x000c or 0x00c0, the float16 denormal c 2^-24 or
// c 2^-20, so two tokens' codes cost one byte permutation per two channels and one mask each (0.75 instructions a code
// against 2.4 with conversions and fmas), products and sums are exact to fp32, and the sums need no exchange between lanes.
// Lane l holds channels CH (l % 16) .. + CH - 1 of tokens 8 (l / 16) .. + 7; steps first, first + skip, ... of 32 tokens.
// sum[c] gets scale * code of channel CH (l % 16) + c plus the zeros, in every lane.
template <int D>
__device__ __forceinline__ void page_sum(const AssignParams& p, const Slot& s, int n2, int first, int skip, int lane, float (&sum)[D / 16]) {
    constexpr int CH = D / 16, BYTES = CH / 2;
    const int col = lane & 15, kq = lane >> 4;
    const uint8_t* base = (const uint8_t*)p.kcache + (long long)s.phys * p.blk_stride + (long long)n2 * p.head_stride + col * BYTES;
    const uint32_t* par = (const uint32_t*)p.key_params + ((long long)s.phys * p.Hkv + n2) * p.block_size;
    f32x4 acc[CH], zero = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int c = 0; c < CH; ++c) acc[c] = f32x4{0.f, 0.f, 0.f, 0.f};
    const uint32_t one2 = 0x3c003c00u;
    const half8 ones = __builtin_bit_cast(half8, uint4{one2, one2, one2, one2});
    struct Step { uint64_t w[8]; uint4 s0, s1; };
    auto load = [&](Step& to, int t0) {
        // block_size is a multiple of 16: eight tokens are in the block or none is (those behind it count for nothing below)
        const int t = t0 + kq * 8, ts = t < p.block_size ? t : 0;
        to.s0 = ((const uint4*)(par + ts))[0];
        to.s1 = ((const uint4*)(par + ts))[1];
        const uint8_t* at = base + (long long)ts * p.tok_stride;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if constexpr (BYTES == 8) to.w[i] = *(const uint64_t*)at;
            else if constexpr (BYTES == 4) to.w[i] = *(const uint32_t*)at;
            else if constexpr (BYTES == 2) to.w[i] = *(const uint16_t*)at;
            else to.w[i] = *at;
            at += p.tok_stride;
        }
    };
    auto add = [&](const Step& d, int t0) {
        const int t = t0 + kq * 8;
        const uint32_t sz[8] = {d.s0.x, d.s0.y, d.s0.z, d.s0.w, d.s1.x, d.s1.y, d.s1.z, d.s1.w};
        uint32_t sc[4], ze[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {      // rows behind the end may hold anything: neither scale nor zero of theirs counts
            const uint32_t lo = t + 2 * i < s.valid ? sz[2 * i] : 0u, hi = t + 2 * i + 1 < s.valid ? sz[2 * i + 1] : 0u;
            sc[i] = __builtin_amdgcn_perm(hi, lo, 0x05040100u);
            ze[i] = __builtin_amdgcn_perm(hi, lo, 0x07060302u);
        }
        const half8 scales = __builtin_bit_cast(half8, uint4{sc[0], sc[1], sc[2], sc[3]});
        zero = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, uint4{ze[0], ze[1], ze[2], ze[3]}), ones, zero, 0, 0, 0);
#pragma unroll
        for (int b = 0; b < BYTES; ++b) {
            uint32_t lo[4], hi[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t w0 = (uint32_t)(d.w[2 * i] >> (b / 4 * 32)), w1 = (uint32_t)(d.w[2 * i + 1] >> (b / 4 * 32));
                const uint32_t two = __builtin_amdgcn_perm(w1, w0, 0x0c040c00u + (uint32_t)(b % 4) * 0x00010001u);
                lo[i] = two & 0x000f000fu;
                hi[i] = two & 0x00f000f0u;
            }
            acc[2 * b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(scales, __builtin_bit_cast(half8, uint4{lo[0], lo[1], lo[2], lo[3]}), acc[2 * b], 0, 0, 0);
            acc[2 * b + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(scales, __builtin_bit_cast(half8, uint4{hi[0], hi[1], hi[2], hi[3]}), acc[2 * b + 1], 0, 0, 0);
        }
    };
    // two steps under way; a step behind the page's end adds zeros
    Step x, y;
    load(x, first * 32);
#pragma unroll 1
    for (int t0 = first * 32; t0 < s.valid; t0 += 2 * skip * 32) {
        load(y, t0 + skip * 32);
        add(x, t0);
        load(x, t0 + 2 * skip * 32);
        add(y, t0 + skip * 32);
    }
#pragma unroll
    for (int c = 0; c < CH; ++c) sum[c] = acc[c][0] * (c % 2 ? 0x1p20f : 0x1p24f) + zero[0];
}

template <int BY>
__device__ __forceinline__ void join_turned(float (&best)[2][4], int (&id)[2][4]) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float so = dpp<0x120 + BY>(best[h][i]);            // rotation within 16 lanes
            const int co = __builtin_amdgcn_update_dpp(0, id[h][i], 0x120 + BY, 0xf, 0xf, true);
            const bool other = (so > best[h][i]) | ((so == best[h][i]) & (co < id[h][i]));
            best[h][i] = other ? so : best[h][i];
            id[h][i] = other ? co : id[h][i];
        }
}

template <int D> constexpr int tile_bytes() { return 16 * D * 2; }           // sixteen centroids
template <int D> constexpr int waves() { return D < 256 ? 16 : 8; }      // (D = 256 needs the registers of two)

template <int D, bool BF>
__global__ __launch_bounds__(waves<D>() * 64) void assign_int4_kernel(const AssignParams p) {
    constexpr int KS = D / 32, CH = D / 16, kWaves = waves<D>();
    extern __shared__ __attribute__((aligned(16))) char smem[];       // the waves' tiles of centroids, two each, then the means
    uint16_t* const a_tile = (uint16_t*)(smem + kWaves * 2 * tile_bytes<D>());
    __shared__ Slot slots[kRows];
    __shared__ int n_slots, n_slices, last;
    __shared__ float parts[kWaves][D];
    __shared__ unsigned long long keys[kRows];       // best (score, cluster) of every page
    const int lane = lane_id(), wave = wave_id();
    const int n2 = blockIdx.x % p.Hkv, rest = blockIdx.x / p.Hkv;
    const int col = lane & 15, kq = lane >> 4, tiles = (p.C + 15) / 16;

    // ---- this workgroup's pages: some of the new pages in the order (sequence, page) ----
    if (wave == 0) {
        // (B max_new Hkv < 2^31, which the host checks: 32-bit counts)
        int total = 0, first = 0, count = 0, incl = 0;
        for (int b0 = 0; b0 < p.B; b0 += 64) {
            count = b0 + lane < p.B ? new_pages(p, b0 + lane, &first) : 0;
            incl = scan64(count, lane);
            total += __builtin_amdgcn_readlane(incl, 63);
        }
        const int each = (int)(((unsigned)total * (unsigned)p.Hkv + kSpread - 1) / kSpread);
        const int rows = max(kFew, min(kRows, each));
        const int groups = max(1, total / rows + (total % rows ? 1 : 0));
        // (every wave of a slice has a tile)
        const int slices = max(1, min((int)((unsigned)kSpread / ((unsigned)groups * (unsigned)p.Hkv)), min(16, tiles / kWaves)));
        const int lo = min(rest / slices, groups) * rows, n = max(0, min(total - lo, rows));
        if (lane == 0) { n_slots = n; n_slices = slices; }
        if (lane < kRows) slots[lane].phys = -1;
        int running = 0;
        for (int b0 = 0; b0 < p.B && running < lo + n; b0 += 64) {
            if (p.B > 64) {
                count = b0 + lane < p.B ? new_pages(p, b0 + lane, &first) : 0;
                incl = scan64(count, lane);
            }
            // lane i looks for page lo + i: the first sequence whose count of pages up to its end exceeds that
            // (all lanes take part in the exchanges: a lane that is switched off answers nothing)
            const int here = __builtin_amdgcn_readlane(incl, 63), q = lo + lane - running;
            int at = 0;
#pragma unroll 1
            for (int step = 32; step > 0; step >>= 1) {
                const int upto = __shfl(incl, at + step - 1);
                at += upto <= q ? step : 0;
            }
            const int begin = __shfl(incl - count, at), page0 = __shfl(first, at);
            if (lane < n && q >= 0 && q < here) {
                Slot s;
                s.b = b0 + at;
                s.page = page0 + (q - begin);
                // a table entry outside the pool names no page: nothing is read and no other page's id is overwritten
                const int raw = p.block_table[(long long)s.b * p.max_page + s.page];
                s.phys = (raw >= 0 && raw < p.n_blocks) ? raw : -1;
                s.valid = (int)min((long long)p.block_size, (long long)p.seq_len[s.b] - (long long)s.page * p.block_size);
                slots[lane] = s;
            }
            running += here;
        }
    }
    if (threadIdx.x < kRows) keys[threadIdx.x] = 0ull;
    for (int t = threadIdx.x; t < kRows * D / 2; t += kWaves * 64) ((uint32_t*)a_tile)[t] = 0u;      // rows beyond the list
    __syncthreads();
    const int R = n_slots, slices = n_slices;
    if (R <= 0) return;

    // ---- centroids on their way ----
    // A tile goes from memory straight into the wave's LDS as it lies, 1024 bytes a load: lanes that follow each other in
    // different rows, as the matrix instruction wants them, load at a quarter of that rate (16 bytes a clock).  The 16-byte
    // pieces of a row are permuted by the row, so that sixteen rows are read back from different banks.
    constexpr int PIECES = D / 8, ROWS = D >= 128 ? 1 : 128 / D;      // pieces of a row; rows of 256 bytes
    auto place = [](int r, int piece) { return piece ^ (r / ROWS & (PIECES - 1) & 15); };
    const int slice = rest % slices, tile0 = (int)((long long)tiles * slice / slices), tile1 = (int)((long long)tiles * (slice + 1) / slices);
    const uint8_t* const cent = (const uint8_t*)p.cent + (long long)n2 * p.C * (2 * D);      // (a head's are below 4 GiB, which the host checks)
    char* const ring = smem + wave * 2 * tile_bytes<D>();
    auto load = [&](int tile, int slot) {
        if (tile >= tile1) return;
#pragma unroll
        for (int k = 0; k < KS; ++k) {
            const int at = k * 64 + lane, r = at / PIECES, c = min(tile * 16 + r, p.C - 1);       // (past the end: the last centroid again)
            pieces_to_lds<false>(cent, (unsigned)c * (2u * D) + (unsigned)place(r, at % PIECES) * 16u, ring + slot * tile_bytes<D>() + k * 1024);
        }
    };
    int t = __builtin_amdgcn_readfirstlane(tile0 + wave);
    load(t, 0);
    load(t + kWaves, 1);

    // ---- means; few pages: a page's steps are shared by 2 to 16 waves, whose sums join in LDS ----
    int share = 1;
    while (share < kWaves && R * share * 2 <= kWaves) share *= 2;
    const int part = wave % share, apart = kWaves / share;
#pragma unroll 1
    for (int r0 = 0; r0 < R; r0 += apart) {
        const int r = r0 + wave / share;
        const bool mine = r < R && slots[min(r, kRows - 1)].phys >= 0;          // (else the row stays zero, its result is dropped)
        float sum[CH];
        if (mine) {
            page_sum<D>(p, slots[r], n2, part, share, lane, sum);
            if (kq == 0 && part != 0)
#pragma unroll
                for (int c = 0; c < CH; ++c) parts[wave][col * CH + c] = sum[c];
        }
        if (share > 1) __syncthreads();          // (share > 1: the loop runs once)
        if (mine && part == 0 && kq == 0) {
            const float inv = 1.f / (float)slots[r].valid;
#pragma unroll 1
            for (int o = 1; o < share; ++o)
#pragma unroll
                for (int c = 0; c < CH; ++c) sum[c] += parts[wave + o][col * CH + c];
            uint32_t* row = (uint32_t*)(a_tile + r * D + col * CH);
#pragma unroll
            for (int c = 0; c < CH; c += 2) {
                const float m0 = sum[c] * inv, m1 = sum[c + 1] * inv;
                row[c / 2] = BF ? __builtin_bit_cast(uint16_t, (__bf16)m0) | (uint32_t)__builtin_bit_cast(uint16_t, (__bf16)m1) << 16
                                : __builtin_bit_cast(uint16_t, (_Float16)m0) | (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)m1) << 16;
            }
        }
    }
    __syncthreads();

    // ---- pages x centroids: lane l holds centroid l % 16 of a tile and pages 4 (l / 16) .. + 3 of each sixteen ----
    uint4 a[2][KS];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int k = 0; k < KS; ++k) a[h][k] = *(const uint4*)(a_tile + (16 * h + col) * D + k * 32 + kq * 8);
    float best[2][4];
    int id[2][4];                                    // (0: of a page whose scores are all NaN)
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i) { best[h][i] = -INFINITY; id[h][i] = 0; }
    auto score = [&](int slot) {
        const int c = min(t * 16 + col, p.C - 1);
        uint4 at[KS];
#pragma unroll
        for (int k = 0; k < KS; ++k) at[k] = *(const uint4*)(ring + slot * tile_bytes<D>() + (col * PIECES + place(col, k * 4 + kq)) * 16);
        // (Both sixteens always, also where the second is empty: with a branch there the compiler left out the waits between the
        // first one's last matrix instruction and the comparison that reads it, two instructions later.)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                if constexpr (BF) s = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a[h][k]), __builtin_bit_cast(bf16x8, at[k]), s, 0, 0, 0);
                else s = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, a[h][k]), __builtin_bit_cast(half8, at[k]), s, 0, 0, 0);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const bool better = s[i] > best[h][i];   // (clusters come in ascending order: ties keep the smallest)
                best[h][i] = better ? s[i] : best[h][i];
                id[h][i] = better ? c : id[h][i];
            }
        }
    };
    for (int slot = 0; t < tile1; t += kWaves, slot ^= 1) {
        if (t + kWaves < tile1) wait_loads<KS>();                     // the next tile's may be under way
        else wait_loads<0>();
        score(slot);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");            // the tile has been read
        load(t + 2 * kWaves, slot);
    }
    // the larger score wins, of equal ones the smaller cluster: over the sixteen lanes of a row by rotating it by 1, 2, 4, 8
    join_turned<1>(best, id);
    join_turned<2>(best, id);
    join_turned<4>(best, id);
    join_turned<8>(best, id);
    if (col == 0)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                atomicMax(&keys[16 * h + 4 * kq + i], (unsigned long long)score_key(best[h][i]) << 32 | ~(uint32_t)id[h][i]);
    __syncthreads();
    const int r = threadIdx.x;
    unsigned long long key = r < R ? keys[r] : 0ull;
    if (slices > 1) {
        // the slices of these pages: slots and arrivals are zeroed before and left zeroed by the last
        const int group = rest / slices * p.Hkv + n2;
        unsigned long long* joined = (unsigned long long*)p.joined + kFew * group;
        unsigned* arrivals = (unsigned*)((unsigned long long*)p.joined + kFew * (kSpread / 2)) + group;
        if (r < R) atomicMax(joined + r, key);
        if (wave == 0) {                                 // (R <= 16: all of them are this wave's)
            __threadfence();
            if (lane == 0) last = atomicAdd(arrivals, 1u) == (unsigned)slices - 1;
            __threadfence();
        }
        __syncthreads();
        if (!last) return;
        if (r < R) key = atomicExch(joined + r, 0ull);
        if (r == 0) atomicExch(arrivals, 0u);
    }
    if (r < R) {
        const Slot s = slots[r];
        if (s.phys >= 0 && s.phys < p.kv_page_len) p.block_ids[(long long)n2 * p.kv_page_len + s.phys] = (int)~(uint32_t)key;
    }
}

template <int D>
hipError_t launch_d(const AssignParams& p, unsigned grid, hipStream_t s) {
    static int limits[2][kMaxDevices];
    const size_t lds = waves<D>() * 2 * tile_bytes<D>() + kRows * D * 2;
    const bool bf = p.qk_dtype == kBF16;
    const hipError_t e = ensure_lds_limit(bf ? (const void*)assign_int4_kernel<D, true> : (const void*)assign_int4_kernel<D, false>, limits[bf], lds);
    if (e != hipSuccess) return e;
    if (bf) hipLaunchKernelGGL((assign_int4_kernel<D, true>), dim3(grid), dim3(waves<D>() * 64), lds, s, p);
    else hipLaunchKernelGGL((assign_int4_kernel<D, false>), dim3(grid), dim3(waves<D>() * 64), lds, s, p);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_assign_int4(const AssignParams& p, hipStream_t s) {
    // groups for any number of new pages up to most: kRows of each, or fewer pages where that fills the card; slices > 1
    // only within kSpread workgroups
    const long long most = (long long)p.B * p.max_new, full = (most + kRows - 1) / kRows, spread = (kSpread + p.Hkv - 1) / p.Hkv;
    const long long groups = most == 0 ? 0 : (full > spread ? full : spread);
    if (groups <= 0 || p.Hkv <= 0) return hipSuccess;
    if (groups * p.Hkv > 0x7fffffffll) return hipErrorInvalidConfiguration;
    const unsigned grid = (unsigned)(groups * p.Hkv);
    count_launch();
    switch (p.D) {
        case 32: return launch_d<32>(p, grid, s);
        case 64: return launch_d<64>(p, grid, s);
        case 128: return launch_d<128>(p, grid, s);
        case 256: return launch_d<256>(p, grid, s);
        default: return hipErrorInvalidValue;
    }
}

}  // namespace spfa
