// gsd_chunk.hip -- attention of a chunk of new tokens per sequence over the
// paged KV cache, for a batch of sequences.
#include <algorithm>
#include <cfloat>

#include "gsd_device.h"
#include "gsd_paged.h"

using namespace gsd;

namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef float float16v __attribute__((ext_vector_type(16)));

constexpr float kLog2e = 1.44269504088896340736f;
constexpr int kWaves = 4, kThreads = 64 * kWaves;
constexpr int kRows = 32 * kWaves;   // query rows (token x head of a KV head's group) of a block's step, 32 per wave
constexpr int kPos = 64;             // positions of a tile
constexpr int kRuns = kPos / 8;      // its runs of eight positions: a page is at least that
constexpr int kCost = 256;           // what an item's start and end weigh beside its positions
constexpr int kWhole = 4;            // an item of so few tiles is not cut
constexpr int kLeastSpan = 256;      // the least a block takes
static_assert(kCost >= 2 * kPos && kLeastSpan >= kPos, "an item's tiles lie within its cost, and every span inside it has one");
constexpr int kPagesHeld = 256;      // page indices in LDS
constexpr int kMostGroups = 1024;
constexpr int kJoinRows = 8;         // rows that a block joins

// ---------------------------------------------------------------------------
//   x_tp = sm_scale q_t.K_p  (p <= the token's position, and within the window),
//   out_t = sum_p e^(x_tp - m_t) V_p / sum_p e^(x_tp - m_t)
//
// in one pass over K and V with a running maximum m and sum l.  An item is 128
// query rows of one sequence and KV head (consecutive tokens x the heads of the
// group); a wave has 32 of them as the columns of S^T = K Q^T and O^T = V^T P^T
// (32 x 32 x 16 both), over tiles of 64 positions in LDS.  A lane (column l &
// 31, half j = l >> 5) gets the scores of positions 8 b + 4 j + i (i < 4) of 32
// and feeds the same ones to the second product, so probabilities stay where
// they are; V comes transposed out of LDS (ds_read_b64_tr_b16: four positions
// of a lane's dim).
//
// fp32 rows meet the cache's 16-bit rows as sums of 16-bit parts, as in the
// decode attention (two fp16 or three bf16 parts of q and P); rows of 16 bits
// are exact as they are, and their P is rounded once to their type: half a step
// of each weight, as much as the rounding of the output.
// ---------------------------------------------------------------------------
struct Joint {   // of an item that several blocks share, at its first one's place
    int parts;   // 0: none
    int token;   // its first row in the call
    int rows;    // token x head rows
};

struct ChunkArgs {
    gsdh_paged_cache c;
    const void* q;
    void* out;
    const int *seqs, *starts;
    // of shared items: outputs [slot][slot_rows][HD], (m, l) [slot][slot_rows][2], slot =
    // 2 (group n_kv + head) + 1 for an item's first part, + 0 for a later one
    float* part;
    float* part_ml;
    Joint* joints;   // [group n_kv + head]
    int64_t q_stride, out_stride;
    int layer, n, n_tokens, group, window, groups, tokens, slot_rows;   // tokens: of an item
    float scale;
};

typedef unsigned long long u64;

struct Chunk {
    int seq, t0, m;   // rows t0 .. t0 + m - 1 of the call; m 0: nothing to do
    int base;         // position of its first token
    int items;
    bool bad;         // its rows become NaN
};

__device__ __forceinline__ Chunk chunk_of(const ChunkArgs& a, int i) {
    Chunk k{a.seqs ? a.seqs[i] : i, a.starts[i], 0, 0, 0, false};
    const int t1 = a.starts[i + 1];
    if (k.seq < 0) return k;
    if (k.t0 < 0 || t1 < k.t0 || t1 > a.n_tokens) {
        page_status(a.c, GSDH_PAGES_BAD_INDEX);
        return k;
    }
    k.m = t1 - k.t0;
    k.items = (k.m + a.tokens - 1) / a.tokens;
    if (k.seq >= a.c.n_seqs) {
        k.bad = true;
        return k;
    }
    const int len = a.c.lens[k.seq];
    k.bad = len < k.m || len > a.c.table_width * a.c.page_size;
    k.base = len - k.m;
    return k;
}
// cost of a chunk's items before item u: their positions, and kCost each
__device__ __forceinline__ u64 cost_before(const ChunkArgs& a, const Chunk& k, int u) {
    u64 s = (u64)u * kCost;
    if (k.bad) return s;
    const u64 n = (u64)u, t = (u64)a.tokens;
    s += n * (u64)k.base + t * (n * (n + 1) / 2);
    if (u == k.items) s -= t * n - (u64)k.m;   // (the last item may be shorter)
    const int64_t low = (int64_t)k.base + 1 - a.window;   // first position of the window of token 0
    if (a.window > 0 && u > 0) {
        const int64_t from = low > 0 ? 0 : -low / a.tokens + 1;   // the first item whose first position is above 0
        if (u > from) s -= (u64)((u - from) * low + (int64_t)a.tokens * ((int64_t)u * (u - 1) / 2 - from * (from - 1) / 2));
    }
    return s;
}

// sum over the lanes up to this one
__device__ __forceinline__ u64 wave_scan64(u64 v) {
#define GSD_SCAN_STEP(ctrl, rows)                                                                                     \
    v += (u64)(unsigned)__builtin_amdgcn_update_dpp(0, (int)(unsigned)v, ctrl, rows, 0xF, false) |                    \
         (u64)(unsigned)__builtin_amdgcn_update_dpp(0, (int)(unsigned)(v >> 32), ctrl, rows, 0xF, false) << 32
    GSD_SCAN_STEP(0x111, 0xF);   // row_shr 1, 2, 4, 8
    GSD_SCAN_STEP(0x112, 0xF);
    GSD_SCAN_STEP(0x114, 0xF);
    GSD_SCAN_STEP(0x118, 0xF);
    GSD_SCAN_STEP(0x142, 0xA);   // row_bcast 15, 31
    GSD_SCAN_STEP(0x143, 0xC);
#undef GSD_SCAN_STEP
    return v;
}
__device__ __forceinline__ u64 readlane64(u64 v, int lane) {
    return (u64)(unsigned)__builtin_amdgcn_readlane((int)(unsigned)v, lane) |
           (u64)(unsigned)__builtin_amdgcn_readlane((int)(unsigned)(v >> 32), lane) << 32;
}

// What a block does of an item.
struct Item {
    int seq;
    int token, rows;     // first row of the call; token x head rows
    int pos;             // position of the first token
    int first, end;      // positions that some row sees
    int t0, t1;          // tiles of 64 of them: the block's
    int split, splits;   // which of the item's parts
    bool bad;
};

// 64 lanes x 16 bytes into LDS at lds + 16 * lane, past the registers; the
// caller waits on vmcnt.  (A write of m0 needs a wait state before its use.)
__device__ __forceinline__ void lds_dma16(const void* base, unsigned off, uint32_t lds) {
    __asm__ volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(off), "s"(base) : "m0", "memory");
}
typedef __attribute__((address_space(3))) unsigned char lds_byte;

template <int CT>
__device__ __forceinline__ float16v mma(const u32x4v a, const u32x4v b, float16v c) {   // 32 x 32 x 16
    if constexpr (CT == GSDH_KV_BF16)
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf8, a), __builtin_bit_cast(bf8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c, 0, 0, 0);
}

// eight fp32 values as operands: parts whose sum they are (22 or 24 bits), or (16-bit rows) rounded once
template <int CT, int NP>
__device__ __forceinline__ void operands(const float (&x)[8], u32x4v (&w)[NP]) {
    if constexpr (NP == 1 && CT == GSDH_KV_BF16) {
        bf8 h;
#pragma unroll
        for (int e = 0; e < 8; e++) h[e] = (__bf16)x[e];
        w[0] = __builtin_bit_cast(u32x4v, h);
    } else if constexpr (NP == 1) {
        half8 h;
#pragma unroll
        for (int e = 0; e < 8; e++) h[e] = (_Float16)x[e];
        w[0] = __builtin_bit_cast(u32x4v, h);
    } else if constexpr (NP == 2) {
        // 11 bits cut off, 11 bits of the rest: two conversions of pairs and a mixed fma per value
        typedef _Float16 half2 __attribute__((ext_vector_type(2)));
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const half2 h = __builtin_bit_cast(half2, __builtin_amdgcn_cvt_pkrtz(x[2 * i], x[2 * i + 1]));
            w[0][i] = __builtin_bit_cast(uint32_t, h);
            w[1][i] = __builtin_bit_cast(uint32_t, half2{(_Float16)__builtin_fmaf((float)h[0], -1.f, x[2 * i]),
                                                         (_Float16)__builtin_fmaf((float)h[1], -1.f, x[2 * i + 1])});
        }
    } else {
        const Parts<CT, 8> p = split<CT, 8>(x);
#pragma unroll
        for (int i = 0; i < NP; i++) w[i] = p.w[i];
    }
}

template <typename T>
__device__ __forceinline__ void store4(T* p, const float (&x)[4]) {
    if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
    } else {
        typedef T t4 __attribute__((ext_vector_type(4)));
        *reinterpret_cast<t4*>(p) = t4{(T)x[0], (T)x[1], (T)x[2], (T)x[3]};
    }
}

// DT: the cache's type; RT: the rows' (float, _Float16, __bf16).  The products
// are in fp16, but bf16 for bf16 caches and rows.
template <int DT, typename RT>
struct Kinds {
    static constexpr bool kWide = sizeof(RT) == 4;
    static constexpr int CT = DT == GSDH_KV_E4M3 ? (std::is_same<RT, __bf16>::value ? GSDH_KV_BF16 : GSDH_KV_F16) : DT;
    static constexpr int NP = !kWide ? 1 : CT == GSDH_KV_BF16 ? 3 : 2;
};
// blocks per CU: registers of a wave that holds the outputs of 32 rows and their q
template <int HD, int NP>
constexpr int blocks_per_cu() {
    return HD == 256 || (HD == 128 && NP == 3) ? 1 : 2;
}

template <int HD, int DT, typename RT>
__global__ void __launch_bounds__(kThreads, (blocks_per_cu<HD, Kinds<DT, RT>::NP>())) chunk_attn_kernel(const ChunkArgs a) {
    constexpr int CT = Kinds<DT, RT>::CT, NP = Kinds<DT, RT>::NP;
    constexpr int ES = DT == GSDH_KV_E4M3 ? 1 : 2, KS = HD / 16, ND = HD / 32;
    constexpr unsigned RB = HD * 2, TILE = kPos * RB;   // a row and a tile of 16-bit values in LDS
    extern __shared__ __attribute__((aligned(1024))) unsigned char lds[];   // K, V of a tile, twice; then the pages
    int* const pages = reinterpret_cast<int*>(lds + 4 * TILE);
    const uint32_t lds_at = (uint32_t)(uintptr_t)(lds_byte*)lds;
    const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6), col = lane & 31, hi = lane >> 5;
    const int G = a.group, nkv = a.c.n_kv_heads, head = (int)(blockIdx.x % (unsigned)nkv), grp = (int)(blockIdx.x / (unsigned)nkv);
    const size_t page_b = (size_t)a.c.page_size * nkv * HD * ES;
    const unsigned row_b = (a.c.head_major ? 1u : (unsigned)nkv) * HD * ES;
    const size_t pool_at = (size_t)a.layer * a.c.n_pages * page_b + (size_t)head * (a.c.head_major ? a.c.page_size : 1) * HD * ES;
    const unsigned char* const kb = static_cast<const unsigned char*>(a.c.k) + pool_at;
    const unsigned char* const vb = static_cast<const unsigned char*>(a.c.v) + pool_at;
    const int psl = __builtin_ctz((unsigned)a.c.page_size), psm = a.c.page_size - 1;
    float kscale = 1.f, vscale = 1.f;
    if constexpr (DT == GSDH_KV_E4M3) {
        kscale = a.c.k_scale[a.layer * nkv + head];
        vscale = a.c.v_scale[a.layer * nkv + head];
    }
    // 16-byte words of a row lie in LDS at word ^ swizzle(row), so that neither the
    // K operand's reads (a word of 32 rows) nor V's (32 or 64 bytes of 4 rows) meet
    // in a bank
    auto swz_k = [](int row) { return HD == 64 ? (row >> 1) & 7 : row & 15; };
    auto swz_v = [](int row) { return HD == 64 ? (row >> 1 & 1) << 2 : (row & 3) << 2; };

    // -- one item's part ----------------------------------------------------
    auto run_item = [&](const Item& it) {
        const int tokens_hi = (it.rows - 1) / G;
        if (it.bad) {
            if (tid == 0 && head == 0) page_status(a.c, GSDH_PAGES_BAD_INDEX);
            for (int i = tid; i < it.rows * (HD / 4); i += kThreads) {
                const int r = i / (HD / 4), d = i % (HD / 4) * 4;
                const float nan = __builtin_nanf("");
                const float x[4] = {nan, nan, nan, nan};
                store4(static_cast<RT*>(a.out) + (int64_t)(it.token + r / G) * a.out_stride + ((int64_t)head * G + r % G) * HD + d, x);
            }
            return;
        }
        // the wave's rows, and what they see
        const int r0 = 32 * wid, row = min(r0 + col, it.rows - 1), tok = row / G, qh = head * G + row % G;
        const bool live = r0 < it.rows;
        const int mypos = it.pos + tok, mylow = a.window > 0 ? mypos - a.window + 1 : 0;
        const int plo = it.pos + min(r0, it.rows - 1) / G, phi = it.pos + min((r0 + 31) / G, tokens_hi);
        const int* const table = a.c.tables + (size_t)(unsigned)it.seq * a.c.table_width;
        const int page_last = (it.end - 1) >> psl;

        // q's operand
        u32x4v q[KS][NP];
        float to_log2 = 1.f;
        if (live) {
            const RT* src = static_cast<const RT*>(a.q) + (int64_t)(it.token + tok) * a.q_stride + (int64_t)qh * HD + 8 * hi;
            const float scale = a.scale * kLog2e * kscale;
            if constexpr (NP == 1 && CT == GSDH_KV_F16) {
                const uint32_t flip = scale < 0.f || (scale == 0.f && __builtin_signbit(scale)) ? 0x80008000u : 0u;
#pragma unroll
                for (int s = 0; s < KS; s++) q[s][0] = *reinterpret_cast<const u32x4v*>(src + 16 * s) ^ flip;
                to_log2 = fabsf(scale);
            } else {
                float x[KS][8], most = 0.f;
#pragma unroll
                for (int s = 0; s < KS; s++) {
                    if constexpr (sizeof(RT) == 4) {
                        const float4 u = *reinterpret_cast<const float4*>(src + 16 * s), w = *reinterpret_cast<const float4*>(src + 16 * s + 4);
                        x[s][0] = u.x; x[s][1] = u.y; x[s][2] = u.z; x[s][3] = u.w;
                        x[s][4] = w.x; x[s][5] = w.y; x[s][6] = w.z; x[s][7] = w.w;
                    } else {
                        const bf8 u = *reinterpret_cast<const bf8*>(src + 16 * s);
#pragma unroll
                        for (int e = 0; e < 8; e++) x[s][e] = (float)u[e];
                    }
#pragma unroll
                    for (int e = 0; e < 8; e++) most = fmaxf(most, fabsf(x[s][e]));
                }
                const auto other = __builtin_amdgcn_permlane32_swap(__float_as_uint(most), __float_as_uint(most), false, false);
                most = fmaxf(__uint_as_float(other[0]), __uint_as_float(other[1]));
                // by a power of two: fp16 parts keep their bits below 1024, bf16 ones stay
                // below 2^-9, so that 256 products with finite K stay below 2^127
                constexpr int kTop = CT == GSDH_KV_BF16 ? -10 : 9;
                unsigned ex = __float_as_uint(most) >> 23;
                ex = min(max(ex, 16u), 253u + (unsigned)min(kTop, 1));
                const float up = copysignf(__uint_as_float((254u + kTop - ex) << 23), scale), down = __uint_as_float((ex - kTop) << 23);
                to_log2 = fabsf(scale) * down;
#pragma unroll
                for (int s = 0; s < KS; s++) {
#pragma unroll
                    for (int e = 0; e < 8; e++) x[s][e] *= up;
                    operands<CT, NP>(x[s], q[s]);
                }
            }
            // (a scale of 0 stays above it: a masked -inf times it is -inf)
            to_log2 = fmaxf(to_log2, FLT_TRUE_MIN);
        }
        // P as 2^14 times itself: what lies below fp16's normal range stays exact longer;
        // bf16: over a power of two that is above the number of positions, so that no
        // sum of finite V passes fp32's range
        const float top_weight = CT == GSDH_KV_BF16 ? (float)(__builtin_clz((unsigned)(it.end - it.first)) - 32) : 14.f;

        float16v acc[ND];
#pragma unroll
        for (int d = 0; d < ND; d++)
#pragma unroll
            for (int r = 0; r < 16; r++) acc[d][r] = 0.f;
        // The running maximum stays unscaled.  A weight is 2^(x to_log2 + nb), nb the
        // rounded top_weight - m to_log2: one fma, whose product is exact, so all of a
        // row's weights are off by the same factor.  Where m to_log2 is beyond 2^20 that
        // factor would not stay near 1 (or the product overflow): such waves (`steep`)
        // take 2^((x - m) to_log2 + shift), which weighs the largest 2^top_weight
        // whatever fp32 rounds off the scaled scores.
        float m = -INFINITY, l = 0.f, nb = 0.f, shift = 0.f;
        bool steep = false;
        constexpr float kSteep = 1048576.f;

        // page indices of the tiles from `held` on
        int held_page = 0, held_to = it.t0;
        const int batch = max(1, (kPagesHeld - 1) * a.c.page_size / kPos);
        auto hold_pages = [&](int t) {   // all waves have read what was held
            held_to = t + batch;
            held_page = max(t * kPos, it.first) >> psl;
            const int pg = table[min(held_page + tid, page_last)];
            pages[tid] = (unsigned)pg < (unsigned)a.c.n_pages ? pg : -1;
            __syncthreads();
        };
        // the page of a run of a tile (runs that no row sees: the nearest page), per lane
        auto page_of = [&](int t, int run) {
            const int p = min(max((t * kPos + 8 * run) >> psl, held_page), page_last);
            return pages[p - held_page];
        };
        unsigned lost = 0, lost_next = 0;   // runs of a tile whose page lies outside the pool
        uint4 raw[DT == GSDH_KV_E4M3 ? 2 * HD / 64 : 1];   // e4m3: the next tile's bytes on their way to LDS
        // K and V of tile t: 16-bit rows straight into LDS, a wave two runs of each
        auto load_tile = [&](int t, int stage) {
            const int pg = page_of(t, lane & (kRuns - 1));
            lost_next = (unsigned)__ballot(pg < 0) & (unsigned)((1 << kRuns) - 1);
            if constexpr (DT != GSDH_KV_E4M3) {
                constexpr int RPI = 1024 / RB, IPR = 8 / RPI, WPR = RB / 16;   // rows of a load, loads of a run, words of a row
#pragma unroll
                for (int rr = 0; rr < 2; rr++) {
                    const int run = 2 * wid + rr, page = max(__builtin_amdgcn_readlane(pg, run), 0);
                    const size_t at = (size_t)page * page_b + (unsigned)((t * kPos + 8 * run) & psm) * row_b;
#pragma unroll
                    for (int k = 0; k < IPR; k++) {
                        const int r = k * RPI + lane / WPR, word = lane % WPR;   // of the run
                        const uint32_t to = lds_at + (unsigned)stage * 2 * TILE + (unsigned)(run * 8 + k * RPI) * RB;
                        lds_dma16(kb + at, (unsigned)r * row_b + 16u * (unsigned)(word ^ swz_k(8 * rr + r)), to);
                        lds_dma16(vb + at, (unsigned)r * row_b + 16u * (unsigned)(word ^ swz_v(8 * rr + r)), to + TILE);
                    }
                }
            } else {
                // a lane: 16 bytes of a row; a load of the wave: 1024 / HD rows, in one run
                constexpr int RPL = 1024 / HD, LPT = kPos / RPL / kWaves;   // loads of a wave and tile
#pragma unroll
                for (int k = 0; k < LPT; k++) {
                    const int r = (k * kWaves + wid) * RPL + lane / (HD / 16), run = r / 8;
                    const int page = max(__shfl(pg, run, 64), 0);
                    const size_t at = (size_t)page * page_b + (unsigned)((t * kPos + r) & psm) * row_b + 16u * (unsigned)(lane % (HD / 16));
                    raw[2 * k] = *reinterpret_cast<const uint4*>(kb + at);
                    raw[2 * k + 1] = *reinterpret_cast<const uint4*>(vb + at);
                }
            }
        };
        auto convert_tile = [&](int stage) {   // e4m3: the bytes as 16-bit values
            if constexpr (DT == GSDH_KV_E4M3) {
                constexpr int RPL = 1024 / HD, LPT = kPos / RPL / kWaves;
#pragma unroll
                for (int k = 0; k < LPT; k++) {
                    const int r = (k * kWaves + wid) * RPL + lane / (HD / 16), word = 2 * (lane % (HD / 16));
#pragma unroll
                    for (int w = 0; w < 2; w++) {
                        const uint4 b = raw[2 * k + w];
                        unsigned char* to = lds + (unsigned)stage * 2 * TILE + w * TILE + (unsigned)r * RB;
                        const int sw = w ? swz_v(r) : swz_k(r);
                        *reinterpret_cast<uint4*>(to + 16 * (word ^ sw)) =
                            make_uint4(e4m3_pair<CT, false>(b.x), e4m3_pair<CT, true>(b.x), e4m3_pair<CT, false>(b.y), e4m3_pair<CT, true>(b.y));
                        *reinterpret_cast<uint4*>(to + 16 * ((word + 1) ^ sw)) =
                            make_uint4(e4m3_pair<CT, false>(b.z), e4m3_pair<CT, true>(b.z), e4m3_pair<CT, false>(b.w), e4m3_pair<CT, true>(b.w));
                    }
                }
            }
        };

        __syncthreads();   // (the last item's tiles and pages are read)
        hold_pages(it.t0);
        load_tile(it.t0, 0);
        convert_tile(0);
        lost = lost_next;
        const unsigned k_at = (unsigned)col * RB, k_word = 16u * (unsigned)(hi ^ swz_k(col));
        const unsigned v_row = (unsigned)(4 * hi + (lane & 15) / 4);
        const unsigned v_at = v_row * RB, v_word = (16u * (unsigned)((2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) ^ swz_v((int)v_row))) + 8u * (lane & 1);
        for (int t = it.t0; t < it.t1; t++) {
            const int stage = (t - it.t0) & 1;
            // tile t is in LDS, and nobody reads tile t - 1 any more
            __asm__ volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();
            const bool more = t + 1 < it.t1;
            if (more) {
                if (t + 1 == held_to) hold_pages(t + 1);
                load_tile(t + 1, stage ^ 1);
            }
            const unsigned char* const kt = lds + (unsigned)stage * 2 * TILE;
            const unsigned char* const vt = kt + TILE;
            const int p0 = t * kPos;
            auto v_frag = [&](int s, int d) {
                typedef short s4 __attribute__((ext_vector_type(4)));
                typedef __attribute__((address_space(3))) s4 lds_s4;
                u32x4v f;
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const unsigned char* p = vt + v_at + (16 * s + 8 * h) * RB + (v_word ^ (64u * d));
                    const auto w = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(lds_byte*)p);
                    const uint2 u = __builtin_bit_cast(uint2, w);
                    f[2 * h] = u.x;
                    f[2 * h + 1] = u.y;
                }
                return f;
            };
            // What a row does not see has weight 0, but 0 times an infinity or a NaN is not
            // 0: where some row does not see all of a tile, such V are looked for, the dims of
            // the rows that do see them become NaN, and they go into the product as zeros.
            if (p0 + kPos - 1 > it.pos || (a.window > 0 && p0 <= it.end - 1 - a.window)) {
                constexpr uint32_t kToTop = CT == GSDH_KV_BF16 ? 0x00800080u : 0x04000400u;   // carries an exponent of ones into the sign
                auto odd = [&](uint32_t w) { return (((w & 0x7FFF7FFFu) + kToTop) & 0x80008000u) >> 15; };   // 1 per half
                u32x4v* const mine = reinterpret_cast<u32x4v*>(lds + (unsigned)stage * 2 * TILE + TILE) + tid;
                constexpr int kWords = TILE / 16 / kThreads;
                uint32_t any = 0;
#pragma unroll
                for (int i = 0; i < kWords; i++) {
                    const u32x4v w = mine[i * kThreads];
                    any |= odd(w[0]) | odd(w[1]) | odd(w[2]) | odd(w[3]);
                }
                if (__syncthreads_or((int)any)) {
                    constexpr uint32_t kOne = CT == GSDH_KV_BF16 ? 0x3F80u : 0x3C00u;
#pragma unroll
                    for (int d = 0; d < ND; d++) {
                        float16v count;
#pragma unroll
                        for (int r = 0; r < 16; r++) count[r] = 0.f;
#pragma unroll 1
                        for (int s = 0; s < 4; s++) {
                            u32x4v f = v_frag(s, d), see;
#pragma unroll
                            for (int w = 0; w < 4; w++) {
                                f[w] = odd(f[w]) * kOne;
                                const int p = p0 + 16 * s + 8 * (w / 2) + 4 * hi + 2 * (w % 2);
                                see[w] = (p <= mypos && p >= mylow ? kOne : 0u) | (p + 1 <= mypos && p + 1 >= mylow ? kOne << 16 : 0u);
                            }
                            count = mma<CT>(f, see, count);
                        }
#pragma unroll
                        for (int r = 0; r < 16; r++)
                            if (count[r] > 0.f) acc[d][r] = __builtin_nanf("");
                    }
                    __syncthreads();
#pragma unroll 1
                    for (int i = 0; i < kWords; i++) {
                        u32x4v w = mine[i * kThreads];
#pragma unroll
                        for (int e = 0; e < 4; e++) w[e] &= ~(odd(w[e]) * 0xFFFFu);
                        mine[i * kThreads] = w;
                    }
                    __syncthreads();
                }
            }
            const bool seen = live && p0 <= phi && (a.window <= 0 || p0 + kPos - 1 >= plo - a.window + 1);
            if (seen) {
                float16v xs[2];
#pragma unroll
                for (int n = 0; n < 2; n++)
#pragma unroll
                    for (int r = 0; r < 16; r++) xs[n][r] = 0.f;
#pragma unroll
                for (int s = 0; s < KS; s++)
#pragma unroll
                    for (int n = 0; n < 2; n++) {
                        const u32x4v f = *reinterpret_cast<const u32x4v*>(kt + k_at + 32 * n * RB + (k_word ^ (32u * s)));
#pragma unroll
                        for (int p = NP - 1; p >= 0; p--) xs[n] = mma<CT>(f, q[s][p], xs[n]);
                    }
                // what a row does not see is -inf
                const bool edge = p0 + kPos - 1 > plo || (a.window > 0 && p0 <= phi - a.window);
                if (edge || lost) {
#pragma unroll
                    for (int e = 0; e < 32; e++) {
                        const int p = p0 + 32 * (e / 16) + 8 * (e % 16 / 4) + 4 * hi + e % 4;
                        if (p > mypos || p < mylow) xs[e / 16][e % 16] = -INFINITY;
                        else if (lost >> (e / 4) & 1) xs[e / 16][e % 16] = __builtin_nanf("");
                    }
                }
                float top = -INFINITY;
#pragma unroll
                for (int e = 0; e < 32; e++) top = fmaxf(top, xs[e / 16][e % 16]);
                const auto both = __builtin_amdgcn_permlane32_swap(__float_as_uint(top), __float_as_uint(top), false, false);
                top = fmaxf(m, fmaxf(__uint_as_float(both[0]), __uint_as_float(both[1])));
                if (__any(top > m)) {
                    const bool was_steep = !(fabsf(m * to_log2) < kSteep), is_steep = !(fabsf(top * to_log2) < kSteep);
                    const float nb1 = is_steep ? 0.f : fmaf(-top, to_log2, top_weight), shift1 = is_steep ? top_weight : fmaf(top, to_log2, nb1);
                    // (nothing seen so far: there is nothing to weigh anew)
                    const float f = m == -INFINITY ? 1.f
                                  : __builtin_amdgcn_exp2f(was_steep || is_steep ? fmaf(m - top, to_log2, shift1 - shift) : nb1 - nb);
#pragma unroll
                    for (int d = 0; d < ND; d++) acc[d] *= f;
                    l *= f;
                    m = top;
                    nb = nb1;
                    shift = shift1;
                    steep = __any(is_steep && top != -INFINITY);
                }
                if (steep) {   // weights in place of scores, as exponents
                    const float base = m == -INFINITY ? 0.f : m;
#pragma unroll
                    for (int e = 0; e < 32; e++) xs[e / 16][e % 16] = fmaf(xs[e / 16][e % 16] - base, to_log2, shift);
                } else {
#pragma unroll
                    for (int e = 0; e < 32; e++) xs[e / 16][e % 16] = fmaf(xs[e / 16][e % 16], to_log2, nb);
                }
                // of 16 positions
                auto weights = [&](int s, u32x4v (&pw)[NP]) {
                    float x[8];
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        x[e] = __builtin_amdgcn_exp2f(xs[s / 2][8 * (s % 2) + e]);
                        l += x[e];
                    }
                    operands<CT, NP>(x, pw);
                };
#pragma unroll
                for (int s = 0; s < 4; s++) {
                    u32x4v pw[NP];
                    weights(s, pw);
#pragma unroll
                    for (int d = 0; d < ND; d++) {
                        const u32x4v f = v_frag(s, d);
#pragma unroll
                        for (int p = NP - 1; p >= 0; p--) acc[d] = mma<CT>(f, pw[p], acc[d]);
                    }
                }
            }
            if (more) convert_tile(stage ^ 1);
            if (lost && tid == 0 && head == 0) page_status(a.c, GSDH_PAGES_BAD_INDEX);
            lost = lost_next;
        }

        // what the weights are relative to, as an exponent of 2 (beyond fp32's range it stays
        // finite: a difference of two is a number)
        if (m != -INFINITY) m = fabsf(m * to_log2) < kSteep ? -nb : fminf(fmaxf(m * to_log2, -FLT_MAX), FLT_MAX) - top_weight;
        l = swap_add32(l, l, false);
        if (r0 + col < it.rows) {
            if (it.splits == 1) {
                const float f = vscale / l;   // (a sum of 0: every score was -inf; NaN)
                RT* o = static_cast<RT*>(a.out) + (int64_t)(it.token + tok) * a.out_stride + (int64_t)qh * HD + 4 * hi;
#pragma unroll
                for (int d = 0; d < ND; d++)
#pragma unroll
                    for (int b = 0; b < 4; b++) {
                        const float x[4] = {f * acc[d][4 * b], f * acc[d][4 * b + 1], f * acc[d][4 * b + 2], f * acc[d][4 * b + 3]};
                        store4(o + 32 * d + 8 * b, x);
                    }
            } else {
                const size_t slot = 2 * ((size_t)grp * nkv + head) + (it.split == 0);
                float* o = a.part + (slot * a.slot_rows + row) * HD + 4 * hi;
#pragma unroll
                for (int d = 0; d < ND; d++)
#pragma unroll
                    for (int b = 0; b < 4; b++)
                        *reinterpret_cast<float4*>(o + 32 * d + 8 * b) = make_float4(acc[d][4 * b], acc[d][4 * b + 1], acc[d][4 * b + 2], acc[d][4 * b + 3]);
                if (hi == 0) *reinterpret_cast<float2*>(a.part_ml + 2 * (slot * a.slot_rows + row)) = make_float2(m, l);
            }
        }
    };

    // -- which items --------------------------------------------------------
    // The chunks' costs lie end to end, and each group of blocks, one per KV
    // head, takes a span of `size` of them: all have as much to do whatever the
    // lengths are.  Every wave finds the block's span by itself.
    Chunk k{};
    u64 mine = 0;
    for (int i = lane; i < a.n; i += 64) {
        k = chunk_of(a, i);
        mine += cost_before(a, k, k.items);
    }
    const u64 total = readlane64(wave_scan64(mine), 63);
    const u64 size = max((total + a.groups - 1) / a.groups, (u64)kLeastSpan);
    const u64 lo = min((u64)grp * size, total), span_hi = min(lo + size, total);
    Joint joint{0, 0, 0};
    u64 base = 0;
    for (int c0 = 0; c0 < a.n && base < span_hi; c0 += 64) {
        if (a.n > 64) k = c0 + lane < a.n ? chunk_of(a, c0 + lane) : Chunk{};
        else if (lane >= a.n) k = Chunk{};
        const u64 cost = cost_before(a, k, k.items), incl = wave_scan64(cost), at = base + incl - cost;
        base += readlane64(incl, 63);
        u64 todo = __ballot(cost > 0 && at < span_hi && at + cost > lo);
        while (todo) {
            const int src = __builtin_ctzll(todo);
            todo &= todo - 1;
            const auto of = [&](int x) { return __builtin_amdgcn_readlane(x, src); };
            const Chunk h{of(k.seq), of(k.t0), of(k.m), of(k.base), of(k.items), of((int)k.bad) != 0};
            const u64 p0 = readlane64(at, src);
            // the first item that ends behind the span's start
            int u = 0;
            for (int below = h.items - 1; u < below;) {
                const int mid = (u + below) / 2;
                if (p0 + cost_before(a, h, mid + 1) > lo) below = mid;
                else u = mid + 1;
            }
            for (; u < h.items; u++) {
                const u64 p = p0 + cost_before(a, h, u);
                if (p >= span_hi) break;
                Item it;
                const int token = u * a.tokens, count = min(a.tokens, h.m - token);
                it.seq = h.seq;
                it.token = h.t0 + token;
                it.rows = count * G;
                it.pos = h.base + token;
                it.bad = h.bad;
                it.first = a.window > 0 ? max(0, it.pos + 1 - a.window) : 0;
                it.end = it.pos + count;
                it.t0 = it.first / kPos;
                it.t1 = (it.end + kPos - 1) / kPos;
                it.split = 0;
                it.splits = 1;
                const int tiles = it.t1 - it.t0;
                if (h.bad || tiles <= kWhole) {
                    if (p < lo) continue;   // (the group has it in whose span it starts)
                } else {
                    const auto cut = [&](u64 x) { return x <= p ? 0 : (int)min((u64)tiles, (x - p) / kPos); };
                    const int c_lo = cut(lo), c_hi = cut(span_hi);
                    if (c_lo >= c_hi) continue;
                    const u64 from = (p + kPos + size - 1) / size - 1, to = (p + (u64)tiles * kPos + size - 1) / size - 1;
                    it.t1 = it.t0 + c_hi;
                    it.t0 += c_lo;
                    it.split = (int)((u64)grp - from);
                    it.splits = (int)(to - from) + 1;
                    if (it.split == 0 && it.splits > 1) joint = Joint{it.splits, it.token, it.rows};
                }
                run_item(it);
            }
        }
    }
    if (tid == 0) a.joints[(size_t)grp * nkv + head] = joint;
}

// The parts of the items that several blocks shared: a block for kJoinRows rows
// of an item (of most places there is none).
template <int HD, typename RT>
__global__ void __launch_bounds__(256) chunk_join_kernel(const ChunkArgs a) {
    const int nkv = a.c.n_kv_heads, slices = a.slot_rows / kJoinRows;
    const int place = (int)(blockIdx.x / (unsigned)slices), r0 = (int)(blockIdx.x % (unsigned)slices) * kJoinRows;
    const Joint j = a.joints[place];
    if (r0 >= j.rows || j.parts == 0) return;
    const int head = place % nkv, grp = place / nkv, G = a.group;
    const float vscale = a.c.dtype == GSDH_KV_E4M3 ? a.c.v_scale[a.layer * nkv + head] : 1.f;
    auto slot_of = [&](int k) { return 2 * ((size_t)(grp + k) * nkv + head) + (k == 0); };
    for (int i = threadIdx.x; i < min(kJoinRows, j.rows - r0) * (HD / 4); i += 256) {
        const int row = r0 + i / (HD / 4), d = i % (HD / 4) * 4;
        float top = -INFINITY, sum = 0.f;
        for (int k = 0; k < j.parts; k++) top = fmaxf(top, a.part_ml[2 * (slot_of(k) * a.slot_rows + row)]);
        const float base = top == -INFINITY ? 0.f : top;
        float o[4] = {0.f, 0.f, 0.f, 0.f};
        // (a part whose weight is 0 is added too: a NaN or an infinity among its V shows)
#pragma unroll 4
        for (int k = 0; k < j.parts; k++) {
            const size_t at = slot_of(k) * a.slot_rows + row;
            const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + 2 * at);
            const float4 y = *reinterpret_cast<const float4*>(a.part + at * HD + d);
            const float f = __builtin_amdgcn_exp2f(ml.x - base);
            sum += f * ml.y;
            o[0] += f * y.x; o[1] += f * y.y; o[2] += f * y.z; o[3] += f * y.w;
        }
        const float f = vscale / sum;
        const float x[4] = {f * o[0], f * o[1], f * o[2], f * o[3]};
        store4(static_cast<RT*>(a.out) + (int64_t)(j.token + row / G) * a.out_stride + ((int64_t)head * G + row % G) * HD + d, x);
    }
}

// ---------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------
struct ChunkSpace {
    int groups, tokens, slot_rows;
    uint64_t joints, ml, part, bytes;   // where each begins
};
ChunkSpace chunk_space(const gsdh_paged_cache& c, int n_tokens, int n_heads, int cus) {
    ChunkSpace s;
    const int group = n_heads / c.n_kv_heads;
    s.groups = std::min(std::max(1, (cus > 0 ? cus : 1) * 2 / c.n_kv_heads), kMostGroups);
    s.tokens = kRows / group;
    s.slot_rows = (int)std::min<int64_t>(kRows, ((int64_t)n_tokens * group + kJoinRows - 1) / kJoinRows * kJoinRows);
    const uint64_t places = (uint64_t)s.groups * c.n_kv_heads, rows = 2 * places * s.slot_rows;
    s.joints = 0;
    s.ml = (places * sizeof(Joint) + 255) / 256 * 256;
    s.part = (s.ml + rows * 8 + 255) / 256 * 256;
    s.bytes = s.part + rows * c.head_dim * 4;
    return s;
}

bool chunk_shape(const gsdh_paged_cache& c, int n, int n_tokens, int n_heads) {
    return n >= 0 && n_tokens >= 0 && n_heads > 0 && n_heads % c.n_kv_heads == 0 && n_heads / c.n_kv_heads <= 16;
}

template <int HD, int DT, typename RT>
hipError_t launch_chunk(ChunkArgs a, bool alone, hipStream_t st) {
    static LdsLimit limit;
    const size_t lds = 4 * (size_t)kPos * HD * 2 + kPagesHeld * 4;
    constexpr int per_cu = blocks_per_cu<HD, Kinds<DT, RT>::NP>();
    a.groups = std::max(1, a.groups * per_cu / 2);
    const hipError_t e = raise_lds_limit(limit, reinterpret_cast<const void*>(chunk_attn_kernel<HD, DT, RT>), lds);
    if (e != hipSuccess) return e;
    const unsigned places = (unsigned)(a.groups * a.c.n_kv_heads);
    hipLaunchKernelGGL((chunk_attn_kernel<HD, DT, RT>), dim3(places), dim3(kThreads), lds, st, a);
    if (!alone) hipLaunchKernelGGL((chunk_join_kernel<HD, RT>), dim3(places * (a.slot_rows / kJoinRows)), dim3(256), 0, st, a);
    return hipGetLastError();
}

template <int HD>
hipError_t launch_chunk_type(const ChunkArgs& a, int rows, bool alone, hipStream_t st) {
    switch (a.c.dtype) {
        case GSDH_KV_F16:
            return rows == GSDH_ROWS_F32 ? launch_chunk<HD, GSDH_KV_F16, float>(a, alone, st) : launch_chunk<HD, GSDH_KV_F16, _Float16>(a, alone, st);
        case GSDH_KV_BF16:
            return rows == GSDH_ROWS_F32 ? launch_chunk<HD, GSDH_KV_BF16, float>(a, alone, st) : launch_chunk<HD, GSDH_KV_BF16, __bf16>(a, alone, st);
        default:
            return rows == GSDH_ROWS_F32 ? launch_chunk<HD, GSDH_KV_E4M3, float>(a, alone, st)
                 : rows == GSDH_ROWS_F16 ? launch_chunk<HD, GSDH_KV_E4M3, _Float16>(a, alone, st)
                                         : launch_chunk<HD, GSDH_KV_E4M3, __bf16>(a, alone, st);
    }
}

}  // namespace

extern "C" {

uint64_t gsdh_paged_chunk_attention_workspace_bytes(const gsdh_paged_cache* c, int n, int n_tokens, int n_heads) {
    if (check_paged_cache(c, "paged_chunk_attention_workspace_bytes", false) || !chunk_shape(*c, n, n_tokens, n_heads)) return 0;
    return chunk_space(*c, n_tokens, n_heads, device_cu_count()).bytes;
}

int gsdh_paged_chunk_attention(void* stream, const gsdh_paged_cache* c, int layer, const void* q, int dtype, int64_t q_stride, const int* seqs,
                               const int* starts, int n, int n_tokens, int n_heads, float sm_scale, int window, void* out, int64_t out_stride,
                               void* workspace, uint64_t workspace_bytes) {
    const char* who = "paged_chunk_attention";
    int rc = check_paged_cache(c, who, false);
    if (rc) return rc;
    if (layer < 0 || layer >= c->n_layers) return fail(-1, "%s: layer %d outside 0..%d", who, layer, c->n_layers - 1);
    if (dtype < GSDH_ROWS_F32 || dtype > GSDH_ROWS_BF16) return fail(-1, "%s: type %d", who, dtype);
    if ((dtype == GSDH_ROWS_F16 && c->dtype == GSDH_KV_BF16) || (dtype == GSDH_ROWS_BF16 && c->dtype == GSDH_KV_F16))
        return fail(-1, "%s: rows of 16 bits are of the cache's type (or over an e4m3 cache)", who);
    if (!chunk_shape(*c, n, n_tokens, n_heads))
        return fail(-1, "%s: %d chunks, %d tokens, %d heads over %d KV heads (1..16 query heads per KV head)", who, n, n_tokens, n_heads,
                    c->n_kv_heads);
    if (n > c->n_seqs && !seqs) return fail(-1, "%s: %d chunks, %d sequences", who, n, c->n_seqs);
    if (window < 0) return fail(-1, "%s: window %d", who, window);
    if (n == 0 || n_tokens == 0) return 0;
    const int64_t width = (int64_t)n_heads * c->head_dim;
    const int unit = dtype == GSDH_ROWS_F32 ? 4 : 8;
    if (!q || !out || (reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) % 16 || q_stride % unit || out_stride % unit ||
        q_stride < 0 || out_stride < width)
        return fail(-1, "%s: rows of q and out need 16-byte alignment, strides of whole 16 bytes and at least %lld for out", who,
                    (long long)width);
    if (!starts) return fail(-1, "%s: null starts", who);
    const ChunkSpace s = chunk_space(*c, n_tokens, n_heads, device_cu_count());
    rc = check_workspace(workspace, workspace_bytes, s.bytes, who);
    if (rc) return rc;
    ChunkArgs a{};
    a.c = *c;
    a.q = q; a.q_stride = q_stride; a.out = out; a.out_stride = out_stride; a.seqs = seqs; a.starts = starts;
    a.layer = layer; a.n = n; a.n_tokens = n_tokens; a.group = n_heads / c->n_kv_heads; a.window = window; a.scale = sm_scale;
    a.groups = s.groups; a.tokens = s.tokens; a.slot_rows = s.slot_rows;
    char* ws = static_cast<char*>(workspace);
    a.joints = reinterpret_cast<Joint*>(ws + s.joints);
    a.part_ml = reinterpret_cast<float*>(ws + s.ml);
    a.part = reinterpret_cast<float*>(ws + s.part);
    // where no table holds more than an item that is not cut, nothing is joined
    const bool alone = (int64_t)c->table_width * c->page_size <= kWhole * kPos;
    hipStream_t st = static_cast<hipStream_t>(stream);
    GSD_PAGED_CHK(c->head_dim == 64 ? launch_chunk_type<64>(a, dtype, alone, st)
                  : c->head_dim == 128 ? launch_chunk_type<128>(a, dtype, alone, st) : launch_chunk_type<256>(a, dtype, alone, st), who);
    return 0;
}

}  // extern "C"
