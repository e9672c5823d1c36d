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
constexpr int kWaveRows = 32;        // query rows (token x head of a KV head's group) of a wave
constexpr int kMostRows = 256;       // of a block
constexpr int kPos = 64;             // positions of a tile
constexpr int kRuns = kPos / 8;      // its runs of eight positions: a page is at least that
// What a block does is measured in quarters of the time that a position of up to 32
// rows takes, whose K and V have to come (a tile of 64 1.2 us); a position of more
// rows is that often more, by the products of its rows' parts (measured: a tile of
// 256 rows 2.1 us in 16 bits, 4.2 us in two parts), and an item's start and end, waits
// under load, are 20 us (a prompt of 4096 tokens took 307 us with 13 us in its place; 16
// chunks of 5 tokens take 68 us, with 10 us in its place 76, with 32 us 70).  All of it
// at 128 dims, 32 heads over 8, fp32 rows over fp16; other head dims and types go by the
// same costs, which only deal the work out.
constexpr int kCost = 4400;
constexpr int kWhole = 4;            // an item of so few tiles is not cut
constexpr int kLeastSpan = 2048;     // the least a block takes
__device__ __forceinline__ int cost_of_rows(bool few, int rows, int parts) {
    return few ? (rows <= 32 ? 4 : max(4, 3 * parts)) : rows <= 128 ? 6 * parts : 8 * parts;
}
static_assert(kCost >= 2 * kPos * 24 && kLeastSpan >= kPos * 24, "an item's tiles lie within its cost, and every span inside it has one");
constexpr int kPagesHeld = 256;      // page indices in LDS
constexpr int kMostGroups = 256;     // of blocks, one per KV head
constexpr int kJoinRows = 8;         // rows that a block joins at a time
// blocks that join an item: four of few rows fill the chip once (of 32 most came and went for nothing: 8 us,
// 5 with four), 256 rows are read by more (22 us with four)
constexpr int kJoinFew = 4, kJoinMany = 16;

// ---------------------------------------------------------------------------
//   x_tp = sm_scale q_t.K_p  (p <= the token's position, and within the window),
//   out_t = sum_p e^(x_tp - m_t) V_p / sum_p e^(x_tp - m_t)
//
// in one pass over K and V with a running maximum m and sum l.  An item is 128 or
// 256 query rows of one sequence and KV head (consecutive tokens x the heads of the
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
// of each weight, as much as the rounding of the output (bf16, 32768 positions: off by
// 2.2e-3 of the result, where the output's rounding alone is 1.7e-3; a second part of P
// would be half as many products again).
// ---------------------------------------------------------------------------
struct Joint {   // of an item that several blocks share, at its first one's place
    int parts;   // 0: none
    int token;   // its first row in the call
    int rows;    // token x head rows
};

// A row's weights so far: the largest score, unscaled, their sum, and what they are
// relative to: 2^(x to_log2 + nb), or (m to_log2 beyond 2^20) the largest's.  A negative
// to_log2: the factor is -2^127 times it, which fp32 does not hold.
struct __attribute__((aligned(16))) Sum {
    float m, l, nb, to_log2;
};

struct ChunkArgs {
    gsdh_paged_cache c;
    const void* q;
    void* out;
    const int *seqs, *starts;
    // of shared items: outputs [slot][slot_rows][HD], sums [slot][slot_rows], slot =
    // 2 (group n_kv + head) + 1 for an item's first part, + 0 for a later one
    float* part;
    Sum* part_sum;
    Joint* joints;   // [group n_kv + head]
    int64_t q_stride, out_stride;
    int layer, n, n_tokens, group, window, groups, slot_rows;
    int tokens, parts;   // of an item; of a row's 32-bit values
    int join_blocks;
    bool few;
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
__device__ __forceinline__ int cost_of_position(const ChunkArgs& a, int rows) { return cost_of_rows(a.few, rows, a.parts); }
// cost of a chunk's items before item u: their positions, by rows, and kCost each
__device__ __forceinline__ u64 cost_before(const ChunkArgs& a, const Chunk& k, int u) {
    u64 s = (u64)u * kCost;
    if (k.bad || u == 0) return s;
    const int64_t low = (int64_t)k.base + 1 - a.window;   // first position of the window of token 0
    const bool all = u == k.items;
    if (all) {   // the last item may be shorter
        const int token = (u - 1) * a.tokens;
        s += (u64)cost_of_position(a, (k.m - token) * a.group) * (u64)((int64_t)k.base + k.m - (a.window > 0 ? max(low + token, (int64_t)0) : 0));
        u--;
    }
    const u64 n = (u64)u, t = (u64)a.tokens;
    u64 p = n * (u64)k.base + t * (n * (n + 1) / 2);
    if (a.window > 0) {
        const int64_t from = low > 0 ? 0 : -low / a.tokens + 1;   // the first item whose first position is above 0
        if (u > from) p -= (u64)((u - from) * low + (int64_t)a.tokens * ((int64_t)u * (u - 1) / 2 - from * (from - 1) / 2));
    }
    return s + p * (u64)cost_of_position(a, a.tokens * a.group);
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

// A chunk and where its costs begin, as they wait in LDS (in registers they would stand in the products' way).
struct Placed {
    Chunk k;
    u64 at;
};

constexpr float kSteep = 1048576.f;   // exponents of 2 beyond which a rounded product would not do
__device__ __forceinline__ bool is_steep(float m, float to_log2) { return to_log2 < 0.f || !(fabsf(m * to_log2) < kSteep); }
// A difference of scores as an exponent of 2 is reach(to_log2) times it, then |to_log2| times
// that (beyond fp32's range: of scores so far apart that the lower one has no weight).
__device__ __forceinline__ float reach(float to_log2) { return to_log2 < 0.f ? 0x1p127f : 1.f; }
// What a part of a row counts beside the part with the row's largest score, top (of
// these the least nb): a difference of scores, however large they are, or of the
// rounded exponents that the weights were formed with.
__device__ __forceinline__ float part_weight(const Sum& s, float top, float nb) {
    if (s.m == -INFINITY) return 0.f;
    return __builtin_amdgcn_exp2f(is_steep(top, s.to_log2) || is_steep(s.m, s.to_log2) ? (s.m - top) * reach(s.to_log2) * fabsf(s.to_log2) : nb - s.nb);
}

// What the first wave has found for the block.
struct Plan {
    u64 size, lo, hi;   // of spans; the block's
    u64 base;           // cost before the next 64 chunks
    u64 todo;           // which of the 64 placed chunks have something in it
    int last;           // no more after these
};

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

// two fp32 values as words of operands: parts whose sum they are (23 or 24 bits), or (16-bit rows) rounded once
template <int CT, int NP>
__device__ __forceinline__ void operand_words(float x, float y, uint32_t (&w)[NP]) {
    typedef _Float16 half2 __attribute__((ext_vector_type(2)));
    typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
    if constexpr (NP == 1 && CT == GSDH_KV_BF16) {
        w[0] = __builtin_bit_cast(uint32_t, bf2{(__bf16)x, (__bf16)y});
    } else if constexpr (NP == 1) {
        w[0] = __builtin_bit_cast(uint32_t, half2{(_Float16)x, (_Float16)y});
        __asm__("" : "+v"(w[0]));   // (the compiler would convert each value once more where its rounded one is summed)
    } else if constexpr (NP == 2) {
        // 11 bits, rounded, and 11 of the rest: two conversions of pairs and a mixed fma per value
        // (of words that the compiler cannot trace: it would convert each value once more)
        w[0] = __builtin_bit_cast(uint32_t, half2{(_Float16)x, (_Float16)y});
        __asm__("" : "+v"(w[0]));
        const half2 h = __builtin_bit_cast(half2, w[0]);
        w[1] = __builtin_bit_cast(uint32_t, half2{(_Float16)__builtin_fmaf((float)h[0], -1.f, x), (_Float16)__builtin_fmaf((float)h[1], -1.f, y)});
    } else {
        // 8 + 8 + 8 bits cut off, exact
#pragma unroll
        for (int i = 0; i < 3; i++) {
            const uint32_t a = __float_as_uint(x), b = __float_as_uint(y);
            w[i] = __builtin_amdgcn_perm(b, a, 0x07060302u);
            x -= __uint_as_float(a & 0xFFFF0000u);
            y -= __uint_as_float(b & 0xFFFF0000u);
        }
    }
}

// l and two weights that are rounded to 16 bits (w): they add up as they are multiplied,
// so an average of V lies among them, and one of equal V is that V.  bf16: by a dot product
// with ones, off by 1.5 units in the last place at most, measured (2048 tokens at the end of
// 32768 positions 1089 us, 1138 with two unpacked sums); fp16's own is off downwards, 0.2 units
// on average, so a mixed fma in its place.
template <int CT>
__device__ __forceinline__ float add_rounded(float l, uint32_t w, float one) {
    if constexpr (CT == GSDH_KV_BF16) {
        typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
        return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf2, w), __builtin_bit_cast(bf2, 0x3F803F80u), l, false);
    } else {
        typedef _Float16 half2 __attribute__((ext_vector_type(2)));
        const half2 h = __builtin_bit_cast(half2, w);
        return l + __builtin_fmaf((float)h[0], one, (float)h[1]);
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

// The compiler moves nothing across: what is asked for ahead of its use stays ahead
// (left to itself it reads each operand right before its product, and waits).
__device__ __forceinline__ void keep_order() { __builtin_amdgcn_sched_barrier(0); }

template <int N>
__device__ __forceinline__ void loads_but() {   // all but the last N loads (and stores) of the wave are done
    __asm__ volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
__device__ __forceinline__ void lds_done() { __asm__ volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// DT: the cache's type; RT: the rows' (float, _Float16, __bf16).  The products
// are in fp16, but bf16 for bf16 caches and rows.
template <int DT, typename RT>
struct Kinds {
    static constexpr bool kWide = sizeof(RT) == 4;
    static constexpr int CT = DT == GSDH_KV_E4M3 ? (std::is_same<RT, __bf16>::value ? GSDH_KV_BF16 : GSDH_KV_F16) : DT;
    static constexpr int NP = !kWide ? 1 : CT == GSDH_KV_BF16 ? 3 : 2;
};
// One block per CU.  Two waves per SIMD, one multiplying while the other weighs, as
// long as the outputs and q of 32 rows fit 256 registers.  (Two blocks of four waves
// per CU read every tile twice, and the one that came first is served first: it ended
// a fifth earlier and left the CU half idle.)
template <int HD, int NP>
constexpr int waves_of() {
    return HD == 256 || (HD == 128 && NP == 3) ? 4 : 8;
}
// tiles in LDS: one is read, the others are on their way
template <int HD, int DT>
constexpr int stages_of() {
    return DT == GSDH_KV_E4M3 || HD == 256 ? 2 : 4;
}

template <int HD, int DT, int NW>
constexpr unsigned tiles_bytes() {
    const unsigned shared = 2u * stages_of<HD, DT>() * kPos * HD * 2, own = NW * 2u * (kPos / 2) * HD * 2;
    return shared > own ? shared : own;
}

// FEW: items of up to 64 rows, whose waves each take positions of their own (32 at a
// time, of the same rows as the waves `blocks` from it), and whose outputs are
// joined at the end: as many bytes under way and as much multiplied as with many
// rows, for a longer start and end.  Else items of 128 or 256 rows, which all waves
// read the same tiles for.  A call takes one way for all its chunks (is_few, with
// both ways' times); in one kernel both had registers spilled in their loops.
//
// Bound by the products and the weights between them, which take turns more than they
// overlap, for prompts: 2048 tokens of 32 heads over 8 of 128 dims at the end of 32768
// positions, bf16, 1056 to 1095 us on several cards, 1.0 PFLOP/s of products (a library's
// product of 8192^3 gets 1.2, and the clock falls under both: 1.8 GHz in this kernel), the
// matrix cores busy for 46 % of the cycles and the VALU for 44 %; 4096 tokens of fp32 rows
// over fp16 285 to 297 us, 0.94 to 0.97 PFLOP/s, two products for each.  By memory for few
// rows: 16 chunks of 5 tokens over up to 8191 positions (199 MB) 68 us, of which the stream
// is 36.
//
// Nothing is spilled in the loops at 64 dims, at 128 over fp16 and bf16 and for many 16-bit
// rows over e4m3, and with 16-bit rows of 256 over fp16 and bf16.  Elsewhere some is: at 256
// with fp32 rows 10 to 32 reloads stand beside a pass of score products, with 16-bit rows
// over e4m3 7 to 16, at 128 over e4m3 1 to 5 with fp32 rows; and beside the loads of few rows
// over e4m3 up to 26.  4096 tokens of 16 heads over 2 of 256 dims take 279 us in fp16, 425 of fp32
// rows over fp16, 647 over bf16, 609 over e4m3 (products alone: 115, 229, 344, 229).
template <int HD, int DT, typename RT, bool FEW>
__global__ void __launch_bounds__((64 * waves_of<HD, Kinds<DT, RT>::NP>()), (waves_of<HD, Kinds<DT, RT>::NP>() / 4))
chunk_attn_kernel(const ChunkArgs a) {
    constexpr int CT = Kinds<DT, RT>::CT, NP = Kinds<DT, RT>::NP;
    constexpr int ES = DT == GSDH_KV_E4M3 ? 1 : 2, KS = HD / 16, ND = HD / 32;
    constexpr int NW = waves_of<HD, NP>(), kThreads = 64 * NW, NS = stages_of<HD, DT>(), kAhead = NS - 1;
    static_assert(kThreads >= kPagesHeld && kRuns % NW == 0, "a thread per page held, whole runs per wave");
    constexpr unsigned RB = HD * 2, TILE = kPos * RB;   // a row and a tile of 16-bit values in LDS
    constexpr unsigned BUF = tiles_bytes<HD, DT, NW>();
    // K, V of NS tiles, or of half a tile for each wave, or the waves' outputs; the pages; the waves' sums
    extern __shared__ __attribute__((aligned(1024))) unsigned char lds[];
    int* const pages = reinterpret_cast<int*>(lds + BUF);
    Sum* const wave_sum = reinterpret_cast<Sum*>(lds + BUF + kPagesHeld * 4);   // [NW][32]
    Plan* const plan = reinterpret_cast<Plan*>(lds + BUF + kPagesHeld * 4 + NW * kWaveRows * sizeof(Sum) + 64 * sizeof(Placed));
    Placed* const placed = reinterpret_cast<Placed*>(lds + BUF + kPagesHeld * 4 + NW * kWaveRows * sizeof(Sum));   // [64]
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
        // the wave's rows, and what they see
        const int blocks = !FEW ? NW : it.rows <= kWaveRows ? 1 : 2;   // of 32 rows
        const int r0 = kWaveRows * (FEW ? wid & (blocks - 1) : wid), row = min(r0 + col, it.rows - 1), tok = row / G, qh = head * G + row % G;
        const bool live = r0 < it.rows;
        const int mypos = it.pos + tok, mylow = a.window > 0 ? mypos - a.window + 1 : 0;
        const int plo = it.pos + min(r0, it.rows - 1) / G, phi = it.pos + min((r0 + kWaveRows - 1) / G, tokens_hi);
        const int* const table = a.c.tables + (size_t)(unsigned)it.seq * a.c.table_width;
        const int page_last = (it.end - 1) >> psl;

        // q's operand
        u32x4v q[KS][NP];
        float to_log2 = 1.f;
        bool steep = false;
        float one = 1.f;   // (that the compiler cannot trace: a mixed fma by 1 would become conversions and a sum)
        __asm__ volatile("" : "+s"(one));
        typedef RT r8 __attribute__((ext_vector_type(8), aligned(16)));
        r8 qrow[KS];   // as it comes: asked for before the pages are, used once the first tiles are asked for
        if (live) {
            const RT* src = static_cast<const RT*>(a.q) + (int64_t)(it.token + tok) * a.q_stride + (int64_t)qh * HD + 8 * hi;
#pragma unroll
            for (int s = 0; s < KS; s++) qrow[s] = *reinterpret_cast<const r8*>(src + 16 * s);
        }
        auto form_q = [&] {
            if (!live) return;
            float scale = a.scale * kLog2e * kscale;
            int back = 127;   // to_log2 is |scale| 2^(back - 127)
            if (fabsf(scale) == INFINITY) {   // (a quarter of it need not be)
                scale = a.scale * (0.25f * kLog2e) * kscale;
                back = 129;
            }
            if constexpr (NP == 1 && CT == GSDH_KV_F16) {
                const uint32_t flip = __builtin_signbit(scale) ? 0x80008000u : 0u;
#pragma unroll
                for (int s = 0; s < KS; s++) q[s][0] = __builtin_bit_cast(u32x4v, qrow[s]) ^ flip;
            } else {
                float most = 0.f;
#pragma unroll
                for (int s = 0; s < KS; s++)
#pragma unroll
                    for (int e = 0; e < 8; e++) most = fmaxf(most, fabsf((float)qrow[s][e]));
                const auto other = __builtin_amdgcn_permlane32_swap(__float_as_uint(most), __float_as_uint(most), false, false);
                most = fmaxf(__uint_as_float(other[0]), __uint_as_float(other[1]));
                // by a power of two: fp16 parts keep their bits below 1024, bf16 ones stay
                // below 2^-9, so that 256 products with finite K stay below 2^127 (that power
                // may be subnormal, and its inverse beyond fp32's range)
                constexpr int kTop = CT == GSDH_KV_BF16 ? -10 : 9;
                const int ex = min(max((int)(__float_as_uint(most) >> 23), 16), 254), to = 254 + kTop - ex;
                back += ex - kTop - 127;
                const float up = copysignf(__uint_as_float(to > 0 ? (unsigned)to << 23 : 1u << (22 + to)), scale);
#pragma unroll
                for (int s = 0; s < KS; s++) {
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        uint32_t w[NP];
                        operand_words<CT, NP>((float)qrow[s][2 * i] * up, (float)qrow[s][2 * i + 1] * up, w);
#pragma unroll
                        for (int p = 0; p < NP; p++) q[s][p][i] = w[p];
                    }
                }
            }
            to_log2 = fabsf(scale) * __uint_as_float((unsigned)min(back, 254) << 23);
            if (back > 254) to_log2 *= __uint_as_float((unsigned)(back - 127) << 23);
            // (a scale of 0 stays above it: a masked -inf times it is -inf; one of NaN makes NaN)
            if (to_log2 < FLT_TRUE_MIN) to_log2 = FLT_TRUE_MIN;
            if (to_log2 == INFINITY && fabsf(scale) != INFINITY) to_log2 = -fminf(fabsf(scale) * __uint_as_float((unsigned)(back - 127) << 23), FLT_MAX);
            steep = __any(to_log2 < 0.f);
        };
        // P as 2^14 times itself: what lies below fp16's normal range stays exact longer;
        // bf16: over a power of two that is more than twice the number of positions, so that
        // no sum of finite V passes fp32's range (nb's rounding makes weights up to 2^(1/16) larger)
        const float top_weight = CT == GSDH_KV_BF16 ? (float)(__builtin_clz((unsigned)(it.end - it.first)) - 33) : 14.f;

        float16v acc[ND];
#pragma unroll
        for (int d = 0; d < ND; d++)
#pragma unroll
            for (int r = 0; r < 16; r++) acc[d][r] = 0.f;
        // The running maximum stays unscaled.  A weight is 2^(x to_log2 + nb), nb the
        // rounded top_weight - m to_log2: one fma, whose product is exact, so all of a
        // row's weights are off by the same factor.  Where m to_log2 is beyond 2^20 that
        // factor would not stay near 1 (or the product overflow), or to_log2 itself
        // beyond fp32's range: such waves (`steep`) take 2^((x - m) to_log2 + shift), which weighs the largest 2^top_weight
        // whatever fp32 rounds off the scaled scores.
        float m = -INFINITY, l = 0.f, nb = 0.f, shift = 0.f;
        constexpr int kDepth = 2;   // operands that are asked for ahead of their products

        // page indices of the tiles from `held` on
        int held_page = 0, held_to = it.t0;
        const int batch = max(1, (kPagesHeld - 1) * a.c.page_size / kPos);
        auto hold_pages = [&](int t) {   // all waves have read what was held
            held_to = t + batch;
            held_page = max(t * kPos, it.first) >> psl;
            const int pg = table[min(held_page + min(tid, kPagesHeld - 1), page_last)];
            if (tid < kPagesHeld) pages[tid] = (unsigned)pg < (unsigned)a.c.n_pages ? pg : -1;
            __syncthreads();
        };
        // the page of a run of eight positions (one that no row sees: the nearest page), per lane
        auto page_of = [&](int pos) { return pages[min(max(pos >> psl, held_page), page_last) - held_page]; };
        // (a lane number that the compiler cannot trace: addresses are formed for each item,
        // not kept beside the choice of items)
        int ln = lane;
        __asm__ volatile("" : "+v"(ln));
        const int v_row = 4 * (ln >> 5) + (ln & 15) / 4;
        const unsigned k_at = (unsigned)(ln & 31) * RB, k_word = 16u * (unsigned)((ln >> 5) ^ swz_k(ln & 31)), v_at = (unsigned)v_row * RB;
        const unsigned v_word = 16u * (unsigned)((2 * (ln >> 4 & 1) + ((ln & 3) >> 1)) ^ swz_v(v_row)) + 8u * (ln & 1);
        // V's operand: positions 16 s + 8 h + 4 hi + 0 .. 3 of dim 32 d + col
        auto v_frag = [&](const unsigned char* vt, int s, int d) {
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
        // What a row does not see has weight 0, but 0 times an infinity or a NaN is not 0:
        // where some row does not see all of N x 32 positions, such V are looked for (thread
        // `who` of T, which `any_of` and `meet` bring together), the dims of the rows that do
        // see them become NaN, and they go into the product as zeros.
        auto odd_values = [&](auto halves, auto threads, int p0, unsigned char* vt, int who, auto any_of, auto meet) {
            constexpr int N = decltype(halves)::value, T = decltype(threads)::value, kWords = N * 32 * RB / 16 / T;
            constexpr uint32_t kToTop = CT == GSDH_KV_BF16 ? 0x00800080u : 0x04000400u;   // carries an exponent of ones into the sign
            auto odd = [&](uint32_t w) { return (((w & 0x7FFF7FFFu) + kToTop) & 0x80008000u) >> 15; };   // 1 per half
            u32x4v* const mine = reinterpret_cast<u32x4v*>(vt) + who;
            uint32_t any = 0;
#pragma unroll
            for (int i = 0; i < kWords; i++) {
                const u32x4v w = mine[i * T];
                any |= odd(w[0]) | odd(w[1]) | odd(w[2]) | odd(w[3]);
            }
            if (!any_of(any)) return;
            constexpr uint32_t kOne = CT == GSDH_KV_BF16 ? 0x3F80u : 0x3C00u;
#pragma unroll
            for (int d = 0; d < ND; d++) {
                float16v count;
#pragma unroll
                for (int r = 0; r < 16; r++) count[r] = 0.f;
#pragma unroll 1
                for (int s = 0; s < 2 * N; s++) {
                    u32x4v f = v_frag(vt, s, d), see;
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
            meet();
#pragma unroll 1
            for (int i = 0; i < kWords; i++) {
                u32x4v w = mine[i * T];
#pragma unroll
                for (int e = 0; e < 4; e++) w[e] &= ~(odd(w[e]) * 0xFFFFu);
                mine[i * T] = w;
            }
            meet();
        };
        // The wave's rows and N x 32 positions from p0 on; gone: runs whose page lies outside the pool.
        auto step = [&](auto halves, int p0, const unsigned char* kt, const unsigned char* vt, unsigned gone, auto scored, auto weighed) {
            constexpr int N = decltype(halves)::value;
            float16v xs[N];
#pragma unroll
            for (int n = 0; n < N; n++)
#pragma unroll
                for (int r = 0; r < 16; r++) xs[n][r] = 0.f;
            auto k_frag = [&](int i) {   // K's operand: positions 32 (i % N) + col, dims 16 (i / N) + 8 hi ..
                return *reinterpret_cast<const u32x4v*>(kt + k_at + 32 * (i % N) * RB + (k_word ^ (32u * (i / N))));
            };
            u32x4v f[kDepth];
#pragma unroll
            for (int i = 0; i < kDepth; i++) f[i] = k_frag(i);
            keep_order();
#pragma unroll
            for (int i = 0; i < KS * N; i++) {
#pragma unroll
                for (int p = NP - 1; p >= 0; p--) xs[i % N] = mma<CT>(f[i % kDepth], q[i / N][p], xs[i % N]);
                if (i + kDepth < KS * N) f[i % kDepth] = k_frag(i + kDepth);
                keep_order();
            }
            scored();
            // what a row does not see is -inf
            if (gone || p0 + 32 * N - 1 > plo || (a.window > 0 && p0 <= phi - a.window)) {
#pragma unroll
                for (int e = 0; e < 16 * N; e++) {
                    const int p = p0 + 32 * (e / 16) + 8 * (e % 16 / 4) + 4 * hi + e % 4;
                    if (p > mypos || p < mylow) xs[e / 16][e % 16] = -INFINITY;
                    else if (gone >> (e / 4) & 1) xs[e / 16][e % 16] = __builtin_nanf("");
                }
            }
            float top = -INFINITY;
#pragma unroll
            for (int e = 0; e < 16 * N; e++) top = fmaxf(top, xs[e / 16][e % 16]);
            const auto both = __builtin_amdgcn_permlane32_swap(__float_as_uint(top), __float_as_uint(top), false, false);
            top = fmaxf(m, fmaxf(__uint_as_float(both[0]), __uint_as_float(both[1])));
            // (its reach is formed where it is needed, not kept beside the products)
            auto factor = [&] {
                float c = to_log2;
                __asm__ volatile("" : "+v"(c));
                return c;
            };
            if (__any(top > m)) {
                const float to_log2 = factor();
                const bool was = is_steep(m, to_log2), is = is_steep(top, to_log2);
                const float nb1 = is ? 0.f : fmaf(-top, to_log2, top_weight), shift1 = is ? top_weight : fmaf(top, to_log2, nb1);
                // (nothing seen so far: there is nothing to weigh anew)
                const float f = m == -INFINITY ? 1.f
                              : __builtin_amdgcn_exp2f(was || is ? fmaf((m - top) * reach(to_log2), fabsf(to_log2), shift1 - shift) : nb1 - nb);
#pragma unroll
                for (int d = 0; d < ND; d++) acc[d] *= f;
                l *= f;
                m = top;
                nb = nb1;
                shift = shift1;
                steep = __any(is && (top != -INFINITY || to_log2 < 0.f));
            }
            if (steep) {   // the weights' exponents in place of the scores
                const float base = m == -INFINITY ? 0.f : m, c = factor(), far = reach(c), per = fabsf(c);
#pragma unroll
                for (int e = 0; e < 16 * N; e++) xs[e / 16][e % 16] = fmaf((xs[e / 16][e % 16] - base) * far, per, shift);
            } else {
#pragma unroll
                for (int e = 0; e < 16 * N; e++) xs[e / 16][e % 16] = fmaf(xs[e / 16][e % 16], to_log2, nb);
            }
            weighed();
            // weights of a pair of positions, as words of an operand
            u32x4v pw[2][NP];
            auto weights = [&](int s, int i) {
                const float x = __builtin_amdgcn_exp2f(xs[s / 2][8 * (s % 2) + 2 * i]), y = __builtin_amdgcn_exp2f(xs[s / 2][8 * (s % 2) + 2 * i + 1]);
                uint32_t w[NP];
                if constexpr (NP > 1) l += x + y;
                operand_words<CT, NP>(x, y, w);
                if constexpr (NP == 1) l = add_rounded<CT>(l, w[0], one);
#pragma unroll
                for (int p = 0; p < NP; p++) pw[s % 2][p][i] = w[p];
            };
#pragma unroll
            for (int i = 0; i < kDepth; i++) f[i] = v_frag(vt, i / ND, i % ND);
#pragma unroll
            for (int i = 0; i < 4; i++) weights(0, i);
            keep_order();
            // the next eight positions' weights are formed between the products of these
#pragma unroll
            for (int i = 0; i < 2 * N * ND; i++) {
                const int s = i / ND, d = i % ND;
#pragma unroll
                for (int p = NP - 1; p >= 0; p--) acc[d] = mma<CT>(f[i % kDepth], pw[s % 2][p], acc[d]);
                if (i + kDepth < 2 * N * ND) f[i % kDepth] = v_frag(vt, (i + kDepth) / ND, (i + kDepth) % ND);
                if (s + 1 < 2 * N) {
#pragma unroll
                    for (int k = 4 * d / ND; k < 4 * (d + 1) / ND; k++) weights(s + 1, k);
                }
                keep_order();
            }
        };
        // some row of the block, or (the wave's own positions) of the wave, does not see all of them
        auto masked = [&](int p0, int n, int low, int high) { return p0 + n - 1 > low || (a.window > 0 && p0 <= high - a.window); };
        using One = std::integral_constant<int, 1>;
        using Two = std::integral_constant<int, 2>;

        // A row of K or V as it comes to LDS: 16-bit ones by loads past the registers, of
        // RPI rows each; e4m3 through `raw`, RPL rows per load of the wave.
        constexpr int RPI = 1024 / RB, IPR = 8 / RPI, WPR = RB / 16, RPL = 1024 / HD;
        auto load_run = [&](const unsigned char* base, int page, int p, uint32_t to, auto swz, int row_in_tile) {
            const unsigned char* const from = base + ((size_t)max(page, 0) * page_b + (unsigned)(p & psm) * row_b);
#pragma unroll
            for (int k = 0; k < IPR; k++) {
                const int r = k * RPI + ln / WPR, word = ln % WPR;   // of the run
                lds_dma16(from, (unsigned)r * row_b + 16u * (unsigned)(word ^ swz(row_in_tile + r)), to + (unsigned)(row_in_tile + k * RPI) * RB);
            }
        };
        auto load_raw = [&](const unsigned char* base, int page, int p) {   // this lane's 16 bytes of position p
            return *reinterpret_cast<const uint4*>(base + ((size_t)max(page, 0) * page_b + (unsigned)(p & psm) * row_b + 16u * (unsigned)(ln % (HD / 16))));
        };
        auto convert = [&](const uint4 b, unsigned char* tile, int r, int sw) {
            unsigned char* const to = tile + (unsigned)r * RB;
            const int word = 2 * (ln % (HD / 16));
            *reinterpret_cast<uint4*>(to + 16 * (word ^ sw)) =
                make_uint4(e4m3_pair<CT, false>(b.x), e4m3_pair<CT, true>(b.x), e4m3_pair<CT, false>(b.y), e4m3_pair<CT, true>(b.y));
            *reinterpret_cast<uint4*>(to + 16 * ((word + 1) ^ sw)) =
                make_uint4(e4m3_pair<CT, false>(b.z), e4m3_pair<CT, true>(b.z), e4m3_pair<CT, false>(b.w), e4m3_pair<CT, true>(b.w));
        };

        __syncthreads();   // (the last item's tiles and pages are read)
        if constexpr (!FEW) {
            u64 lost = 0;   // runs whose page lies outside the pool: a byte for the tile at hand and each ahead
            constexpr int LPT = 2 * kPos / RPL / NW;   // loads of a wave and tile (e4m3): K's, then V's
            uint4 raw[DT == GSDH_KV_E4M3 ? LPT : 1];
            auto load_tile = [&](int t, int stage, int ahead) {
                const int pg = page_of(t * kPos + 8 * (lane & (kRuns - 1)));
                lost |= (u64)((unsigned)__ballot(pg < 0) & (unsigned)((1 << kRuns) - 1)) << 8 * ahead;
                if constexpr (DT != GSDH_KV_E4M3) {
#pragma unroll
                    for (int rr = 0; rr < kRuns / NW; rr++) {
                        const int run = kRuns / NW * wid + rr, page = __builtin_amdgcn_readlane(pg, run);
                        const uint32_t to = lds_at + (unsigned)stage * 2 * TILE;
                        load_run(kb, page, t * kPos + 8 * run, to, swz_k, 8 * run);
                        load_run(vb, page, t * kPos + 8 * run, to + TILE, swz_v, 8 * run);
                    }
                } else {
#pragma unroll
                    for (int k = 0; k < LPT; k++) {
                        const int load = wid * LPT + k, r = load % (kPos / RPL) * RPL + ln / (HD / 16);
                        raw[k] = load_raw(load < kPos / RPL ? kb : vb, __shfl(pg, r / 8, 64), t * kPos + r);
                    }
                }
            };
            auto convert_tile = [&](int stage) {
                if constexpr (DT == GSDH_KV_E4M3) {
#pragma unroll
                    for (int k = 0; k < LPT; k++) {
                        const int load = wid * LPT + k, r = load % (kPos / RPL) * RPL + ln / (HD / 16);
                        const bool of_v = load >= kPos / RPL;
                        convert(raw[k], lds + (unsigned)stage * 2 * TILE + (of_v ? TILE : 0u), r, of_v ? swz_v(r) : swz_k(r));
                    }
                }
            };
            hold_pages(it.t0);
#pragma unroll
            for (int i = 0; i < kAhead; i++)
                if (it.t0 + i < it.t1) load_tile(it.t0 + i, i, i);
            form_q();   // (while the first tiles are on their way)
            convert_tile(0);
            for (int t = it.t0; t < it.t1; t++) {
                const int stage = (t - it.t0) % NS;
                // tile t is in LDS, the loads of those behind it may be under way; and nobody
                // reads tile t - 1 any more, whose place the tile kAhead behind t takes
                constexpr int kLoads = DT == GSDH_KV_E4M3 ? 0 : 2 * (int)TILE / 1024 / NW;   // of a wave and tile
                if (kAhead >= 3 && t + 2 < it.t1) loads_but<kAhead >= 3 ? 2 * kLoads : 0>();
                else if (kAhead >= 2 && t + 1 < it.t1) loads_but<kAhead >= 2 ? kLoads : 0>();
                else loads_but<0>();
                lds_barrier();
                const bool more = t + kAhead < it.t1;
                if (more) {
                    if (t + kAhead == held_to) hold_pages(t + kAhead);
                    load_tile(t + kAhead, (stage + kAhead) % NS, kAhead);
                }
                unsigned char* const kt = lds + (unsigned)stage * 2 * TILE;
                const int p0 = t * kPos;
                const unsigned gone = (unsigned)lost & 0xFFu;
                if (masked(p0, kPos, it.pos, it.end - 1))
                    odd_values(Two{}, std::integral_constant<int, kThreads>{}, p0, kt + TILE, tid, [](uint32_t any) { return __syncthreads_or((int)any); },
                               [] { __syncthreads(); });
                if (live && p0 <= phi && (a.window <= 0 || p0 + kPos - 1 >= plo - a.window + 1))
                    step(Two{}, p0, kt, kt + TILE, gone, [] {}, [] {});
                if (more) convert_tile((stage + kAhead) % NS);
                if (gone && tid == 0 && head == 0) page_status(a.c, GSDH_PAGES_BAD_INDEX);
                lost >>= 8;
            }
        } else {
            constexpr unsigned HALF = TILE / 2;
            constexpr int kLoads = (int)HALF / 1024, LPH = kPos / 2 / RPL;   // of K or of V
            unsigned char* const kt = lds + (unsigned)wid * 2 * HALF;
            const uint32_t to = lds_at + (unsigned)wid * 2 * HALF;
            const int every = NW / blocks;
            uint4 raw[DT == GSDH_KV_E4M3 ? 2 * LPH : 1];
            int pg = 0;   // pages of a half's runs (lane & 3)
            auto pages_for = [&](int h) { pg = page_of(32 * h + 8 * (ln & 3)); };
            auto load_half = [&](int h, const unsigned char* base, uint32_t at, auto swz) {
#pragma unroll
                for (int run = 0; run < 4; run++) load_run(base, __builtin_amdgcn_readlane(pg, run), 32 * h + 8 * run, at, swz, 8 * run);
            };
            auto load_bytes = [&](int h) {
                if constexpr (DT == GSDH_KV_E4M3) {
#pragma unroll
                    for (int k = 0; k < 2 * LPH; k++) {
                        const int r = k % LPH * RPL + ln / (HD / 16);
                        raw[k] = load_raw(k < LPH ? kb : vb, __shfl(pg, r / 8, 64), 32 * h + r);
                    }
                }
            };
            // the halves of tiles that the wave's rows see, of those whose pages are held
            int u = 0, u1 = 0;
            auto begin = [&](int tb) {
                hold_pages(tb);
                u = max(max(2 * tb, it.first / 32), a.window > 0 ? max(0, plo - a.window + 1) / 32 : 0) + wid / blocks;
                u1 = live ? min(2 * min(tb + batch, it.t1), phi / 32 + 1) : 0;
                if (u >= u1) return;
                pages_for(u);
                if constexpr (DT == GSDH_KV_E4M3) {
                    load_bytes(u);
                } else {
                    load_half(u, kb, to, swz_k);
                    load_half(u, vb, to + HALF, swz_v);
                }
            };
            begin(it.t0);
            form_q();
            for (int tb = it.t0;;) {
                for (; u < u1; u += every) {
                    const int next = u + every, p0 = 32 * u;
                    const bool more = next < u1;
                    const unsigned gone = (unsigned)__ballot(pg < 0) & 15u;
                    if (gone && lane == 0 && head == 0) page_status(a.c, GSDH_PAGES_BAD_INDEX);
                    if constexpr (DT == GSDH_KV_E4M3) {
#pragma unroll
                        for (int k = 0; k < 2 * LPH; k++) {
                            const int r = k % LPH * RPL + ln / (HD / 16);
                            convert(raw[k], kt + (k < LPH ? 0u : HALF), r, k < LPH ? swz_k(r) : swz_v(r));
                        }
                        if (more) {
                            pages_for(next);
                            load_bytes(next);
                        }
                    }
                    const bool edge = masked(p0, 32, plo, phi);
                    if (DT == GSDH_KV_E4M3) {
                    } else if (edge) {
                        loads_but<0>();   // K and V are in LDS
                    } else {
                        loads_but<kLoads>();   // K is
                    }
                    if (edge)
                        odd_values(One{}, std::integral_constant<int, 64>{}, p0, kt + HALF, lane, [](uint32_t any) { return __any(any != 0); },
                                   [] { lds_done(); });
                    step(One{}, p0, kt, kt + HALF, gone,
                         [&] {
                             if constexpr (DT != GSDH_KV_E4M3) {
                                 if (more) {   // K is read: the next one's may take its place
                                     pages_for(next);
                                     lds_done();
                                     load_half(next, kb, to, swz_k);
                                 }
                             }
                         },
                         [&] {
                             if (DT == GSDH_KV_E4M3 || edge) return;
                             if (more) loads_but<kLoads>();   // V is in LDS
                             else loads_but<0>();
                         });
                    if constexpr (DT != GSDH_KV_E4M3) {
                        if (more) {
                            lds_done();
                            load_half(next, vb, to + HALF, swz_v);
                        }
                    }
                }
                tb += batch;
                if (tb >= it.t1) break;
                __syncthreads();   // (the pages held are read)
                begin(tb);
            }
        }

        l = swap_add32(l, l, false);
        auto slot_row = [&](int r) { return (2 * ((size_t)grp * nkv + head) + (it.split == 0)) * a.slot_rows + r; };
        auto out_row = [&](int r) { return static_cast<RT*>(a.out) + (int64_t)(it.token + r / G) * a.out_stride + ((int64_t)head * G + r % G) * HD; };
        if constexpr (!FEW) {
            if (r0 + col >= it.rows) return;
            if (it.splits == 1) {
                const float f = vscale / l;   // (a sum of 0: every score was -inf; NaN)
                RT* o = out_row(row) + 4 * hi;
#pragma unroll
                for (int d = 0; d < ND; d++)
#pragma unroll
                    for (int b = 0; b < 4; b++) {
                        const float x[4] = {f * acc[d][4 * b], f * acc[d][4 * b + 1], f * acc[d][4 * b + 2], f * acc[d][4 * b + 3]};
                        store4(o + 32 * d + 8 * b, x);
                    }
            } else {
                float* o = a.part + slot_row(row) * HD + 4 * hi;
#pragma unroll
                for (int d = 0; d < ND; d++)
#pragma unroll
                    for (int b = 0; b < 4; b++)
                        *reinterpret_cast<float4*>(o + 32 * d + 8 * b) = make_float4(acc[d][4 * b], acc[d][4 * b + 1], acc[d][4 * b + 2], acc[d][4 * b + 3]);
                if (hi == 0) a.part_sum[slot_row(row)] = Sum{m, l, nb, to_log2};
            }
            return;
        }
        // the waves' outputs, 16-byte words at word ^ row, joined in LDS
        constexpr int kWords = HD / 4;
        float4* const red = reinterpret_cast<float4*>(lds);   // [NW][32][kWords]
        __syncthreads();   // (all halves are read)
#pragma unroll
        for (int d = 0; d < ND; d++)
#pragma unroll
            for (int b = 0; b < 4; b++)
                red[(wid * kWaveRows + col) * kWords + ((8 * d + 2 * b + hi) ^ (col & (kWords - 1)))] =
                    make_float4(acc[d][4 * b], acc[d][4 * b + 1], acc[d][4 * b + 2], acc[d][4 * b + 3]);
        if (hi == 0) wave_sum[wid * kWaveRows + col] = Sum{m, l, nb, to_log2};
        __syncthreads();
        if (tid < it.rows) {   // a thread per row: what each wave's outputs count
            float top = -INFINITY, low = INFINITY, sum = 0.f;
            const int w0 = tid / kWaveRows, c = tid % kWaveRows;
            const float to = wave_sum[tid].to_log2;
#pragma unroll
            for (int w = 0; w < NW; w++)
                if ((w & (blocks - 1)) == w0) top = fmaxf(top, wave_sum[w * kWaveRows + c].m);
#pragma unroll
            for (int w = 0; w < NW; w++) {
                const Sum p = wave_sum[w * kWaveRows + c];
                if ((w & (blocks - 1)) == w0 && p.m == top) low = fminf(low, p.nb);
            }
#pragma unroll
            for (int w = 0; w < NW; w++) {
                if ((w & (blocks - 1)) != w0) continue;
                const Sum p = wave_sum[w * kWaveRows + c];
                const float f = part_weight(p, top, low);
                sum += f * p.l;
                wave_sum[w * kWaveRows + c].m = f;
            }
            if (it.splits == 1) wave_sum[tid].l = vscale / sum;   // (a sum of 0: every score was -inf; NaN)
            else a.part_sum[slot_row(tid)] = Sum{top, sum, low, to};
        }
        __syncthreads();
        for (int i = tid; i < it.rows * kWords; i += kThreads) {
            const int r = i / kWords, word = i % kWords, c = r % kWaveRows;
            float o[4] = {0.f, 0.f, 0.f, 0.f};
            for (int w = r / kWaveRows; w < NW; w += blocks) {
                const float4 y = red[(w * kWaveRows + c) * kWords + (word ^ (c & (kWords - 1)))];
                const float f = wave_sum[w * kWaveRows + c].m;
                o[0] += f * y.x; o[1] += f * y.y; o[2] += f * y.z; o[3] += f * y.w;
            }
            if (it.splits == 1) {
                const float f = wave_sum[r].l, x[4] = {f * o[0], f * o[1], f * o[2], f * o[3]};
                store4(out_row(r) + 4 * word, x);
            } else {
                *reinterpret_cast<float4*>(a.part + slot_row(r) * HD + 4 * word) = make_float4(o[0], o[1], o[2], o[3]);
            }
        }
    };

    auto bad_item = [&](const Item& it) {
        if (tid == 0 && head == 0) page_status(a.c, GSDH_PAGES_BAD_INDEX);
        for (int i = tid; i < it.rows * (HD / 4); i += kThreads) {
            const int r = i / (HD / 4), d = i % (HD / 4) * 4;
            const float nan = __builtin_nanf("");
            const float x[4] = {nan, nan, nan, nan};
            store4(static_cast<RT*>(a.out) + (int64_t)(it.token + r / G) * a.out_stride + ((int64_t)head * G + r % G) * HD + d, x);
        }
    };
    // -- which items --------------------------------------------------------
    // The chunks' costs lie end to end, and each group of blocks, one per KV
    // head, takes a span of `size` of them: all have as much to do whatever the
    // lengths are.  The first wave finds the block's chunks, 64 at a time; the others
    // take them from LDS (what each read for itself could differ, and so the barriers
    // that they meet at, if somebody changed the lengths meanwhile).
    Joint joint{0, 0, 0};
    for (int c0 = 0;; c0 += 64) {
        if (wid == 0) {
            Chunk k{};
            if (c0 == 0) {
                u64 mine = 0;
                for (int i = lane; i < a.n; i += 64) {
                    k = chunk_of(a, i);
                    mine += cost_before(a, k, k.items);
                }
                const u64 total = readlane64(wave_scan64(mine), 63);
                const u64 size = max((total + a.groups - 1) / a.groups, (u64)kLeastSpan);
                const u64 lo = min((u64)grp * size, total);
                plan->size = size;
                plan->lo = lo;
                plan->hi = min(lo + size, total);
                plan->base = 0;
            }
            if (a.n > 64) k = c0 + lane < a.n ? chunk_of(a, c0 + lane) : Chunk{};   // (up to 64 are at hand)
            const u64 lo = plan->lo, end = plan->hi;
            u64 base = plan->base;
            const u64 cost = cost_before(a, k, k.items), incl = wave_scan64(cost), at = base + incl - cost;
            base += readlane64(incl, 63);
            const u64 mine = __ballot(cost > 0 && at < end && at + cost > lo);
            placed[lane] = Placed{k, at};
            plan->todo = mine;
            plan->base = base;
            plan->last = c0 + 64 >= a.n || base >= end;
        }
        __syncthreads();
        const u64 size = readlane64(plan->size, 0), lo = readlane64(plan->lo, 0), span_hi = readlane64(plan->hi, 0);
        u64 todo = readlane64(plan->todo, 0);
        const bool last = __builtin_amdgcn_readfirstlane(plan->last) != 0;
        while (todo) {
            const int src = __builtin_ctzll(todo);
            todo &= todo - 1;
            const auto of = [](int x) { return __builtin_amdgcn_readfirstlane(x); };
            const Placed c = placed[src];
            const Chunk h{of(c.k.seq), of(c.k.t0), of(c.k.m), of(c.k.base), of(c.k.items), of((int)c.k.bad) != 0};
            const u64 p0 = readlane64(c.at, 0);
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
                    const u64 tile_cost = (u64)kPos * (u64)cost_of_position(a, it.rows);
                    const auto cut = [&](u64 x) { return x <= p ? 0 : (int)min((u64)tiles, (x - p) / tile_cost); };
                    const int c_lo = cut(lo), c_hi = cut(span_hi);
                    if (c_lo >= c_hi) continue;
                    const u64 from = (p + tile_cost + size - 1) / size - 1, to = (p + (u64)tiles * tile_cost + size - 1) / size - 1;
                    it.t1 = it.t0 + c_hi;
                    it.t0 += c_lo;
                    it.split = (int)((u64)grp - from);
                    it.splits = (int)(min(to, (u64)a.groups - 1) - from) + 1;
                    if (it.split == 0 && it.splits > 1) joint = Joint{it.splits, it.token, it.rows};
                }
                if (it.bad) bad_item(it);
                else run_item(it);
            }
        }
        if (last) break;
        __syncthreads();   // (the plan is read)
    }
    if (tid == 0) a.joints[(size_t)grp * nkv + head] = joint;
}

// The parts of the items that several blocks shared: join_blocks blocks for an
// item (at most places there is none), kJoinRows rows at a time.  The weights of all
// parts first, in LDS, then their outputs, eight loads under way at a time.
template <int HD, typename RT>
__global__ void __launch_bounds__(256) chunk_join_kernel(const ChunkArgs a) {
    __shared__ float weight[kJoinRows][kMostGroups], inv[kJoinRows];
    const int nkv = a.c.n_kv_heads, place = (int)(blockIdx.x / (unsigned)a.join_blocks), head = place % nkv, grp = place / nkv, G = a.group;
    const Joint j = a.joints[place];
    if (j.parts == 0) return;
    const float vscale = a.c.dtype == GSDH_KV_E4M3 ? a.c.v_scale[a.layer * nkv + head] : 1.f;
    auto slot_of = [&](int k) { return 2 * ((size_t)(grp + k) * nkv + head) + (k == 0); };
    for (int r0 = (int)(blockIdx.x % (unsigned)a.join_blocks) * kJoinRows; r0 < j.rows; r0 += a.join_blocks * kJoinRows) {
        const int rows = min(kJoinRows, j.rows - r0);
        const int r = threadIdx.x / 32, lane = threadIdx.x % 32;   // 32 threads per row
        // (the first 32 parts' sums are loaded once)
        const Sum* const sums = a.part_sum + r0 + r;
        const int parts = r < rows ? j.parts : 0;
        auto sum_of = [&](int k) { return sums[slot_of(k) * a.slot_rows]; };
        Sum p0{-INFINITY, 0.f, INFINITY, 1.f};
        if (lane < parts) p0 = sum_of(lane);
        float top = p0.m, sum = 0.f;
        for (int k = lane + 32; k < parts; k += 32) top = fmaxf(top, sum_of(k).m);
#pragma unroll
        for (int o = 16; o >= 1; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 32));
        float low = p0.m == top ? p0.nb : INFINITY;
        for (int k = lane + 32; k < parts; k += 32) {
            const Sum p = sum_of(k);
            if (p.m == top) low = fminf(low, p.nb);
        }
#pragma unroll
        for (int o = 16; o >= 1; o >>= 1) low = fminf(low, __shfl_xor(low, o, 32));
        for (int k = lane; k < parts; k += 32) {
            const Sum p = k == lane ? p0 : sum_of(k);
            const float f = part_weight(p, top, low);
            weight[r][k] = f;
            sum += f * p.l;
        }
#pragma unroll
        for (int o = 16; o >= 1; o >>= 1) sum += __shfl_xor(sum, o, 32);
        if (r < rows && lane == 0) inv[r] = vscale / sum;
        __syncthreads();
        for (int i = threadIdx.x; i < rows * (HD / 4); i += 256) {
            const int c = i / (HD / 4), row = r0 + c, d = i % (HD / 4) * 4;
            float o[4] = {0.f, 0.f, 0.f, 0.f};
            // (a part whose weight is 0 is added too: a NaN or an infinity among its V shows)
#pragma unroll 8
            for (int k = 0; k < j.parts; k++) {
                const float4 y = *reinterpret_cast<const float4*>(a.part + (slot_of(k) * a.slot_rows + row) * HD + d);
                const float f = weight[c][k];
                o[0] += f * y.x; o[1] += f * y.y; o[2] += f * y.z; o[3] += f * y.w;
            }
            const float x[4] = {inv[c] * o[0], inv[c] * o[1], inv[c] * o[2], inv[c] * o[3]};
            store4(static_cast<RT*>(a.out) + (int64_t)(j.token + row / G) * a.out_stride + ((int64_t)head * G + row % G) * HD + d, x);
        }
        __syncthreads();   // (the weights are read)
    }
}

// ---------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------
struct ChunkSpace {
    int groups, slot_rows;
    uint64_t joints, sums, part, bytes;   // where each begins
};
ChunkSpace chunk_space(const gsdh_paged_cache& c, int n_tokens, int n_heads, int cus) {
    ChunkSpace s;
    s.groups = std::min(std::max(1, (cus > 0 ? cus : 1) / c.n_kv_heads), kMostGroups);
    s.slot_rows = (int)std::min<int64_t>(kMostRows, ((int64_t)n_tokens * (n_heads / c.n_kv_heads) + kJoinRows - 1) / kJoinRows * kJoinRows);
    const uint64_t places = (uint64_t)s.groups * c.n_kv_heads, rows = 2 * places * s.slot_rows;
    s.joints = 0;
    s.sums = (places * sizeof(Joint) + 255) / 256 * 256;
    s.part = (s.sums + rows * sizeof(Sum) + 255) / 256 * 256;
    s.bytes = s.part + rows * c.head_dim * 4;
    return s;
}

bool chunk_shape(const gsdh_paged_cache& c, int n, int n_tokens, int n_heads) {
    return n >= 0 && n <= 1 << 20 && n_tokens >= 0 && n_tokens <= 1 << 30 && n_heads > 0 && n_heads % c.n_kv_heads == 0 && n_heads / c.n_kv_heads <= 16;
}

// Chunks of at most 64 rows on average, over tables that hold 1024 positions or more
// (the lengths themselves are on the device).  Both ways' times, few and many rows'
// (us, 32 heads over 8 of 128 dims, fp32 rows over fp16): 16 chunks over 3400 positions
// of 20 rows 61 and 73, of 64 rows 72 and 78, of 96 rows 94 and 83; of 20 rows over 256
// positions 26 and 21, over 1024 35 and 37, over 4096 69 and 84.  Other head dims and
// types go by the same rule.
bool is_few(const ChunkArgs& a) {
    return (int64_t)a.n_tokens * a.group <= (int64_t)2 * kWaveRows * a.n && (int64_t)a.c.table_width * a.c.page_size >= 1024;
}

template <int HD, int DT, typename RT, bool FEW>
hipError_t launch_chunk(ChunkArgs a, bool alone, hipStream_t st) {
    static LdsLimit limit;
    constexpr int waves = waves_of<HD, Kinds<DT, RT>::NP>();
    const size_t lds = (size_t)tiles_bytes<HD, DT, waves>() + kPagesHeld * 4 + waves * kWaveRows * sizeof(Sum) + 64 * sizeof(Placed) + sizeof(Plan);
    a.few = FEW;
    a.join_blocks = FEW ? kJoinFew : kJoinMany;
    a.tokens = kWaveRows * (FEW ? 2 : waves) / a.group;
    a.parts = Kinds<DT, RT>::NP;
    const hipError_t e = raise_lds_limit(limit, reinterpret_cast<const void*>(chunk_attn_kernel<HD, DT, RT, FEW>), lds);
    if (e != hipSuccess) return e;
    const unsigned places = (unsigned)(a.groups * a.c.n_kv_heads);
    hipLaunchKernelGGL((chunk_attn_kernel<HD, DT, RT, FEW>), dim3(places), dim3(64 * waves), lds, st, a);
    if (!alone) hipLaunchKernelGGL((chunk_join_kernel<HD, RT>), dim3(places * (unsigned)a.join_blocks), dim3(256), 0, st, a);
    return hipGetLastError();
}
template <int HD, int DT, typename RT>
hipError_t launch_chunk(const ChunkArgs& a, bool alone, hipStream_t st) {
    return is_few(a) ? launch_chunk<HD, DT, RT, true>(a, alone, st) : launch_chunk<HD, DT, RT, false>(a, alone, st);
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
        return fail(-1, "%s: %d chunks (at most 2^20), %d tokens (2^30), %d heads over %d KV heads (1..16 query heads per KV head)", who, n, n_tokens, n_heads,
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
    a.groups = s.groups; a.slot_rows = s.slot_rows;
    char* ws = static_cast<char*>(workspace);
    a.joints = reinterpret_cast<Joint*>(ws + s.joints);
    a.part_sum = reinterpret_cast<Sum*>(ws + s.sums);
    a.part = reinterpret_cast<float*>(ws + s.part);
    // where no table holds more than an item that is not cut, nothing is joined
    const bool alone = (int64_t)c->table_width * c->page_size <= kWhole * kPos;
    hipStream_t st = static_cast<hipStream_t>(stream);
    GSD_PAGED_CHK(c->head_dim == 64 ? launch_chunk_type<64>(a, dtype, alone, st)
                  : c->head_dim == 128 ? launch_chunk_type<128>(a, dtype, alone, st) : launch_chunk_type<256>(a, dtype, alone, st), who);
    return 0;
}

}  // extern "C"
