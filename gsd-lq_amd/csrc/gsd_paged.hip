// gsd_paged.hip -- decode attention over a paged KV cache for a batch of
// sequences, and RoPE with the append of K/V rows to its pages.
#include <algorithm>
#include <cfloat>

#include "gsd_device.h"
#include "gsd_paged.h"

using namespace gsd;

namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));

constexpr float kLog2e = 1.44269504088896340736f;
constexpr int kWaves = 4;          // waves of a block, each on every fourth tile of its part
constexpr int kRowCost = 128;      // what a row's start and end weigh beside its positions
constexpr int kLeastSpan = 16;     // the least a block takes, in tiles
static_assert(kLeastSpan >= 2 * kWaves, "every span inside a row has tiles of it");
constexpr int kFan = 16;           // parts whose words a thread loads at once when it joins them
constexpr int kMostFans = 16;      // sets of parts of a row and KV head that are joined on their own
// positions of a tile, the step of a wave: 8 KB of K and V (4 KB of rows of 64 bytes, 16 KB of rows of 512)
constexpr int tile_positions(int row_bytes) { return row_bytes <= 128 ? 32 : 16; }
constexpr int kMaxGroup = 16;      // query heads per KV head: the columns of one matrix product

// ---------------------------------------------------------------------------
// attention of one token per sequence
//
//   x_p = sm_scale q.K_p,  out = sum_p e^(x_p - m) V_p / sum_p e^(x_p - m)
//
// in one pass over K and V with a running maximum m and sum l.  A step of a
// wave is a tile of 16 or 32 positions of one row and KV head, whose query
// heads are the columns of the matrix products: S^T = K Q^T (16 x 16 x 32) and
// O^T = V^T P^T (16 x 16 x 16, or x 32 of 32 positions).  The positions are
// dealt to the products' rows so that the probabilities come out of the first
// product in the lane that the second one needs them in: lane l (column =
// head l & 15, group j = l >> 4) gets the scores of positions 4 j + r, and 16
// + 4 j + r of a tile of 32 (r < 4), and feeds the same positions, for which
// it also loads V's rows (dims NT (l & 15) .., NT = head_dim / 16), so nothing
// goes through LDS or other lanes.  V's rows are transposed in registers by
// byte permutes.
//
// fp32 inputs meet the cache's 16-bit rows as sums of 16-bit parts: two fp16
// parts (22 bits; q scaled by a power of two so that its largest element is
// below 1024, P by 2^14, so that small parts keep their bits) or three bf16
// parts (24 bits).  e4m3 rows are exact in fp16.  bf16 rows have fp32's range,
// and the powers of two keep all sums within it: q's largest element is below
// 2^-9 (256 products of such with finite K stay below 2^127), and a row's P add up
// to less than 1.  What falls below fp32's least normal number for it, 2^-126, is
// lost: parts of weights under 2^-80 of the largest, and bits of V under 2^-70.
// ---------------------------------------------------------------------------
struct AttendArgs {
    gsdh_paged_cache c;
    const float* q;
    const int* seqs;
    float* out;
    unsigned* counters;   // arrivals of split rows [n][n_kv], counter_step words apart; zero between launches
    // of rows with several parts: outputs [slot][G][HD], (m, l) [slot][G][2], for a span
    // and KV head the part that continues a row, then the one that starts a row
    float* part;
    float* part_ml;
    int64_t q_stride, out_stride;
    int layer, n, group, window;
    int groups, few;      // of blocks, one per KV head: in the launch, and used for long rows
    unsigned counter_step;
    float scale;
};

struct Row {
    int seq;     // < 0: padding
    int first;   // positions first .. end - 1 (empty: first == end)
    int end;
    bool bad;
};

__device__ __forceinline__ Row row_of(const AttendArgs& a, int i) {
    Row r{a.seqs ? a.seqs[i] : i, 0, 0, false};
    if (r.seq < 0) return r;
    if (r.seq >= a.c.n_seqs) {
        r.bad = true;
        return r;
    }
    const int len = a.c.lens[r.seq];
    if (len < 0 || len > a.c.table_width * a.c.page_size) {
        r.bad = true;
        return r;
    }
    r.end = len;
    r.first = a.window > 0 && len > a.window ? len - a.window : 0;
    return r;
}
template <int TP>
__device__ __forceinline__ int tiles_of(const Row& r) {
    return r.end > r.first ? (r.end - 1) / TP - r.first / TP + 1 : 0;
}
// what a row weighs in the split of the work: its tiles and, for the start and
// the end of it, kRowCost more
template <int TP>
__device__ __forceinline__ unsigned cost_of(const Row& r) {
    return r.seq < 0 ? 0u : (unsigned)(tiles_of<TP>(r) + kRowCost / TP);
}

// A part of a row and KV head: what one block does at a time.
struct Unit {
    Row row;
    int i;                // row of the call
    int t0, t1;           // tiles
    int split, splits;    // which of the row's parts
    int span;             // of the row's first part
};

// Sum over the lanes up to this one, in VALU: rows of 16 by shifts, then the
// last lanes of rows 0 and 2, and of the first half, into what follows them.
__device__ __forceinline__ unsigned wave_scan(unsigned v) {
#define GSD_SCAN_STEP(ctrl, rows) v += (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, ctrl, rows, 0xF, false)
    GSD_SCAN_STEP(0x111, 0xF);   // row_shr 1, 2, 4, 8
    GSD_SCAN_STEP(0x112, 0xF);
    GSD_SCAN_STEP(0x114, 0xF);
    GSD_SCAN_STEP(0x118, 0xF);
    GSD_SCAN_STEP(0x142, 0xA);   // row_bcast 15, 31
    GSD_SCAN_STEP(0x143, 0xC);
#undef GSD_SCAN_STEP
    return v;
}

// The parts of the rows that a block does.  The rows' costs lie one after
// another, and every group of blocks (one block per KV head: what they read
// together lies together) takes a span of `size` of them, so that all blocks
// have as much to do whatever the lengths are.  A row is cut at multiples of
// kWaves tiles.  Every wave goes through the rows by itself, 64 at a time, so
// that no barrier comes before the first loads; with thousands of short rows
// that and their starts count as much as memory (8 KV heads of 128 dims in fp16:
// 4096 rows of 100 575 us, 1024 148, 128 rows of 3200, as many positions as the
// 4096, 292).
struct RowSpan {
    Row r;                     // the lane's row of the 64 at hand
    unsigned lo, hi, size;     // the block's span
    unsigned base, at, tiles;  // cost before the 64, before the lane's row; its tiles
    int k;                     // which 64
    unsigned long long mask;   // lanes whose rows have a part in the span, not yet done
};

// tiles of a row before cost x (the row starts at cost p)
__device__ __forceinline__ unsigned cut(unsigned p, unsigned tiles, unsigned x) {
    if (x <= p) return 0;
    return x - p >= tiles ? tiles : (x - p) / kWaves * kWaves;
}

template <int TP>
__device__ __forceinline__ void hold_rows(const AttendArgs& a, RowSpan& o, bool again) {
    const int i = o.k * 64 + (int)(threadIdx.x & 63);
    if (again) o.r = i < a.n ? row_of(a, i) : Row{-1, 0, 0, false};
    const unsigned c = cost_of<TP>(o.r), incl = wave_scan(c);
    o.at = o.base + incl - c;
    o.base += (unsigned)__builtin_amdgcn_readlane((int)incl, 63);
    o.tiles = (unsigned)tiles_of<TP>(o.r);
    const bool part = o.tiles ? cut(o.at, o.tiles, o.hi) > cut(o.at, o.tiles, o.lo) : c && o.at >= o.lo && o.at < o.hi;
    o.mask = __ballot(part);
}

template <int TP>
__device__ __forceinline__ RowSpan parts_of(const AttendArgs& a, unsigned group) {
    const int lane = threadIdx.x & 63;
    RowSpan o{};
    unsigned mine = 0;
    for (int i = lane; i < a.n; i += 64) {
        o.r = row_of(a, i);
        mine += cost_of<TP>(o.r);
    }
    if (lane >= a.n) o.r = Row{-1, 0, 0, false};
    const unsigned total = (unsigned)__builtin_amdgcn_readlane((int)wave_scan(mine), 63);
    // Long rows keep memory busy with a wave per SIMD, and more only wait longer
    // for it; many short rows are a chain of waits each, which a second one fills
    // (fp16 rows of 128 dims: 64 rows of up to 8191 positions 127 us with one, 134
    // with two; 128 rows of 100 23 and 19 us, 512 of 200 133 and 115).
    // e4m3 rows cost more instructions a byte, which a second wave hides, too, where
    // its span is no shorter than the chain of waits around it (48 rows of up to 4096:
    // 50 and 55 us; 16 rows of 1000: 14 us with one, 19 with two).
    const bool all = (a.n >= a.groups && total < (unsigned)a.n * ((1024 + kRowCost) / TP)) ||
                     (a.c.dtype == GSDH_KV_E4M3 && total >= 24u * (unsigned)a.groups);
    const unsigned groups = (unsigned)(all ? a.groups : a.few);
    o.size = max((total + groups - 1) / groups, (unsigned)kLeastSpan);
    // (groups * size is below 2^32: the launch's limit on positions)
    o.lo = group < groups ? min(group * o.size, total) : total;
    o.hi = min(o.lo + o.size, total);
    hold_rows<TP>(a, o, a.n > 64);   // (up to 64 rows are at hand)
    return o;
}

// The block's next part, or false.
template <int TP>
__device__ __forceinline__ bool next_part(const AttendArgs& a, RowSpan& o, Unit& u) {
    while (!o.mask) {
        o.k++;
        if (o.base >= o.hi || o.k * 64 >= a.n) return false;
        hold_rows<TP>(a, o, true);
    }
    const int src = __builtin_ctzll(o.mask);
    o.mask &= o.mask - 1;
    const auto of = [&](int x) { return __builtin_amdgcn_readlane(x, src); };
    u.i = o.k * 64 + src;
    u.row = Row{of(o.r.seq), of(o.r.first), of(o.r.end), of((int)o.r.bad) != 0};
    const unsigned p = (unsigned)of((int)o.at), tiles = (unsigned)of((int)o.tiles), t = (unsigned)(u.row.first / TP);
    u.t0 = (int)(t + cut(p, tiles, o.lo));
    u.t1 = (int)(t + cut(p, tiles, o.hi));
    // the row's first part is in the span whose end cuts off something of it, its last where the row ends
    const unsigned from = (p + min(tiles, (unsigned)kWaves) - 1) / o.size, to = tiles ? (p + tiles - 1) / o.size : from;
    u.span = (int)from;
    u.splits = (int)(to - from) + 1;
    u.split = (int)(o.lo / o.size - from);
    return true;
}

__device__ __forceinline__ float max_over_groups(float v) {   // over lanes l, l ^ 16, l ^ 32, l ^ 48
    auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
    r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float sum_over_groups(float v) { return swap_add32(swap_add16(v, v), swap_add16(v, v), false); }

template <int DT>
__device__ __forceinline__ float4v mma(const u32x4v a, const u32x4v b, float4v c) {   // 16 x 16 x 32
    if constexpr (DT == GSDH_KV_BF16)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8, a), __builtin_bit_cast(bf8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c, 0, 0, 0);
}

typedef uint32_t u32x2v __attribute__((ext_vector_type(2)));
template <int DT>
__device__ __forceinline__ float4v mma(const u32x2v a, const u32x2v b, float4v c) {   // 16 x 16 x 16
    typedef short s4 __attribute__((ext_vector_type(4)));
    typedef _Float16 half4 __attribute__((ext_vector_type(4)));
    if constexpr (DT == GSDH_KV_BF16)
        return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(s4, a), __builtin_bit_cast(s4, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(half4, a), __builtin_bit_cast(half4, b), c, 0, 0, 0);
}

// The rows of one tile as a lane holds them, and where they come from.
template <int HD, int DT>
struct Tile {
    static constexpr int ES = DT == GSDH_KV_E4M3 ? 1 : 2;
    static constexpr int KS = HD / 32;            // products over the head dims
    static constexpr int KL = HD * ES / 64;       // 16-byte loads of a lane's part of a K row
    static constexpr int NT = HD / 16;            // dims of a lane's part of a V row
    static constexpr int VW = NT * ES / 4;        // its words
    static constexpr int TP = tile_positions(HD * ES), H = TP / 16;   // positions, halves of 16 of them
    typedef uint32_t Words __attribute__((ext_vector_type(2 * H)));   // of a lane's 4 H positions, in 16 bits
    uint4 k[H][KL];
    uint32_t v[4 * H][VW];

    // dim of element 0 of product s's eight, lane group j
    static __device__ __forceinline__ int dim(int s, int j) {
        return DT == GSDH_KV_E4M3 ? (s >> 1) * 64 + j * 16 + (s & 1) * 8 : s * 32 + j * 8;
    }
    __device__ __forceinline__ void load_k(int h, const unsigned char* p) {
#pragma unroll
        for (int i = 0; i < KL; i++) k[h][i] = *reinterpret_cast<const uint4*>(p + 64 * i);
    }
    __device__ __forceinline__ void load_v(int r, const unsigned char* p) {
        if constexpr (VW == 1) {
            v[r][0] = *reinterpret_cast<const uint32_t*>(p);
        } else if constexpr (VW == 2) {
            const uint2 w = *reinterpret_cast<const uint2*>(p);
            v[r][0] = w.x;
            v[r][1] = w.y;
        } else {
#pragma unroll
            for (int i = 0; i < VW / 4; i++) {
                const uint4 w = *reinterpret_cast<const uint4*>(p + 16 * i);
                v[r][4 * i] = w.x;
                v[r][4 * i + 1] = w.y;
                v[r][4 * i + 2] = w.z;
                v[r][4 * i + 3] = w.w;
            }
        }
    }
    // K's operand of product s
    __device__ __forceinline__ uint4 kfrag(int h, int s) const {
        if constexpr (DT == GSDH_KV_E4M3) {
            const uint4 w = k[h][s >> 1];
            const uint32_t a = s & 1 ? w.z : w.x, b = s & 1 ? w.w : w.y;
            return make_uint4(e4m3x2<false>(a), e4m3x2<true>(a), e4m3x2<false>(b), e4m3x2<true>(b));
        } else {
            return k[h][s];
        }
    }
    // V's operands of the four (e4m3) or two dims of word w: the lane's positions of each dim
    __device__ __forceinline__ void vfrags(int w, Words* f) const {
#pragma unroll
        for (int p = 0; p < 2 * H; p++) {
            const uint32_t a = v[2 * p][w], b = v[2 * p + 1][w];
            if constexpr (DT == GSDH_KV_E4M3) {
                const uint32_t x = __builtin_amdgcn_perm(b, a, 0x05010400u), y = __builtin_amdgcn_perm(b, a, 0x07030602u);
                f[0][p] = e4m3x2<false>(x);
                f[1][p] = e4m3x2<true>(x);
                f[2][p] = e4m3x2<false>(y);
                f[3][p] = e4m3x2<true>(y);
            } else {
                f[0][p] = __builtin_amdgcn_perm(b, a, 0x05040100u);
                f[1][p] = __builtin_amdgcn_perm(b, a, 0x07060302u);
            }
        }
    }
};

// Parts that one block joins at a time: two rounds of loads where the outputs
// are a word per thread, one where they are several (a second level of joins
// costs 2.5 us, a round 0.7).
__device__ __forceinline__ int fan_of(int outputs) { return outputs <= 512 ? 2 * kFan : kFan; }

// Joins `count` (up to 2 kFan) parts of a row, first, first + step ..: into
// the row's output, or into the place of the first.  The loads of kFan words
// are in flight before the weights are formed (one after another the loads of
// 64 parts took 12 us).
template <int HD>
__device__ __forceinline__ void join_parts(const AttendArgs& a, const Unit& u, int head, int first, int step, int count, bool whole,
                                           float* red, float* out, float vscale) {
    const int tid = threadIdx.x, G = a.group;
    constexpr int kThreads = 64 * kWaves;
    static_assert(kThreads >= kFan * kMaxGroup && kFan == 16, "a thread per two parts and head, a row of lanes per head");
    auto slot_of = [&](int k) {
        const int w = first + min(k, count - 1) * step;
        return (unsigned)(((u.span + w) * a.c.n_kv_heads + head) * 2 + (w == 0));
    };
    float *weight = red, *inv = red + 2 * kFan * kMaxGroup;   // [2 kFan][G], 0 behind the last part; [G]
    const int words = G * HD / 2, eg = tid / kFan, ew = tid % kFan;
    float2 e[2];
#pragma unroll
    for (int j = 0; j < 2; j++) {
        const int k = ew + j * kFan;
        e[j] = eg < G && k < count ? get2(a.part_ml + (slot_of(k) * G + eg) * 2) : make_float2(-INFINITY, 0.f);
    }
    for (int i = tid; i == tid || i < words; i += kThreads) {   // (all threads meet at the first's barrier)
        const int word = min(i, words - 1), g = word / (HD / 2);
        float2 o = make_float2(0.f, 0.f);
#pragma unroll 1
        for (int k0 = 0; k0 < count; k0 += kFan) {
            float2 y[kFan];
#pragma unroll
            for (int k = 0; k < kFan; k++) y[k] = get2(a.part + slot_of(k0 + k) * (unsigned)(G * HD) + 2 * word);
            if (i == tid && k0 == 0) {
                const float top = row16_max(fmaxf(e[0].x, e[1].x)), base = top == -INFINITY ? 0.f : top;
                float f[2], part = 0.f;
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    f[j] = ew + j * kFan < count ? __builtin_amdgcn_exp2f(e[j].x - base) : 0.f;
                    part += f[j] * e[j].y;
                }
                const float sum = row16_sum(part);
                if (eg < G) {
                    weight[ew * G + eg] = f[0];
                    weight[(ew + kFan) * G + eg] = f[1];
                    if (ew == 0) {
                        inv[eg] = vscale / sum;   // (sum 0: every score was -inf; NaN)
                        if (!whole) put2(a.part_ml + (slot_of(0) * G + eg) * 2, top, sum);
                    }
                }
                __syncthreads();
            }
#pragma unroll
            for (int k = 0; k < kFan; k++) {
                // (behind the last part: 0 times its words again.  A part whose weight is 0
                // is added too, a NaN or an infinity among its V shows wherever it lies.)
                const float f = weight[(k0 + k) * G + g];
                o.x += f * y[k].x;
                o.y += f * y[k].y;
            }
        }
        if (i >= words) break;
        if (whole) *reinterpret_cast<float2*>(out + 2 * word) = make_float2(inv[g] * o.x, inv[g] * o.y);
        else put2(a.part + slot_of(0) * (unsigned)(G * HD) + 2 * word, o.x, o.y);
    }
}

// What a wave reads of a unit.
struct Span {
    int first, end;        // positions the mask keeps
    int mine, final_, t1;  // the wave's first and last tile (every kWaves-th); none: mine >= t1
    const unsigned char *kb, *vb;
    const int* table;
};

// One block per KV head and span, as many as fit the chip at once, so that all
// start together, read at the same rate and end together: units handed out
// one by one left the last 50 us of a batch of 64 (147 us) to a few of them.
//
// While a part streams, the next one's q rows and page indices come in, and
// its first tile's rows are on their way before this one's waves are joined:
// with memory saturated each of these waits takes 3 to 5 us.
//
// Bound by memory: 64 rows of up to 8191 positions (8 KV heads of 128 dims in
// fp16, 668 MB) 126 us, 5.3 TB/s; one row of 131072 in bf16 (537 MB) 99 us; 48
// rows of e4m3 in a window of 4096 (205 MB) 50 us; loads alone in this order
// reach 5.7 TB/s.  One row of 8192 (34 MB) takes 14.5 us, of which the stream
// is 4 and the rest the waits before it and the join behind it.
template <int HD, int DT>
__global__ void __launch_bounds__(64 * kWaves, HD == 256 ? 1 : 2) paged_attn_kernel(const AttendArgs a) {
    typedef Tile<HD, DT> T;
    constexpr int TP = T::TP, H = T::H, NP = Parts<DT, 4 * H>::N, NT = T::NT, DPW = 4 / T::ES;   // dims of a V word
    constexpr int kThreads = 64 * kWaves;
    constexpr int QN = (kMaxGroup * HD / 4 + kThreads - 1) / kThreads;   // 16-byte words of q a thread brings in
    extern __shared__ float lds[];
    __shared__ int last;
    const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6, col = lane & 15, grp = lane >> 4;
    const int G = a.group, nkv = a.c.n_kv_heads, head = (int)(blockIdx.x % (unsigned)nkv);
    float *qbuf = lds, *red = lds + G * HD;   // q [G][HD]; outputs [kWaves][G][HD], (m, l) [kWaves][16][2]

    const size_t page_b = (size_t)a.c.page_size * nkv * HD * T::ES;
    const unsigned row_b = (a.c.head_major ? 1u : (unsigned)nkv) * HD * T::ES;
    const size_t layer_b = (size_t)a.layer * a.c.n_pages * page_b;
    const int psl = __builtin_ctz((unsigned)a.c.page_size), psm = a.c.page_size - 1;
    auto span_of = [&](const Unit& u) {
        Span s;
        s.first = u.row.first;
        s.end = u.row.end;
        s.t1 = u.t1;
        s.mine = __builtin_amdgcn_readfirstlane(u.t0 + wid);
        s.final_ = s.mine < s.t1 ? s.mine + (s.t1 - 1 - s.mine) / kWaves * kWaves : s.mine;
        const size_t off = layer_b + (size_t)head * (a.c.head_major ? a.c.page_size : 1) * HD * T::ES;
        s.kb = static_cast<const unsigned char*>(a.c.k) + off;
        s.vb = static_cast<const unsigned char*>(a.c.v) + off;
        s.table = a.c.tables + (size_t)(unsigned)max(u.row.seq, 0) * a.c.table_width;
        return s;
    };
    // The pages of a tile's runs of eight positions (a page is at least that)
    // come from a lane each, kAhead of the wave's tiles per load and a load
    // ahead: a lookup of its own for each tile would come back behind the rows
    // in flight.
    constexpr int kRuns = 2 * H, kAhead = 64 / kRuns;
    auto run_at = [&](int t) { return (t + lane / kRuns * kWaves) * TP + 8 * (lane % kRuns); };   // of tiles t, t + kWaves ..
    auto pages_from = [&](const Span& s, int t) {
        return s.table[min(max(run_at(t), s.first), s.end - 1) >> psl];   // (a run without a position: the nearest page)
    };
    // byte offsets of the runs' first rows; a page outside the pool is not read
    auto offsets = [&](int t, int pg, bool& lost) {
        const bool bad = (unsigned)pg >= (unsigned)a.c.n_pages;
        lost |= bad;
        return (size_t)(bad ? 0u : (unsigned)pg) * page_b + (unsigned)(run_at(t) & psm) * row_b;
    };
    struct Runs {
        size_t at[kRuns];
    };
    auto runs_of = [&](size_t held, int k) {   // of the k-th tile held
        Runs p;
#pragma unroll
        for (int j = 0; j < kRuns; j++)
            p.at[j] = (size_t)(unsigned)__builtin_amdgcn_readlane((int)(unsigned)held, kRuns * k + j) |
                      (size_t)(unsigned)__builtin_amdgcn_readlane((int)(unsigned)(held >> 32), kRuns * k + j) << 32;
        return p;
    };
    // Whole runs are loaded, also the rows of the first and last tile that the
    // mask drops (they lie in pages of the pool; V's are cleared before use).
    const unsigned k_at = (col & 7) * row_b + 16 * grp, v_at = (4 * grp & 7) * row_b + NT * T::ES * col;
    T tile;
    auto load_k = [&](const Span& s, const Runs& runs) {
#pragma unroll
        for (int h = 0; h < H; h++) tile.load_k(h, s.kb + ((col < 8 ? runs.at[2 * h] : runs.at[2 * h + 1]) + k_at));
    };
    auto load_v = [&](const Span& s, const Runs& runs) {
#pragma unroll
        for (int h = 0; h < H; h++) {
            const unsigned char* p = s.vb + ((grp < 2 ? runs.at[2 * h] : runs.at[2 * h + 1]) + v_at);
#pragma unroll
            for (int r = 0; r < 4; r++) tile.load_v(4 * h + r, p + r * row_b);
        }
    };

    RowSpan parts = parts_of<TP>(a, blockIdx.x / (unsigned)nkv);
    float kscale = 1.f, vscale = 1.f;
    if constexpr (DT == GSDH_KV_E4M3) {
        kscale = a.c.k_scale[a.layer * nkv + head];
        vscale = a.c.v_scale[a.layer * nkv + head];
    }
    Unit u{};
    Span s{};
    size_t held = 0;
    bool have = false, lost = false;
    for (;;) {
        // the next part: its q and pages
        Unit un{};
        Span sn{};
        float4v qn[QN];
#pragma unroll
        for (int j = 0; j < QN; j++) qn[j] = float4v{0.f, 0.f, 0.f, 0.f};
        size_t heldn = 0;
        int pagesn = 0;
        bool lostn = false;
        const bool more = next_part<TP>(a, parts, un);
        if (more) {
            sn = span_of(un);
            lostn = un.row.bad;
            if (sn.mine < sn.t1) pagesn = pages_from(sn, sn.mine);
            const float4v* qp = reinterpret_cast<const float4v*>(a.q + (int64_t)un.i * a.q_stride + (int64_t)head * G * HD);
#pragma unroll
            for (int j = 0; j < QN; j++)
                qn[j] = qp[min(tid + j * kThreads, G * HD / 4 - 1)];
        }

        float4v acc[NT];
        // m: the largest unscaled score; times reach and to_log2: as an exponent of 2 (reach
        // 1, but 2^127 where the factor is beyond fp32's range)
        float m = -INFINITY, l = 0.f, to_log2 = 1.f, reach = 1.f;
#pragma unroll
        for (int t = 0; t < NT; t++) acc[t] = float4v{0.f, 0.f, 0.f, 0.f};
        if (have && s.mine < s.t1) {
            // q's operand: head `col`, zeros beyond the group
            Parts<DT, 8> q[T::KS];
            {
                float x[T::KS][8], most = 0.f;
                const float* qp = qbuf + (col < G ? col : 0) * HD;
#pragma unroll
                for (int i = 0; i < T::KS; i++) {
                    const float4 lo = *reinterpret_cast<const float4*>(qp + T::dim(i, grp));
                    const float4 hi = *reinterpret_cast<const float4*>(qp + T::dim(i, grp) + 4);
                    const float w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        x[i][e] = col < G ? w[e] : 0.f;
                        most = fmaxf(most, fabsf(x[i][e]));
                    }
                }
                // 2^(kTop - exponent of the largest): it may be subnormal, and its inverse
                // times the scale beyond fp32's range
                constexpr int kTop = DT == GSDH_KV_BF16 ? -10 : 9;
                const int ex = min(max((int)(__float_as_uint(max_over_groups(most)) >> 23), 16), 254), to = 254 + kTop - ex;
                // (a negative scale is in q's sign; one of 0 stays above it, so that a
                // masked -inf times it stays -inf, and no farther than 2^-149: a bf16
                // row's unscaled scores reach 2^127)
                float scale = a.scale * kLog2e * kscale;
                int back = ex - kTop;   // to_log2 is |scale| 2^(back - 127)
                if (fabsf(scale) == INFINITY) {   // (a quarter of it need not be)
                    scale = a.scale * (0.25f * kLog2e) * kscale;
                    back += 2;
                }
                const float up = copysignf(__uint_as_float(to > 0 ? (unsigned)to << 23 : 1u << (22 + to)), scale);
                to_log2 = fabsf(scale) * __uint_as_float((unsigned)min(back, 254) << 23);
                if (back > 254) to_log2 *= __uint_as_float((unsigned)(back - 127) << 23);
                if (to_log2 == INFINITY && fabsf(scale) != INFINITY) {
                    to_log2 = fminf(fabsf(scale) * __uint_as_float((unsigned)(back - 127) << 23), FLT_MAX);
                    reach = 0x1p127f;
                }
                if (to_log2 < FLT_TRUE_MIN) to_log2 = FLT_TRUE_MIN;
#pragma unroll
                for (int i = 0; i < T::KS; i++) {
#pragma unroll
                    for (int e = 0; e < 8; e++) x[i][e] *= up;
                    q[i] = split<DT, 8>(x[i]);
                }
            }
            // The next tile's K is loaded once this one's scores are formed, its V
            // once the output is: half a tile or more is always in flight.  The
            // loads are unconditional (after the wave's last tile that one again,
            // from the cache), so that a wait never has to drain those behind a
            // branch.
            // P as 2^14 times itself: the parts below fp16's normal range stay exact; bf16:
            // as P over a power of two that is above the row's number of positions
            const float weight_of_top = DT == GSDH_KV_BF16 ? (float)(__builtin_clz((unsigned)(s.end - s.first)) - 32) : 14.f;
            const bool far = __any(reach != 1.f);
            int ahead = pages_from(s, s.mine + kAhead * kWaves), place = 0;   // the next kAhead tiles' pages; the next tile among the held
            for (int t = s.mine; t < s.t1; t += kWaves) {
                float4v xs[H];
#pragma unroll
                for (int h = 0; h < H; h++) xs[h] = float4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int i = 0; i < T::KS; i++)
#pragma unroll
                    for (int h = 0; h < H; h++) {
                        const u32x4v f = __builtin_bit_cast(u32x4v, tile.kfrag(h, i));
#pragma unroll
                        for (int p = NP - 1; p >= 0; p--) xs[h] = mma<DT>(f, q[i].w[p], xs[h]);
                    }
                const int to = min(t + kWaves, s.final_);
                place += to != t;
                if (place == kAhead) {
                    held = offsets(to, ahead, lost);
                    ahead = pages_from(s, to + kAhead * kWaves);
                    place = 0;
                }
                const Runs runs = runs_of(held, place);
                load_k(s, runs);
                // Scores and their maximum stay unscaled: what the exponential gets is the
                // difference, so the largest has weight 1 whatever fp32 rounds off the
                // scaled scores.  Rows that the mask drops are -inf.
                float x[4 * H], top = -INFINITY;
#pragma unroll
                for (int e = 0; e < 4 * H; e++) x[e] = xs[e / 4][e % 4];
                const bool edge = t * TP < s.first || (t + 1) * TP > s.end;
                if (edge) {
#pragma unroll
                    for (int e = 0; e < 4 * H; e++) {
                        const int p = t * TP + 16 * (e / 4) + 4 * grp + e % 4;
                        if (p < s.first || p >= s.end) x[e] = -INFINITY;
                    }
                }
#pragma unroll
                for (int e = 0; e < 4 * H; e++) top = fmaxf(top, x[e]);
                top = fmaxf(m, max_over_groups(top));
                if (__any(top > m)) {
                    const float f = top == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((m - top) * reach * to_log2);
#pragma unroll
                    for (int n = 0; n < NT; n++) acc[n] *= f;
                    l *= f;
                    m = top;
                }
                const float base = m == -INFINITY ? 0.f : m;
#pragma unroll
                for (int e = 0; e < 4 * H; e++) x[e] -= base;
                if (far) {
#pragma unroll
                    for (int e = 0; e < 4 * H; e++) x[e] *= reach;
                }
#pragma unroll
                for (int e = 0; e < 4 * H; e++) {
                    x[e] = __builtin_amdgcn_exp2f(fmaf(x[e], to_log2, weight_of_top));
                    l += x[e];
                }
                const Parts<DT, 4 * H> p = split<DT, 4 * H>(x);
                if (edge) {
                    // what lies outside may be anything, NaN among it: it meets no product
#pragma unroll
                    for (int e = 0; e < 4 * H; e++) {
                        const int q = t * TP + 16 * (e / 4) + 4 * grp + e % 4;
                        if (q < s.first || q >= s.end)
#pragma unroll
                            for (int w = 0; w < T::VW; w++) tile.v[e][w] = 0u;
                    }
                }
#pragma unroll
                for (int w = 0; w < T::VW; w++) {
                    typename T::Words f[DPW];
                    tile.vfrags(w, f);
#pragma unroll
                    for (int d = 0; d < DPW; d++)
#pragma unroll
                        for (int n = NP - 1; n >= 0; n--) acc[DPW * w + d] = mma<DT>(f[d], p.w[n], acc[DPW * w + d]);
                }
                load_v(s, runs);
            }
        }
        // the next part's first rows
        if (more && sn.mine < sn.t1) {
            heldn = offsets(sn.mine, pagesn, lostn);
            const Runs runs = runs_of(heldn, 0);
            load_k(sn, runs);
            load_v(sn, runs);
        }

        if (have) {
            // Parts of a row meet by their largest scores as exponents of 2.  Those beyond 2^100
            // go by the unscaled score's bits, which rise with it, from 2^100 on: finite, and 2^77
            // apart or more but where they agree to 2^-15 of themselves (below 2^108 a step is 2^84,
            // of 2^7 bits; all of fp32's positive numbers have 2^31).
            if (m != -INFINITY) {
                const float y = m * reach * to_log2;
                if (fabsf(y) > 0x1p100f) {
                    const int first = (int)__float_as_uint(0x1p100f / reach / to_log2), at = (int)__float_as_uint(fabsf(m));
                    m = copysignf(0x1p100f + (float)max(at - first, 0) * 0x1p77f, y);
                } else {
                    m = y;
                }
            }
            l = sum_over_groups(l);
            if (__any(lost)) {
                l = __builtin_nanf("");
                if (lane == 0 && head == 0) page_status(a.c, GSDH_PAGES_BAD_INDEX);
            }
            // the waves' outputs, joined in LDS
            float* ml = red + kWaves * G * HD;
            if (col < G) {
                float* o = red + ((size_t)wid * G + col) * HD + 4 * NT * grp;
#pragma unroll
                for (int r = 0; r < 4; r++)
#pragma unroll
                    for (int t = 0; t < NT; t += 4)
                        *reinterpret_cast<float4*>(o + r * NT + t) = make_float4(acc[t][r], acc[t + 1][r], acc[t + 2][r], acc[t + 3][r]);
                if (grp == 0) *reinterpret_cast<float2*>(ml + (wid * kMaxGroup + col) * 2) = make_float2(m, l);
            }
            __syncthreads();
            const bool whole = u.splits == 1;
            float* out = a.out + (int64_t)u.i * a.out_stride + (int64_t)head * G * HD;
            for (int i = tid; i < G * HD / 4; i += kThreads) {
                const int g = i / (HD / 4);
                float top = -INFINITY, sum = 0.f;
#pragma unroll
                for (int w = 0; w < kWaves; w++) top = fmaxf(top, ml[(w * kMaxGroup + g) * 2]);
                const float base = top == -INFINITY ? 0.f : top;
                float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int w = 0; w < kWaves; w++) {
                    const float2 e = *reinterpret_cast<const float2*>(ml + (w * kMaxGroup + g) * 2);
                    const float f = __builtin_amdgcn_exp2f(e.x - base);
                    const float4 y = *reinterpret_cast<const float4*>(red + ((size_t)w * G * HD + 4 * i));
                    sum += f * e.y;
                    o.x += f * y.x; o.y += f * y.y; o.z += f * y.z; o.w += f * y.w;
                }
                if (whole) {
                    // (nothing to attend to: zeros; scores that are all -inf: NaN)
                    const float f = u.row.end == u.row.first && sum == 0.f ? 0.f : vscale / sum;
                    *reinterpret_cast<float4*>(out + 4 * i) = make_float4(f * o.x, f * o.y, f * o.z, f * o.w);
                } else {
                    const size_t slot = (size_t)((u.span + u.split) * nkv + head) * 2 + (u.split == 0);
                    float* to = a.part + slot * G * HD + 4 * i;
                    put2(to, o.x, o.y);
                    put2(to + 2, o.z, o.w);
                    if (i % (HD / 4) == 0) put2(a.part_ml + (slot * G + g) * 2, top, sum);
                }
            }
            if (!whole) {
                // The block that arrives last of `many` neighbouring parts joins them,
                // the last of these (or the only one) all of the row: which parts
                // are added to which does not depend on who arrives when.
                unsigned* counter = a.counters + ((size_t)u.i * nkv + head) * a.counter_step;
                const int many = fan_of(G * HD), fans = (u.splits + many - 1) / many, fan = u.split / many;
                int first = fan * many, step = 1, count = min(many, u.splits - first), index = fans == 1 ? 0 : 1 + fan;
                for (bool done = fans == 1;; done = true) {
                    published();
                    __syncthreads();
                    if (tid == 0) last = arrive(counter + index, (unsigned)count);
                    __syncthreads();
                    if (!last) break;
                    join_parts<HD>(a, u, head, first, step, count, done, red, out, vscale);
                    if (done) break;
                    first = 0;
                    step = many;
                    count = fans;
                    index = 0;
                }
            }
        }
        if (!more) break;
#pragma unroll
        for (int j = 0; j < QN; j++)
            if (tid + j * kThreads < G * HD / 4) reinterpret_cast<float4v*>(qbuf)[tid + j * kThreads] = qn[j];
        __syncthreads();
        u = un;
        s = sn;
        held = heldn;
        lost = lostn;
        have = true;
    }
}

// ---------------------------------------------------------------------------
// RoPE and the append of K/V rows
// ---------------------------------------------------------------------------
struct StoreArgs {
    gsdh_paged_cache c;
    const float *q, *k, *v, *angles;
    float* q_out;
    const int *seqs, *positions;
    int64_t q_stride, k_stride, v_stride, q_out_stride;
    int layer, n_heads, n_angles, interleaved, parts;   // parts: blocks of a token
};

// eight values in the cache's type; e4m3: beyond +-448 clamped, NaN kept
template <int DT>
__device__ __forceinline__ void to_cache(const float (&x)[8], float scale, uint32_t (&w)[4]) {
    if constexpr (DT == GSDH_KV_E4M3) {
        float y[8];
#pragma unroll
        for (int e = 0; e < 8; e++) {
            y[e] = x[e] / scale;
            y[e] = y[e] > 448.f ? 448.f : y[e] < -448.f ? -448.f : y[e];
        }
#pragma unroll
        for (int i = 0; i < 2; i++) {
            int r = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * i], y[4 * i + 1], 0, false);
            w[i] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[4 * i + 2], y[4 * i + 3], r, true);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if constexpr (DT == GSDH_KV_BF16) {
                typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
                w[i] = __builtin_bit_cast(uint32_t, bf2{(__bf16)x[2 * i], (__bf16)x[2 * i + 1]});
            } else {
                w[i] = (uint32_t)f2h(x[2 * i]) | (uint32_t)f2h(x[2 * i + 1]) << 16;
            }
        }
    }
}

// One thread: four rotation pairs of a q or K head, or eight values of a V
// head.  Bound by its launch and the chain sequence -> page -> row for the
// tokens of a decode step (64 tokens 3.7 us), by memory for a prompt's (4099
// tokens into an e4m3 cache, 178 MB, 35 us: 5.1 TB/s).  The rotation is
// evaluated without contraction, as the one-token append evaluates it.
template <int DT>
__global__ void __launch_bounds__(256) paged_store_kernel(const StoreArgs a) {
#pragma clang fp contract(off)
    const int tok = blockIdx.x / a.parts, item = (blockIdx.x % a.parts) * 256 + threadIdx.x;
    const int hd = a.c.head_dim, nkv = a.c.n_kv_heads, per = hd / 8, head = item / per, j = item % per;
    if (head >= a.n_heads + 2 * nkv) return;
    const int seq = a.seqs[tok], pos = a.positions[tok];
    if (seq < 0) return;
    uint32_t bad = 0;
    int page = 0;
    if (seq >= a.c.n_seqs || pos < 0 || pos >= a.n_angles || pos >= a.c.table_width * a.c.page_size || pos >= a.c.lens[seq]) {
        bad = GSDH_PAGES_BAD_INDEX;
    } else {
        page = a.c.tables[(size_t)seq * a.c.table_width + pos / a.c.page_size];
        if ((unsigned)page >= (unsigned)a.c.n_pages) bad = GSDH_PAGES_BAD_INDEX;
        else if (a.c.refs && a.c.refs[page] != 1) bad = GSDH_PAGES_SHARED;
    }
    if (bad) {
        if (item == 0) page_status(a.c, bad);
        return;
    }
    const bool is_q = head < a.n_heads, is_v = head >= a.n_heads + nkv;
    const int h = is_q ? head : head - a.n_heads - (is_v ? nkv : 0);
    const float* src = (is_q ? a.q + tok * a.q_stride : is_v ? a.v + tok * a.v_stride : a.k + tok * a.k_stride) + h * hd;
    // the two runs of four: one run of eight (V, interleaved pairs) or one in each half of the head
    const int i0 = is_v || a.interleaved ? 8 * j : 4 * j, i1 = is_v || a.interleaved ? i0 + 4 : i0 + hd / 2;
    const float4 u = *reinterpret_cast<const float4*>(src + i0), w = *reinterpret_cast<const float4*>(src + i1);
    float x[8] = {u.x, u.y, u.z, u.w, w.x, w.y, w.z, w.w};
    if (!is_v) {
        const float4* cs = reinterpret_cast<const float4*>(a.angles + ((size_t)pos * (hd / 2) + 4 * j) * 2);
        const float4 c0 = cs[0], c1 = cs[1];
        const float c[4] = {c0.x, c0.z, c1.x, c1.z}, s[4] = {c0.y, c0.w, c1.y, c1.w};
#pragma unroll
        for (int p = 0; p < 4; p++) {
            const float y = a.interleaved ? x[2 * p] : x[p], z = a.interleaved ? x[2 * p + 1] : x[p + 4];
            const float r0 = y * c[p] - z * s[p], r1 = y * s[p] + z * c[p];
            if (a.interleaved) {
                x[2 * p] = r0;
                x[2 * p + 1] = r1;
            } else {
                x[p] = r0;
                x[p + 4] = r1;
            }
        }
    }
    if (is_q) {
        float* o = a.q_out + tok * a.q_out_stride + h * hd;
        *reinterpret_cast<float4*>(o + i0) = make_float4(x[0], x[1], x[2], x[3]);
        *reinterpret_cast<float4*>(o + i1) = make_float4(x[4], x[5], x[6], x[7]);
        return;
    }
    uint32_t y[4];
    float scale = 1.f;
    if constexpr (DT == GSDH_KV_E4M3) scale = (is_v ? a.c.v_scale : a.c.k_scale)[a.layer * nkv + h];
    to_cache<DT>(x, scale, y);
    constexpr int ES = DT == GSDH_KV_E4M3 ? 1 : 2;
    const int ps = a.c.page_size, slot = pos % ps;
    const size_t at = ((size_t)a.layer * a.c.n_pages + page) * ps * nkv * hd +
                      (a.c.head_major ? (size_t)h * ps + slot : (size_t)slot * nkv + h) * hd;
    unsigned char* dst = static_cast<unsigned char*>(is_v ? a.c.v : a.c.k) + at * ES;
    if constexpr (DT == GSDH_KV_E4M3) {
        *reinterpret_cast<uint32_t*>(dst + i0) = y[0];
        *reinterpret_cast<uint32_t*>(dst + i1) = y[1];
    } else {
        *reinterpret_cast<uint2*>(dst + 2 * i0) = make_uint2(y[0], y[1]);
        *reinterpret_cast<uint2*>(dst + 2 * i1) = make_uint2(y[2], y[3]);
    }
}

// ---------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------
// waves per SIMD that a launch has (it uses one of them for long rows)
constexpr int waves_per_simd(int hd) { return hd < 256 ? 2 : 1; }

// Blocks that fit the chip, as groups of one per KV head, at most 255 (what a
// row's fans can join); two partials of each (of a row that it continues and one
// that it starts).  KV heads that do not divide the CUs leave the rest of them
// idle, and a single one has no second wave per SIMD (128 rows of up to 4000, 8
// heads over 1: 26 us, 3.2 TB/s).
constexpr int kCounters = 1 + kMostFans;   // of a row and KV head: the row's, its fans'
struct AttendSpace {
    int groups, few;
    size_t slots;
    uint64_t bytes;
};
AttendSpace attend_space(const gsdh_paged_cache& c, int n, int n_heads, int cus) {
    AttendSpace s;
    auto fit = [&](int waves) {
        return std::min(std::max(1, (cus > 0 ? cus : 1) * waves * 4 / kWaves / c.n_kv_heads), kFan * kMostFans - 1);
    };
    s.groups = fit(waves_per_simd(c.head_dim));
    s.few = fit(1);
    s.slots = 2 * (size_t)s.groups * c.n_kv_heads;
    s.bytes = counted_workspace((uint64_t)n * c.n_kv_heads * kCounters, 4 * (uint64_t)s.slots * (n_heads / c.n_kv_heads) * (c.head_dim + 2));
    return s;
}

// the rows' costs add up in 32 bits
bool positions_fit(const gsdh_paged_cache& c, int n) {
    return n < 0 || (int64_t)n * ((int64_t)c.table_width * c.page_size / 16 + 2 + kRowCost) < 0x7FFFFFFF;
}

bool attend_shape(const gsdh_paged_cache& c, int n, int n_heads) {
    return n >= 0 && n_heads > 0 && n_heads % c.n_kv_heads == 0 && n_heads / c.n_kv_heads <= kMaxGroup &&
           (int64_t)n * c.n_kv_heads < (1 << 30);
}

template <int HD, int DT>
hipError_t launch_attend(const AttendArgs& a, hipStream_t st) {
    static LdsLimit limit;
    // q; then the waves' outputs and their (m, l), or (less) the join's weights and 1 / sums
    const size_t lds = 4 * ((size_t)(1 + kWaves) * a.group * HD + kWaves * kMaxGroup * 2 + (2 * kFan + 1) * kMaxGroup);
    const hipError_t e = raise_lds_limit(limit, reinterpret_cast<const void*>(paged_attn_kernel<HD, DT>), lds);
    if (e != hipSuccess) return e;
    const unsigned grid = (unsigned)(a.groups * a.c.n_kv_heads);
    hipLaunchKernelGGL((paged_attn_kernel<HD, DT>), dim3(grid), dim3(64 * kWaves), lds, st, a);
    return hipGetLastError();
}

template <int HD>
hipError_t launch_attend_type(const AttendArgs& a, hipStream_t st) {
    return a.c.dtype == GSDH_KV_F16 ? launch_attend<HD, GSDH_KV_F16>(a, st)
         : a.c.dtype == GSDH_KV_BF16 ? launch_attend<HD, GSDH_KV_BF16>(a, st)
                                     : launch_attend<HD, GSDH_KV_E4M3>(a, st);
}

bool rows_fit(const void* p, int64_t stride, int64_t width, bool written) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride % 4 == 0 && stride >= (written ? width : 0);
}

}  // namespace

namespace gsd {

int check_paged_cache(const gsdh_paged_cache* c, const char* who, bool needs_refs) {
    if (!c) return fail(-1, "%s: null cache", who);
    if (c->dtype < GSDH_KV_F16 || c->dtype > GSDH_KV_E4M3) return fail(-1, "%s: cache type %d", who, c->dtype);
    if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256)
        return fail(-1, "%s: head_dim %d not in {64,128,256}", who, c->head_dim);
    if (c->page_size < 8 || c->page_size > 256 || (c->page_size & (c->page_size - 1)))
        return fail(-1, "%s: page_size %d is not a power of two in 8..256", who, c->page_size);
    if (c->n_layers <= 0 || c->n_pages <= 0 || c->n_kv_heads <= 0 || c->table_width <= 0)
        return fail(-1, "%s: %d layers, %d pages, %d KV heads, tables of %d pages", who, c->n_layers, c->n_pages,
                    c->n_kv_heads, c->table_width);
    if (c->n_pages > 1 << 20) return fail(-1, "%s: %d pages (at most 2^20)", who, c->n_pages);
    if (c->n_kv_heads > 1024) return fail(-1, "%s: %d KV heads", who, c->n_kv_heads);
    if (c->n_seqs <= 0 || c->n_seqs > 8192) return fail(-1, "%s: n_seqs %d outside 1..8192", who, c->n_seqs);
    if ((int64_t)c->table_width * c->page_size > (1 << 30))
        return fail(-1, "%s: tables of %d pages of %d positions", who, c->table_width, c->page_size);
    if (!c->k || !c->v || !c->tables || !c->lens || !c->status || (needs_refs && !c->refs))
        return fail(-1, "%s: null buffer in the cache", who);
    if ((reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v)) % 16)
        return fail(-1, "%s: the pools are not 16-byte aligned", who);
    if (c->dtype == GSDH_KV_E4M3 ? !c->k_scale || !c->v_scale : c->k_scale || c->v_scale)
        return fail(-1, "%s: scales go with an e4m3 cache, and only with one", who);
    return 0;
}

int check_workspace(const void* ws, uint64_t have, uint64_t need, const char* who) {
    if (need && (!ws || have < need)) return fail(-1, "%s: %llu bytes of workspace, needs %llu", who,
                                                  (unsigned long long)(ws ? have : 0), (unsigned long long)need);
    if (need && reinterpret_cast<uintptr_t>(ws) % 16) return fail(-1, "%s: the workspace is not 16-byte aligned", who);
    return 0;
}

}  // namespace gsd

extern "C" {

uint64_t gsdh_paged_attention_workspace_bytes(const gsdh_paged_cache* c, int n, int n_heads) {
    if (check_paged_cache(c, "paged_attention_workspace_bytes", false) || !positions_fit(*c, n) ||
        !attend_shape(*c, n, n_heads))
        return 0;
    return attend_space(*c, n, n_heads, device_cu_count()).bytes;
}

int gsdh_paged_attention(void* stream, const gsdh_paged_cache* c, int layer, const float* q, int64_t q_stride,
                         const int* seqs, int n, int n_heads, float sm_scale, int window, float* out,
                         int64_t out_stride, void* workspace, uint64_t workspace_bytes) {
    const char* who = "paged_attention";
    int rc = check_paged_cache(c, who, false);
    if (rc) return rc;
    if (layer < 0 || layer >= c->n_layers) return fail(-1, "%s: layer %d outside 0..%d", who, layer, c->n_layers - 1);
    if (!positions_fit(*c, n))
        return fail(-1, "%s: %d rows of up to %lld positions in one call", who, n, (long long)c->table_width * c->page_size);
    if (!attend_shape(*c, n, n_heads))
        return fail(-1, "%s: %d rows of %d heads over %d KV heads (1..16 query heads per KV head)", who, n, n_heads,
                    c->n_kv_heads);
    if (!seqs && n > c->n_seqs) return fail(-1, "%s: %d rows, %d sequences", who, n, c->n_seqs);
    if (window < 0) return fail(-1, "%s: window %d", who, window);
    if (n == 0) return 0;
    const int64_t width = (int64_t)n_heads * c->head_dim;
    if (!q || !out || !rows_fit(q, q_stride, width, false) || !rows_fit(out, out_stride, width, true))
        return fail(-1, "%s: rows of q and out need 16-byte alignment, strides that are multiples of 4 and at least %lld for out",
                    who, (long long)width);
    const AttendSpace s = attend_space(*c, n, n_heads, device_cu_count());
    rc = check_workspace(workspace, workspace_bytes, s.bytes, who);
    if (rc) return rc;
    AttendArgs a{};
    a.c = *c;
    a.q = q; a.q_stride = q_stride; a.seqs = seqs; a.out = out; a.out_stride = out_stride;
    a.layer = layer; a.n = n; a.group = n_heads / c->n_kv_heads; a.window = window; a.groups = s.groups; a.few = s.few; a.scale = sm_scale;
    a.counters = static_cast<unsigned*>(workspace);
    // lines of their own where there is room: arrivals at one line wait for each other
    a.counter_step = (unsigned)std::min<size_t>(32, counter_bytes(workspace_bytes) / 4 / ((size_t)n * c->n_kv_heads));
    a.part = static_cast<float*>(workspace) + counter_bytes(workspace_bytes) / 4;
    a.part_ml = a.part + s.slots * a.group * c->head_dim;
    hipStream_t st = static_cast<hipStream_t>(stream);
    GSD_PAGED_CHK(c->head_dim == 64 ? launch_attend_type<64>(a, st)
                  : c->head_dim == 128 ? launch_attend_type<128>(a, st) : launch_attend_type<256>(a, st), who);
    return 0;
}

int gsdh_paged_rope_store(void* stream, const gsdh_paged_cache* c, int layer, const float* q, int64_t q_stride,
                          const float* k, int64_t k_stride, const float* v, int64_t v_stride, float* q_out,
                          int64_t q_out_stride, const int* seqs, const int* positions, int n, int n_heads,
                          const float* angles, int n_angles, int interleaved) {
    const char* who = "paged_rope_store";
    const int rc = check_paged_cache(c, who, false);
    if (rc) return rc;
    if (layer < 0 || layer >= c->n_layers) return fail(-1, "%s: layer %d outside 0..%d", who, layer, c->n_layers - 1);
    if (n < 0 || n_heads <= 0 || n_heads > 16384) return fail(-1, "%s: %d tokens of %d heads", who, n, n_heads);
    if (n_angles < 0) return fail(-1, "%s: angles of %d positions", who, n_angles);
    if (n == 0) return 0;
    if (!q || !k || !v || !q_out || !seqs || !positions || !angles) return fail(-1, "%s: null buffer", who);
    const int64_t width = (int64_t)n_heads * c->head_dim;
    if (!rows_fit(q, q_stride, width, false) || !rows_fit(k, k_stride, 0, false) || !rows_fit(v, v_stride, 0, false) ||
        !rows_fit(q_out, q_out_stride, width, true) || reinterpret_cast<uintptr_t>(angles) % 16)
        return fail(-1, "%s: rows need 16-byte alignment, strides that are multiples of 4 and at least %lld for q_out", who,
                    (long long)width);
    if (q_out == q && q_out_stride != q_stride) return fail(-1, "%s: q rotated in place needs one stride", who);
    StoreArgs a{};
    a.c = *c;
    a.q = q; a.k = k; a.v = v; a.q_out = q_out; a.angles = angles; a.seqs = seqs; a.positions = positions;
    a.q_stride = q_stride; a.k_stride = k_stride; a.v_stride = v_stride; a.q_out_stride = q_out_stride;
    a.layer = layer; a.n_heads = n_heads; a.n_angles = n_angles; a.interleaved = interleaved != 0;
    a.parts = (int)(((int64_t)(n_heads + 2 * c->n_kv_heads) * c->head_dim / 8 + 255) / 256);
    if ((int64_t)n * a.parts > 0x7FFFFFFF) return fail(-1, "%s: %d tokens of %d heads in one call", who, n, n_heads);
    hipStream_t st = static_cast<hipStream_t>(stream);
    const dim3 grid((unsigned)(n * a.parts)), block(256);
    switch (c->dtype) {
        case GSDH_KV_F16: hipLaunchKernelGGL(paged_store_kernel<GSDH_KV_F16>, grid, block, 0, st, a); break;
        case GSDH_KV_BF16: hipLaunchKernelGGL(paged_store_kernel<GSDH_KV_BF16>, grid, block, 0, st, a); break;
        default: hipLaunchKernelGGL(paged_store_kernel<GSDH_KV_E4M3>, grid, block, 0, st, a); break;
    }
    GSD_PAGED_CHK(hipGetLastError(), who);
    return 0;
}

}  // extern "C"
