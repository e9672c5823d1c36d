// gsd_paged.hip -- decode attention over a paged KV cache for a batch of
// sequences, and RoPE with the append of K/V rows to its pages.
#include "gsd_device.h"
#include "gsd_paged.h"

using namespace gsd;

namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));

constexpr float kLog2e = 1.44269504088896340736f;
constexpr int kTile = 32;          // positions of one step of a wave
constexpr int kWaves = 4;          // waves of a block, each on every fourth tile of its unit
constexpr int kUnitsPerCu = 4;     // units that a launch is split into, per CU (about)
constexpr int kMaxGroup = 16;      // query heads per KV head: the columns of one matrix product

// ---------------------------------------------------------------------------
// attention of one token per sequence
//
//   x_p = sm_scale q.K_p,  out = sum_p e^(x_p - m) V_p / sum_p e^(x_p - m)
//
// in one pass over K and V with a running maximum m and sum l.  A unit is a
// run of 32-position tiles of one (row, KV head), whose query heads are the
// columns of the matrix products: S^T = K Q^T and O^T = V^T P^T, 16 x 16 x 32.
// The keys of a tile are dealt to the products' rows so that the
// probabilities come out of the first product in the lane that the second
// one needs them in: lane l (column = head l & 15, group j = l >> 4) gets the
// scores of positions 4 j + r and 16 + 4 j + r (r < 4) and feeds the same
// eight positions, for which it also loads V's rows (dims NT (l & 15) ..,
// NT = head_dim / 16), so nothing goes through LDS or other lanes.  V's
// eight rows are transposed in registers by byte permutes.
//
// fp32 inputs meet the cache's 16-bit rows as sums of 16-bit parts: two fp16
// parts (22 bits; q scaled by a power of two so that its largest element is
// below 1024, P by 2^14, so that small parts keep their bits) or three bf16
// parts (24 bits).  e4m3 rows are exact in fp16.
// ---------------------------------------------------------------------------
struct AttendArgs {
    gsdh_paged_cache c;
    const float* q;
    const int* seqs;
    float* out;
    unsigned* counters;   // [n][n_kv] arrivals of split rows, zero between launches
    float* part;          // partial outputs [slot][G][HD], then (m, l) [slot][G][2]
    float* part_ml;
    int64_t q_stride, out_stride;
    int layer, n, group, window, target;   // target: units to split the work into
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
__device__ __forceinline__ int tiles_of(const Row& r) {
    return r.end > r.first ? (r.end - 1) / kTile - r.first / kTile + 1 : 0;
}
// units of a row and KV head (a row without positions has one: it writes the row)
__device__ __forceinline__ int units_of(const Row& r, int chunk) {
    if (r.seq < 0) return 0;
    const int t = tiles_of(r);
    return t <= chunk ? 1 : (t + chunk - 1) / chunk;
}

struct Unit {
    Row row;
    int i;        // row of the call
    int head;     // KV head
    int split, splits;
    int chunk;    // tiles per unit
    int slot;     // of split 0's partial (splits > 1)
};

// The unit of this block: every wave scans the rows by itself (lane l takes
// a run of them), so that no barrier comes before the first loads.  The
// chunk makes about `target` units of the launch's tiles, whatever the
// lengths are; rows of a few tiles make one each beyond that.
__device__ bool find_unit(const AttendArgs& a, unsigned u, Unit& o) {
    const int lane = threadIdx.x & 63, per = (a.n + 63) / 64, lo = lane * per, hi = min(a.n, lo + per);
    const int nkv = a.c.n_kv_heads;
    long long mine = 0;
    for (int i = lo; i < hi; i++) mine += tiles_of(row_of(a, i));
    long long total = mine;
#pragma unroll
    for (int s = 32; s >= 1; s >>= 1) total += __shfl_xor(total, s, 64);
    total *= nkv;
    long long ch = (total + a.target - 1) / a.target;
    ch = (ch + kWaves - 1) / kWaves * kWaves;
    // (2^25 tiles hold the longest sequence)
    const int chunk = (int)(ch < kWaves ? kWaves : ch > (1 << 25) ? 1 << 25 : ch);
    // units in the low half, slots of split rows in the high half
    unsigned long long cnt = 0;
    for (int i = lo; i < hi; i++) {
        const unsigned k = (unsigned)units_of(row_of(a, i), chunk);
        cnt += k + ((unsigned long long)(k > 1 ? k : 0) << 32);
    }
    unsigned long long incl = cnt;
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) {
        const unsigned long long b = __shfl_up(incl, s, 64);
        if (lane >= s) incl += b;
    }
    const unsigned v = u / (unsigned)nkv;
    unsigned before = (unsigned)(incl - cnt), slots = (unsigned)((incl - cnt) >> 32);
    const bool here = v >= before && v < (unsigned)incl;
    const unsigned long long who = __ballot(here);
    if (!who) return false;
    int i = lo, k = 0;
    if (here)
        for (;; i++) {
            k = units_of(row_of(a, i), chunk);
            if (v < before + (unsigned)k) break;
            before += k;
            slots += k > 1 ? k : 0;
        }
    const int src = __builtin_ctzll(who);
    o.i = __builtin_amdgcn_readlane(i, src);
    o.splits = __builtin_amdgcn_readlane(k, src);
    o.split = (int)v - __builtin_amdgcn_readlane((int)before, src);
    o.slot = __builtin_amdgcn_readlane((int)slots, src) * nkv;
    o.head = (int)(u - v * (unsigned)nkv);
    o.slot += o.head * o.splits;
    o.chunk = chunk;
    o.row = row_of(a, o.i);
    return true;
}

__device__ __forceinline__ float max_over_groups(float v) {   // over lanes l, l ^ 16, l ^ 32, l ^ 48
    auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
    r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float sum_over_groups(float v) { return swap_add32(swap_add16(v, v), swap_add16(v, v), false); }

// Eight fp32 values as parts of 16 bits whose sum they are
template <int DT>
struct Parts {
    static constexpr int N = DT == GSDH_KV_BF16 ? 3 : 2;
    uint4 w[N];
};
template <int DT>
__device__ __forceinline__ Parts<DT> split8(const float (&x)[8]) {
    Parts<DT> p;
    if constexpr (DT == GSDH_KV_BF16) {
        // truncated parts: 8 + 8 + 8 bits, exact
        uint32_t h[8], m[8], l[8];
#pragma unroll
        for (int e = 0; e < 8; e++) {
            h[e] = __float_as_uint(x[e]);
            const float r = x[e] - __uint_as_float(h[e] & 0xFFFF0000u);
            m[e] = __float_as_uint(r);
            l[e] = __float_as_uint(r - __uint_as_float(m[e] & 0xFFFF0000u));
        }
        auto pack = [](const uint32_t (&v)[8]) {
            return make_uint4(__builtin_amdgcn_perm(v[1], v[0], 0x07060302u), __builtin_amdgcn_perm(v[3], v[2], 0x07060302u),
                              __builtin_amdgcn_perm(v[5], v[4], 0x07060302u), __builtin_amdgcn_perm(v[7], v[6], 0x07060302u));
        };
        p.w[0] = pack(h);
        p.w[1] = pack(m);
        p.w[2] = pack(l);
    } else {
        half8 h, l;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            h[e] = (_Float16)x[e];
            l[e] = (_Float16)(x[e] - (float)h[e]);
        }
        p.w[0] = __builtin_bit_cast(uint4, h);
        p.w[1] = __builtin_bit_cast(uint4, l);
    }
    return p;
}

template <int DT>
__device__ __forceinline__ float4v mma(const uint4 a, const uint4 b, float4v c) {
    if constexpr (DT == GSDH_KV_BF16)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8, a), __builtin_bit_cast(bf8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c, 0, 0, 0);
}

// two e4m3 values (the low or the high half of w) as fp16: exact
template <bool HI>
__device__ __forceinline__ uint32_t e4m3x2(uint32_t w) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, HI));
}

// The rows of one tile as a lane holds them, and where they come from.
template <int HD, int DT>
struct Tile {
    static constexpr int ES = DT == GSDH_KV_E4M3 ? 1 : 2;
    static constexpr int KS = HD / 32;            // products over the head dims
    static constexpr int KL = HD * ES / 64;       // 16-byte loads of a lane's part of a K row
    static constexpr int NT = HD / 16;            // dims of a lane's part of a V row
    static constexpr int VW = NT * ES / 4;        // its words
    uint4 k[2][KL];
    uint32_t v[8][VW];

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
    // V's operands of the four (e4m3) or two dims of word w: positions 0 .. 7 of each dim
    __device__ __forceinline__ void vfrags(int w, uint4* f) const {
        uint32_t t[4][4];
#pragma unroll
        for (int p = 0; p < 4; p++) {
            const uint32_t a = v[2 * p][w], b = v[2 * p + 1][w];
            if constexpr (DT == GSDH_KV_E4M3) {
                const uint32_t x = __builtin_amdgcn_perm(b, a, 0x05010400u), y = __builtin_amdgcn_perm(b, a, 0x07030602u);
                t[0][p] = e4m3x2<false>(x);
                t[1][p] = e4m3x2<true>(x);
                t[2][p] = e4m3x2<false>(y);
                t[3][p] = e4m3x2<true>(y);
            } else {
                t[0][p] = __builtin_amdgcn_perm(b, a, 0x05040100u);
                t[1][p] = __builtin_amdgcn_perm(b, a, 0x07060302u);
            }
        }
#pragma unroll
        for (int d = 0; d < 4 / ES; d++) f[d] = make_uint4(t[d][0], t[d][1], t[d][2], t[d][3]);
    }
};

template <int HD, int DT>
__global__ void __launch_bounds__(64 * kWaves, HD == 256 ? 1 : 2) paged_attn_kernel(const AttendArgs a) {
    typedef Tile<HD, DT> T;
    constexpr int NP = Parts<DT>::N, NT = T::NT, DPW = 4 / T::ES;   // dims of a V word
    extern __shared__ float red[];                                  // [kWaves][G][HD], then (m, l) [kWaves][16][2]
    Unit u;
    if (!find_unit(a, blockIdx.x, u)) return;
    const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6, col = lane & 15, grp = lane >> 4;
    const int G = a.group, nkv = a.c.n_kv_heads, first = u.row.first, end = u.row.end;
    const float* kscale = a.c.k_scale ? a.c.k_scale + a.layer * nkv + u.head : nullptr;
    const float vscale = DT == GSDH_KV_E4M3 ? a.c.v_scale[a.layer * nkv + u.head] : 1.0f;
    float* out = a.out + (int64_t)u.i * a.out_stride + (int64_t)u.head * G * HD;

    // q's operand: head `col`, zeros beyond the group
    Parts<DT> q[T::KS];
    float to_log2;
    {
        float x[T::KS][8], most = 0.f;
        const float* qp = a.q + (int64_t)u.i * a.q_stride + ((int64_t)u.head * G + (col < G ? col : 0)) * HD;
#pragma unroll
        for (int s = 0; s < T::KS; s++) {
            const float4 lo = *reinterpret_cast<const float4*>(qp + T::dim(s, grp));
            const float4 hi = *reinterpret_cast<const float4*>(qp + T::dim(s, grp) + 4);
            const float w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
            for (int e = 0; e < 8; e++) {
                x[s][e] = col < G ? w[e] : 0.f;
                most = fmaxf(most, fabsf(x[s][e]));
            }
        }
        // 2^(9 - exponent of the largest), kept within the range of normal floats
        unsigned ex = __float_as_uint(max_over_groups(most)) >> 23;
        ex = ex < 16u ? 16u : ex > 254u ? 254u : ex;
        const float up = __uint_as_float((263u - ex) << 23), down = __uint_as_float((ex - 9u) << 23);
        to_log2 = a.scale * kLog2e * (DT == GSDH_KV_E4M3 ? *kscale : 1.0f) * down;
#pragma unroll
        for (int s = 0; s < T::KS; s++) {
#pragma unroll
            for (int e = 0; e < 8; e++) x[s][e] *= up;
            q[s] = split8<DT>(x[s]);
        }
    }

    float4v acc[NT];
#pragma unroll
    for (int t = 0; t < NT; t++) acc[t] = float4v{0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.f;
    bool lost = u.row.bad;

    const int t0 = first / kTile + u.split * u.chunk;
    const int t1 = end > first ? min(t0 + u.chunk, (end - 1) / kTile + 1) : 0;
    const size_t page_b = (size_t)a.c.page_size * nkv * HD * T::ES;
    const unsigned row_b = (a.c.head_major ? 1u : (unsigned)nkv) * HD * T::ES;
    const size_t head_b = (size_t)u.head * (a.c.head_major ? a.c.page_size : 1) * HD * T::ES;
    const unsigned char* kb = static_cast<const unsigned char*>(a.c.k) + (size_t)a.layer * a.c.n_pages * page_b + head_b;
    const unsigned char* vb = static_cast<const unsigned char*>(a.c.v) + (size_t)a.layer * a.c.n_pages * page_b + head_b;
    const int* table = a.c.tables + (size_t)u.row.seq * a.c.table_width;
    const int psl = __builtin_ctz((unsigned)a.c.page_size), psm = a.c.page_size - 1;
    // positions outside first .. end - 1 (rows of the first and last tile that
    // the mask drops) read the nearest row inside: what lies beyond, NaN
    // among it, meets no product
    auto inside = [&](int p) { return min(max(p, first), end - 1); };
    auto page_of = [&](int p) {
        const int pg = table[p >> psl];
        if ((unsigned)pg < (unsigned)a.c.n_pages) return pg;
        lost = true;
        return 0;
    };
    T tile;
    auto load_k = [&](int t) {
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int p = inside(t * kTile + 16 * h + col);
            tile.load_k(h, kb + (size_t)page_of(p) * page_b + (unsigned)(p & psm) * row_b + 16 * grp);
        }
    };
    auto load_v = [&](int t) {
#pragma unroll
        for (int h = 0; h < 2; h++) {
            // four positions from a multiple of 4 on share a page
            const int g = t * kTile + 16 * h + 4 * grp;
            const unsigned char* pb = vb + (size_t)page_of(inside(g)) * page_b + NT * T::ES * col;
#pragma unroll
            for (int r = 0; r < 4; r++) tile.load_v(4 * h + r, pb + (unsigned)(inside(g + r) & psm) * row_b);
        }
    };
    if (t0 + wid < t1) {
        load_k(t0 + wid);
        load_v(t0 + wid);
    }
    for (int t = t0 + wid; t < t1; t += kWaves) {
        float4v s[2] = {float4v{0.f, 0.f, 0.f, 0.f}, float4v{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
        for (int i = 0; i < T::KS; i++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const uint4 f = tile.kfrag(h, i);
#pragma unroll
                for (int p = NP - 1; p >= 0; p--) s[h] = mma<DT>(f, q[i].w[p], s[h]);
            }
        const bool more = t + kWaves < t1;
        if (more) load_k(t + kWaves);
        float x[8], top = -INFINITY;
        const int p0 = t * kTile + 4 * grp;
        if (p0 - 4 * grp >= first && p0 - 4 * grp + kTile <= end) {
#pragma unroll
            for (int e = 0; e < 8; e++) x[e] = s[e >> 2][e & 3] * to_log2;
        } else {
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const int p = p0 + 16 * (e >> 2) + (e & 3);
                x[e] = p >= first && p < end ? s[e >> 2][e & 3] * to_log2 : -INFINITY;
            }
        }
#pragma unroll
        for (int e = 0; e < 8; e++) top = fmaxf(top, x[e]);
        top = fmaxf(m, max_over_groups(top));
        if (__any(top > m)) {
            const float f = top == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - top);
#pragma unroll
            for (int n = 0; n < NT; n++) acc[n] *= f;
            l *= f;
            m = top;
        }
        // P as 2^14 times itself: the parts below fp16's normal range stay exact
        const float base = m == -INFINITY ? 0.f : m - 14.f;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            x[e] = __builtin_amdgcn_exp2f(x[e] - base);
            l += x[e];
        }
        const Parts<DT> p = split8<DT>(x);
#pragma unroll
        for (int w = 0; w < T::VW; w++) {
            uint4 f[DPW];
            tile.vfrags(w, f);
#pragma unroll
            for (int d = 0; d < DPW; d++)
#pragma unroll
                for (int n = NP - 1; n >= 0; n--) acc[DPW * w + d] = mma<DT>(f[d], p.w[n], acc[DPW * w + d]);
        }
        if (more) load_v(t + kWaves);
    }
    l = sum_over_groups(l);
    if (__any(lost)) {
        l = __builtin_nanf("");
        if (lane == 0 && u.head == 0) page_status(a.c, GSDH_PAGES_BAD_INDEX);
    }

    // the four waves' outputs, joined in LDS
    float* ml = red + kWaves * G * HD;
    if (col < G) {
        float* o = red + ((size_t)wid * G + col) * HD + 4 * NT * grp;
#pragma unroll
        for (int r = 0; r < 4; r++)
#pragma unroll
            for (int t = 0; t < NT; t += 4)
                *reinterpret_cast<float4*>(o + r * NT + t) = make_float4(acc[t][r], acc[t + 1][r], acc[t + 2][r], acc[t + 3][r]);
        if (grp == 0) {
            ml[(wid * kMaxGroup + col) * 2] = m;
            ml[(wid * kMaxGroup + col) * 2 + 1] = l;
        }
    }
    __syncthreads();
    const bool whole = u.splits == 1;
    for (int i = threadIdx.x; i < G * HD / 4; i += 64 * kWaves) {
        const int g = i / (HD / 4);
        float top = -INFINITY, sum = 0.f;
#pragma unroll
        for (int w = 0; w < kWaves; w++) top = fmaxf(top, ml[(w * kMaxGroup + g) * 2]);
        const float base = top == -INFINITY ? 0.f : top;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kWaves; w++) {
            const float f = __builtin_amdgcn_exp2f(ml[(w * kMaxGroup + g) * 2] - base);
            const float4 y = *reinterpret_cast<const float4*>(red + ((size_t)w * G * HD + 4 * i));
            sum += f * ml[(w * kMaxGroup + g) * 2 + 1];
            o.x += f * y.x; o.y += f * y.y; o.z += f * y.z; o.w += f * y.w;
        }
        if (whole) {
            const float f = sum == 0.f ? 0.f : vscale / sum;
            *reinterpret_cast<float4*>(out + 4 * i) = make_float4(f * o.x, f * o.y, f * o.z, f * o.w);
        } else {
            const size_t slot = (size_t)u.slot + u.split;
            *reinterpret_cast<float4*>(a.part + slot * G * HD + 4 * i) = o;
            if (i % (HD / 4) == 0) *reinterpret_cast<float2*>(a.part_ml + (slot * G + g) * 2) = make_float2(top, sum);
        }
    }
    if (whole) return;

    // the last of the row's units to arrive joins all of them, in their order
    __shared__ int last;
    __syncthreads();
    if (threadIdx.x == 0) {
        unsigned* c = a.counters + (size_t)u.i * nkv + u.head;
        __threadfence();
        last = __hip_atomic_fetch_add(c, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (unsigned)u.splits - 1u;
        __threadfence();
        if (last) __hip_atomic_store(c, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    if (!last) return;
    const float* part = a.part + (size_t)u.slot * G * HD;
    const float* pml = a.part_ml + (size_t)u.slot * G * 2;
    for (int i = threadIdx.x; i < G * HD / 4; i += 64 * kWaves) {
        const int g = i / (HD / 4);
        float top = -INFINITY, sum = 0.f;
        for (int w = 0; w < u.splits; w++) top = fmaxf(top, pml[(w * G + g) * 2]);
        const float base = top == -INFINITY ? 0.f : top;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
        for (int w = 0; w < u.splits; w++) {
            const float2 e = *reinterpret_cast<const float2*>(pml + (w * G + g) * 2);
            const float4 y = *reinterpret_cast<const float4*>(part + (size_t)w * G * HD + 4 * i);
            const float f = __builtin_amdgcn_exp2f(e.x - base);
            sum += f * e.y;
            o.x += f * y.x; o.y += f * y.y; o.z += f * y.z; o.w += f * y.w;
        }
        const float f = sum == 0.f ? 0.f : vscale / sum;
        *reinterpret_cast<float4*>(out + 4 * i) = make_float4(f * o.x, f * o.y, f * o.z, f * o.w);
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
// tokens of a decode step, by memory for a prompt's.  The rotation is
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
// partials of split rows: a launch of `target` units' worth of tiles has less
// than 2 target units in rows of several
struct AttendSpace {
    int target;
    size_t slots;
    uint64_t bytes;
};
AttendSpace attend_space(const gsdh_paged_cache& c, int n, int n_heads, int cus) {
    AttendSpace s;
    s.target = kUnitsPerCu * (cus > 0 ? cus : 1);
    s.slots = 2 * (size_t)s.target + c.n_kv_heads;
    s.bytes = counted_workspace((uint64_t)n * c.n_kv_heads, 4 * (uint64_t)s.slots * (n_heads / c.n_kv_heads) * (c.head_dim + 2));
    return s;
}

bool attend_shape(const gsdh_paged_cache& c, int n, int n_heads) {
    return n >= 0 && n_heads > 0 && n_heads % c.n_kv_heads == 0 && n_heads / c.n_kv_heads <= kMaxGroup &&
           (int64_t)n * c.n_kv_heads < (1 << 30);
}

template <int HD, int DT>
hipError_t launch_attend(const AttendArgs& a, hipStream_t st) {
    static LdsLimit limit;
    const size_t lds = 4 * ((size_t)kWaves * a.group * HD + kWaves * kMaxGroup * 2);
    const hipError_t e = raise_lds_limit(limit, reinterpret_cast<const void*>(paged_attn_kernel<HD, DT>), lds);
    if (e != hipSuccess) return e;
    const unsigned grid = (unsigned)(a.target + (int64_t)a.n * a.c.n_kv_heads);
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
    if (check_paged_cache(c, "paged_attention_workspace_bytes", false) || !attend_shape(*c, n, n_heads)) return 0;
    return attend_space(*c, n, n_heads, device_cu_count()).bytes;
}

int gsdh_paged_attention(void* stream, const gsdh_paged_cache* c, int layer, const float* q, int64_t q_stride,
                         const int* seqs, int n, int n_heads, float sm_scale, int window, float* out,
                         int64_t out_stride, void* workspace, uint64_t workspace_bytes) {
    const char* who = "paged_attention";
    int rc = check_paged_cache(c, who, false);
    if (rc) return rc;
    if (layer < 0 || layer >= c->n_layers) return fail(-1, "%s: layer %d outside 0..%d", who, layer, c->n_layers - 1);
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
    a.layer = layer; a.n = n; a.group = n_heads / c->n_kv_heads; a.window = window; a.target = s.target; a.scale = sm_scale;
    a.counters = static_cast<unsigned*>(workspace);
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
