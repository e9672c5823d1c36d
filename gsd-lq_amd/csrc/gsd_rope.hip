// gsd_rope.hip -- rotary positions: rows of q and K turned by angles that are
// formed from the positions, to rows or into the paged cache.
#include <cmath>

#include "gsd_device.h"
#include "gsd_paged.h"

using namespace gsd;

namespace {

constexpr int kThreads = 256;
constexpr int kMostPairs = 1024;   // of a block's tokens
constexpr int kMany = 4;           // items of a thread
constexpr int kFewBlocks = 2048;   // blocks of one item per thread that the chip takes at once

struct TurnArgs {
    const void *x, *k, *v;   // rows to rows: x alone
    void* out;
    const double* freqs;
    const int *seqs, *positions;
    gsdh_paged_cache c;
    int64_t x_stride, k_stride, v_stride, out_stride;
    int n, heads, nkv, hd;        // heads: of x
    int pairs, interleaved;
    int turned_runs, head_runs;   // threads' runs of a head that is turned: of four pairs; with those that follow
    int tokens, parts;            // of a block; blocks of a token
    int layer, in_place, many;    // many: kMany items per thread
    float scale;
};

template <typename T>
struct Vec {
    typedef T four __attribute__((ext_vector_type(4)));
};

template <typename RT, bool VEC>
__device__ __forceinline__ void load_run(const RT* p, int count, float* x) {   // up to four values
    if constexpr (VEC) {
        const auto w = *reinterpret_cast<const typename Vec<RT>::four*>(p);
#pragma unroll
        for (int e = 0; e < 4; e++) x[e] = (float)w[e];
    } else {
#pragma unroll
        for (int e = 0; e < 4; e++) x[e] = e < count ? (float)p[e] : 0.f;
    }
}
template <typename RT, bool VEC>
__device__ __forceinline__ void store_run(RT* p, int count, const float* x) {
    if constexpr (VEC) {
        typename Vec<RT>::four w;
#pragma unroll
        for (int e = 0; e < 4; e++) w[e] = (RT)x[e];
        *reinterpret_cast<typename Vec<RT>::four*>(p) = w;
    } else {
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (e < count) p[e] = (RT)x[e];
    }
}
// the same into a cache of type DT (bytes at p); e4m3: divided by the scale, beyond +-448 clamped, NaN kept
template <int DT, bool VEC>
__device__ __forceinline__ void cache_run(unsigned char* p, int count, const float* x, float scale) {
    if constexpr (DT == GSDH_KV_F16) {
        store_run<_Float16, VEC>(reinterpret_cast<_Float16*>(p), count, x);
    } else if constexpr (DT == GSDH_KV_BF16) {
        store_run<__bf16, VEC>(reinterpret_cast<__bf16*>(p), count, x);
    } else {
        float y[4];
#pragma unroll
        for (int e = 0; e < 4; e++) {
            y[e] = x[e] / scale;
            y[e] = y[e] > 448.f ? 448.f : y[e] < -448.f ? -448.f : y[e];
        }
        const uint32_t w =
            (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false), true);
        if constexpr (VEC) {
            *reinterpret_cast<uint32_t*>(p) = w;
        } else {
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (e < count) p[e] = (unsigned char)(w >> 8 * e);
        }
    }
}

// y_i = c x_i - s x_j, y_j = s x_i + c x_j, (c, s) = scale (cos, sin)(position *
// frequency): turns t = position * (frequency / 2 pi) in fp64, so that far
// positions keep their angles (an fp32 product is off by 2^-24 of it: half a
// degree at position 131072 and frequency 1), t's fraction rounded once to fp32.
//
// An item: four pairs of a head, or up to eight values that are not turned (the
// rest of a head, V).  A block's angles are formed once, in LDS, while its rows
// and, for the cache, sequence -> page come in.  DT < 0: rows to rows; else K and V
// go to the cache.  VEC: runs of four values are aligned (else element by element).
// U: items of a thread, 1 where that is few blocks (a step of 64 tokens: the launch
// and its chain of loads count, 3.4 us, 4.2 into the cache), else kMany, a token's items
// in one block: its chain is waited for once.  4099 tokens of 48 heads of 128 dims in
// bf16 into an e4m3 cache (92 MB) 26.4 us, 3.5 TB/s, 32.7 with one item per thread; 8191
// tokens of 40 heads, bf16 rows to rows (168 MB), 37.2 us, 4.5 TB/s, and 38.1.
template <typename RT, int DT, bool VEC, int U>
__global__ void __launch_bounds__(kThreads) turn_kernel(const TurnArgs a) {
    __shared__ float2 cs[kMostPairs];
    constexpr bool kPaged = DT >= 0;
    const int turned_items = (a.heads + (kPaged ? a.nkv : 0)) * a.head_runs, per_token = turned_items + (kPaged ? a.nkv * (a.hd / 8) : 0);
    const int first = a.tokens > 1 ? (int)blockIdx.x * a.tokens : (int)(blockIdx.x / (unsigned)a.parts);
    const int item0 = a.tokens > 1 ? (int)threadIdx.x : (int)(blockIdx.x % (unsigned)a.parts) * kThreads * U + (int)threadIdx.x;

    struct Item {
        int head, i0, i1, n0, n1, run;   // the two runs of up to four values
        bool is_k, is_v, turns, live;
    };
    Item it[U];
    float x[U][8];
    const int tok = U == 1 ? first + item0 / per_token : first;   // (one token: item0 < per_token, or nothing to do)
    const bool token = tok < a.n;
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int item = item0 + u * kThreads, in_token = U == 1 ? item % per_token : item;
        Item& t = it[u];
        t.live = token && item < a.tokens * per_token;
        t.is_v = kPaged && in_token >= turned_items;
        t.head = t.is_v ? (in_token - turned_items) / (a.hd / 8) : in_token / a.head_runs;
        t.run = t.is_v ? (in_token - turned_items) % (a.hd / 8) : in_token % a.head_runs;
        t.is_k = kPaged && !t.is_v && t.head >= a.heads;
        t.turns = !t.is_v && t.run < a.turned_runs;
        if (t.is_k) t.head -= a.heads;
        if (t.turns) {
            const int left = a.pairs - 4 * t.run;
            t.i0 = a.interleaved ? 8 * t.run : 4 * t.run;
            t.i1 = a.interleaved ? t.i0 + 4 : t.i0 + a.pairs;
            t.n0 = a.interleaved ? min(4, 2 * left) : min(4, left);
            t.n1 = a.interleaved ? max(0, min(4, 2 * left - 4)) : min(4, left);
        } else {
            t.i0 = t.is_v ? 8 * t.run : 2 * a.pairs + 8 * (t.run - a.turned_runs);
            t.i1 = t.i0 + 4;
            t.n0 = min(4, a.hd - t.i0);
            t.n1 = max(0, min(4, a.hd - t.i1));
            if (!t.is_k && !t.is_v && a.in_place) t.live = false;
        }
        if (t.live) {   // (rows that are left out below are read, too: they are there)
            const RT* src = static_cast<const RT*>(t.is_v ? a.v : t.is_k ? a.k : a.x) +
                            (int64_t)tok * (t.is_v ? a.v_stride : t.is_k ? a.k_stride : a.x_stride) + (int64_t)t.head * a.hd;
            load_run<RT, VEC>(src + t.i0, t.n0, x[u]);
            load_run<RT, VEC>(src + t.i1, t.n1, x[u] + 4);
        }
    }
    int pos = 0, page = 0;
    bool left_out = false;
    if constexpr (kPaged) {
        if (token && item0 < a.tokens * per_token) {
            const int seq = a.seqs[tok];
            pos = a.positions[tok];
            left_out = seq < 0;
            uint32_t bad = 0;
            if (!left_out) {
                if (seq >= a.c.n_seqs || pos < 0 || pos >= a.c.table_width * a.c.page_size || pos >= a.c.lens[seq]) {
                    bad = GSDH_PAGES_BAD_INDEX;
                } else {
                    page = a.c.tables[(size_t)seq * a.c.table_width + pos / a.c.page_size];
                    if ((unsigned)page >= (unsigned)a.c.n_pages) bad = GSDH_PAGES_BAD_INDEX;
                    else if (a.c.refs && a.c.refs[page] != 1) bad = GSDH_PAGES_SHARED;
                }
                if (bad && item0 % per_token == 0) page_status(a.c, bad);
                left_out = bad != 0;
            }
        }
    }
    for (int p = threadIdx.x; p < a.tokens * a.pairs; p += kThreads) {
        const int t = first + p / a.pairs;
        if (t >= a.n) break;
        const double turn = (double)a.positions[t] * (a.freqs[p % a.pairs] * 0.15915494309189533577);   // 1 / 2 pi
        float s, c;
        sincospif((float)(2.0 * (turn - rint(turn))), &s, &c);
        cs[p] = make_float2(c * a.scale, s * a.scale);
    }
    lds_barrier();   // (the rows need not be here yet)
    if (left_out) return;
#pragma unroll
    for (int u = 0; u < U; u++) {
        const Item& t = it[u];
        if (!t.live) continue;
        float (&y)[8] = x[u];
        if (t.turns) {
            const float2* const w = cs + (tok - first) * a.pairs + 4 * t.run;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                if (!VEC && 4 * t.run + e >= a.pairs) break;
                const float2 r = w[e];
                const float p = a.interleaved ? y[2 * e] : y[e], q = a.interleaved ? y[2 * e + 1] : y[e + 4];
                const float c = p * r.x - q * r.y, d = p * r.y + q * r.x;
                y[a.interleaved ? 2 * e : e] = c;
                y[a.interleaved ? 2 * e + 1 : e + 4] = d;
            }
        }
        if constexpr (kPaged) {
            if (t.is_k || t.is_v) {
                constexpr int ES = DT == GSDH_KV_E4M3 ? 1 : 2;
                const int ps = a.c.page_size, slot = pos % ps;
                const float scale = DT == GSDH_KV_E4M3 ? (t.is_v ? a.c.v_scale : a.c.k_scale)[a.layer * a.nkv + t.head] : 1.f;
                const size_t at = ((size_t)a.layer * a.c.n_pages + page) * ps * a.nkv * a.hd +
                                  (a.c.head_major ? (size_t)t.head * ps + slot : (size_t)slot * a.nkv + t.head) * a.hd;
                unsigned char* dst = static_cast<unsigned char*>(t.is_v ? a.c.v : a.c.k) + at * ES;
                cache_run<DT, VEC>(dst + (size_t)t.i0 * ES, t.n0, y, scale);
                cache_run<DT, VEC>(dst + (size_t)t.i1 * ES, t.n1, y + 4, scale);
                continue;
            }
        }
        RT* dst = static_cast<RT*>(a.out) + (int64_t)tok * a.out_stride + (int64_t)t.head * a.hd;
        store_run<RT, VEC>(dst + t.i0, t.n0, y);
        store_run<RT, VEC>(dst + t.i1, t.n1, y + 4);
    }
}

int check_rope(const gsdh_rope* r, int head_dim, int dtype, const char* who) {
    if (!r) return fail(-1, "%s: null rope", who);
    if (r->rotary_dim < 2 || r->rotary_dim % 2 || r->rotary_dim > head_dim)
        return fail(-1, "%s: rotary_dim %d is not even or outside 2..%d", who, r->rotary_dim, head_dim);
    if (dtype < GSDH_ROWS_F32 || dtype > GSDH_ROWS_BF16) return fail(-1, "%s: type %d", who, dtype);
    if (!r->freqs || reinterpret_cast<uintptr_t>(r->freqs) % 8) return fail(-1, "%s: frequencies null or not aligned", who);
    return 0;
}

bool rows_fit(const void* p, int64_t stride, int64_t width, int dtype) {
    const int unit = dtype == GSDH_ROWS_F32 ? 4 : 8;
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride % unit == 0 && stride >= width;
}

// the blocks' shape; false: too many
bool plan_turn(TurnArgs& a, const gsdh_rope& r, bool paged) {
    a.freqs = r.freqs;
    a.pairs = r.rotary_dim / 2;
    a.interleaved = r.interleaved != 0;
    a.scale = r.scale;
    a.turned_runs = (a.pairs + 3) / 4;
    a.head_runs = a.turned_runs + (a.hd - r.rotary_dim + 7) / 8;
    const int64_t items = (int64_t)(a.heads + (paged ? a.nkv : 0)) * a.head_runs + (paged ? (int64_t)a.nkv * (a.hd / 8) : 0);
    // short tokens share a block
    a.tokens = (int)(items <= kThreads / 2 ? kThreads / items : 1);
    if (a.tokens * a.pairs > kMostPairs) a.tokens = kMostPairs / a.pairs;
    a.parts = (int)((items + kThreads - 1) / kThreads);
    a.many = a.tokens == 1 && (int64_t)a.n * a.parts > kFewBlocks;
    if (a.many) a.parts = (int)((items + kMany * kThreads - 1) / (kMany * kThreads));
    return (a.tokens > 1 ? (int64_t)a.n : (int64_t)a.n * a.parts) <= 0x7FFFFFFF;
}

template <typename RT, int DT, bool VEC>
void launch_turn(const TurnArgs& a, hipStream_t st) {
    const dim3 grid((unsigned)(a.tokens > 1 ? (a.n + a.tokens - 1) / a.tokens : a.n * a.parts)), block(kThreads);
    if (a.many) hipLaunchKernelGGL((turn_kernel<RT, DT, VEC, kMany>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((turn_kernel<RT, DT, VEC, 1>), grid, block, 0, st, a);
}
template <typename RT, int DT>
void launch_turn(const TurnArgs& a, bool vec, hipStream_t st) {
    if (vec) launch_turn<RT, DT, true>(a, st);
    else launch_turn<RT, DT, false>(a, st);
}
template <int DT>
void launch_turn_rows(const TurnArgs& a, int dtype, bool vec, hipStream_t st) {
    if (dtype == GSDH_ROWS_F32) launch_turn<float, DT>(a, vec, st);
    else if (dtype == GSDH_ROWS_F16) launch_turn<_Float16, DT>(a, vec, st);
    else launch_turn<__bf16, DT>(a, vec, st);
}

}  // namespace

extern "C" {

int gsdh_rope_frequencies(int kind, double theta, int rotary_dim, double factor, double context, double low, double high, double* freqs) {
    const char* who = "rope_frequencies";
    if (kind < GSDH_ROPE_PLAIN || kind > GSDH_ROPE_BY_PARTS) return fail(-1, "%s: kind %d", who, kind);
    if (rotary_dim < 2 || rotary_dim % 2) return fail(-1, "%s: rotary_dim %d", who, rotary_dim);
    if (!(theta > 0) || std::isinf(theta)) return fail(-1, "%s: theta %g", who, theta);
    if (kind != GSDH_ROPE_PLAIN && (!(factor > 0) || std::isinf(factor))) return fail(-1, "%s: factor %g", who, factor);
    if (kind == GSDH_ROPE_NTK && rotary_dim == 2) return fail(-1, "%s: one pair has no base to change", who);
    if (kind == GSDH_ROPE_BY_PARTS && (!(context > 0) || !(high > low)))
        return fail(-1, "%s: a context of %g positions, turns from %g to %g", who, context, low, high);
    if (!freqs) return fail(-1, "%s: null buffer", who);
    if (kind == GSDH_ROPE_NTK) theta *= std::pow(factor, (double)rotary_dim / (rotary_dim - 2));
    if (std::isinf(theta)) return fail(-1, "%s: frequencies of an infinite theta", who);
    auto frequency = [&](int i) {
        const double f = std::pow(theta, -2.0 * i / rotary_dim);
        if (kind == GSDH_ROPE_LINEAR) return f / factor;
        if (kind != GSDH_ROPE_BY_PARTS) return f;
        const double turns = context * f * 0.15915494309189533577;   // 1 / 2 pi
        double keep = (turns - low) / (high - low);
        keep = keep < 0 ? 0 : keep > 1 ? 1 : keep;
        return keep * f + (1 - keep) * (f / factor);
    };
    for (int i = 0; i < rotary_dim / 2; i++)
        if (!std::isfinite(frequency(i))) return fail(-1, "%s: frequency %d is not a finite number", who, i);
    for (int i = 0; i < rotary_dim / 2; i++) freqs[i] = frequency(i);
    return 0;
}

int gsdh_rope_rows(void* stream, const gsdh_rope* r, const void* x, int dtype, int64_t x_stride, void* out, int64_t out_stride,
                   const int* positions, int n, int n_heads, int head_dim) {
    const char* who = "rope_rows";
    if (head_dim < 8 || head_dim > 1024 || head_dim % 8) return fail(-1, "%s: head_dim %d is not a multiple of 8 in 8..1024", who, head_dim);
    const int rc = check_rope(r, head_dim, dtype, who);
    if (rc) return rc;
    if (n < 0 || n > 1 << 30 || n_heads <= 0 || n_heads > 16384) return fail(-1, "%s: %d tokens of %d heads", who, n, n_heads);
    if (n == 0) return 0;
    if (!x || !out || !positions) return fail(-1, "%s: null buffer", who);
    const int64_t width = (int64_t)n_heads * head_dim;
    if (!rows_fit(x, x_stride, x == out ? width : 0, dtype) || !rows_fit(out, out_stride, width, dtype))
        return fail(-1, "%s: rows need 16-byte alignment, strides of whole 16 bytes and at least %lld for out", who, (long long)width);
    if (x == out && x_stride != out_stride) return fail(-1, "%s: rows turned in place need one stride", who);
    TurnArgs a{};
    a.x = x; a.x_stride = x_stride; a.out = out; a.out_stride = out_stride; a.positions = positions;
    a.n = n; a.heads = n_heads; a.hd = head_dim; a.in_place = x == out;
    if (!plan_turn(a, *r, false)) return fail(-1, "%s: %d tokens of %d heads in one call", who, n, n_heads);
    launch_turn_rows<-1>(a, dtype, r->rotary_dim % 8 == 0, static_cast<hipStream_t>(stream));
    GSD_PAGED_CHK(hipGetLastError(), who);
    return 0;
}

int gsdh_paged_rope_append(void* stream, const gsdh_paged_cache* c, int layer, const gsdh_rope* r, int dtype, const void* q, int64_t q_stride,
                           const void* k, int64_t k_stride, const void* v, int64_t v_stride, void* q_out, int64_t q_out_stride,
                           const int* seqs, const int* positions, int n, int n_heads) {
    const char* who = "paged_rope_append";
    int rc = check_paged_cache(c, who, false);
    if (rc) return rc;
    rc = check_rope(r, c->head_dim, dtype, who);
    if (rc) return rc;
    if (layer < 0 || layer >= c->n_layers) return fail(-1, "%s: layer %d outside 0..%d", who, layer, c->n_layers - 1);
    if (n < 0 || n > 1 << 30 || n_heads <= 0 || n_heads > 16384) return fail(-1, "%s: %d tokens of %d heads", who, n, n_heads);
    if (n == 0) return 0;
    if (!q || !k || !v || !q_out || !seqs || !positions) return fail(-1, "%s: null buffer", who);
    const int64_t width = (int64_t)n_heads * c->head_dim;
    if (!rows_fit(q, q_stride, q == q_out ? width : 0, dtype) || !rows_fit(k, k_stride, 0, dtype) || !rows_fit(v, v_stride, 0, dtype) ||
        !rows_fit(q_out, q_out_stride, width, dtype))
        return fail(-1, "%s: rows need 16-byte alignment, strides of whole 16 bytes and at least %lld for q_out", who, (long long)width);
    if (q_out == q && q_out_stride != q_stride) return fail(-1, "%s: q turned in place needs one stride", who);
    TurnArgs a{};
    a.c = *c;
    a.x = q; a.x_stride = q_stride; a.k = k; a.k_stride = k_stride; a.v = v; a.v_stride = v_stride; a.out = q_out; a.out_stride = q_out_stride;
    a.seqs = seqs; a.positions = positions; a.n = n; a.heads = n_heads; a.nkv = c->n_kv_heads; a.hd = c->head_dim; a.layer = layer;
    a.in_place = q == q_out;
    if (!plan_turn(a, *r, true)) return fail(-1, "%s: %d tokens of %d heads in one call", who, n, n_heads);
    const bool vec = r->rotary_dim % 8 == 0;
    hipStream_t st = static_cast<hipStream_t>(stream);
    switch (c->dtype) {
        case GSDH_KV_F16: launch_turn_rows<GSDH_KV_F16>(a, dtype, vec, st); break;
        case GSDH_KV_BF16: launch_turn_rows<GSDH_KV_BF16>(a, dtype, vec, st); break;
        default: launch_turn_rows<GSDH_KV_E4M3>(a, dtype, vec, st); break;
    }
    GSD_PAGED_CHK(hipGetLastError(), who);
    return 0;
}

}  // extern "C"
