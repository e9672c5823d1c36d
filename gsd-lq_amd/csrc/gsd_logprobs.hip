// gsd_logprobs.hip -- log probabilities of given tokens, entropy and the
// largest alternatives of rows of logits, each logit read once.
#include <algorithm>

#include "gsd_device.h"
#include "gsd_paged.h"

using namespace gsd;

namespace {

constexpr int kThreads = 256;
constexpr int kGroups = 64;         // of kThreads / 64 threads
constexpr int kMaxSeg = 128;        // segments of a row
constexpr int kBlocks = 512;        // that a launch is split into where it has fewer rows: two per CU
constexpr int kNV = 4;              // 16-byte words of a thread in one chunk
constexpr int chunk_of(int dtype) { return kThreads * kNV * (dtype == GSDH_LOGITS_F32 ? 4 : 8); }   // logits of a chunk
constexpr int kMaxTop = 32;
constexpr int kMaxVocab = (1 << 20) - 8;
constexpr int kMaxCand = 1024;      // keys that are ranked at once
constexpr int kHeld = 2;            // keys of other segments that a thread holds
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.693147180559945309417f;

// A logit and its place as one word that orders them: larger logits first,
// then lower indices.  0 is below every key.  -0 counts as +0, NaN as -inf.
__device__ __forceinline__ uint64_t key_of(float x, int index) {
    const uint32_t b = __float_as_uint(fmaxf(x, -INFINITY) + 0.f);
    const uint32_t o = b & 0x80000000u ? ~b : b | 0x80000000u;
    return (uint64_t)o << 32 | (uint32_t)~index;
}
__device__ __forceinline__ int index_of(uint64_t key) { return (int)~(uint32_t)key; }
__device__ __forceinline__ float value_of(uint64_t key) {
    const uint32_t o = (uint32_t)(key >> 32);
    return __uint_as_float(o & 0x80000000u ? o & 0x7FFFFFFFu : ~o);
}

struct LogprobArgs {
    const void* logits;
    const int* tokens;
    float *logprob, *entropy, *top_lp;
    int* top_ids;
    unsigned* counters;       // [n], zero between launches
    float* part;              // [n][nseg] (m, s, t, -)
    uint64_t* part_keys;      // [n][nseg][top]
    int64_t stride;
    int vocab, top, nseg, chunks;   // chunks of a segment
};

template <int DT>
__device__ __forceinline__ float logit_at(const void* p, int64_t i) {
    if constexpr (DT == GSDH_LOGITS_F32) return static_cast<const float*>(p)[i];
    else if constexpr (DT == GSDH_LOGITS_F16) return h2f(static_cast<const uint16_t*>(p)[i]);
    else return __uint_as_float((uint32_t)static_cast<const uint16_t*>(p)[i] << 16);
}

__device__ __forceinline__ uint64_t shfl_max(uint64_t k, int mask) {
    const uint64_t o = __shfl_xor((unsigned long long)k, mask, 64);
    return o > k ? o : k;
}
// over lanes l, l ^ 1, l ^ 2, l ^ 3, in VALU
__device__ __forceinline__ uint64_t quad_max(uint64_t k) {
#define GSD_QUAD_STEP(ctrl)                                                                                              \
    {                                                                                                                    \
        const uint32_t lo = (uint32_t)__builtin_amdgcn_mov_dpp((int)(uint32_t)k, ctrl, 0xF, 0xF, true);                  \
        const uint32_t hi = (uint32_t)__builtin_amdgcn_mov_dpp((int)(uint32_t)(k >> 32), ctrl, 0xF, 0xF, true);          \
        const uint64_t o = (uint64_t)hi << 32 | lo;                                                                      \
        k = o > k ? o : k;                                                                                               \
    }
    GSD_QUAD_STEP(0xB1);   // quad_perm 1 0 3 2
    GSD_QUAD_STEP(0x4E);   // quad_perm 2 3 0 1
#undef GSD_QUAD_STEP
    return k;
}

// How many of the first `count` (<= 64) keys are above each: every wave counts
// a quarter of them for key `lane`, all waves have the sums.  All threads take
// part; keys and `partial` were last used before a barrier.  (One wave's loop
// over 64 keys took 1 us.)
typedef int Partial[kThreads / 64][64];
__device__ __forceinline__ int count_above(const uint64_t* keys, int count, uint64_t mine, Partial& partial) {
    const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6, per = (count + kThreads / 64 - 1) / (kThreads / 64);
    int above = 0;
#pragma unroll 8
    for (int i = wid * per; i < min(wid * per + per, count); i++) above += keys[i] > mine;
    partial[wid][lane] = above;
    __syncthreads();
    above = 0;
#pragma unroll
    for (int w = 0; w < kThreads / 64; w++) above += partial[w][lane];
    return above;
}

// The `want`-th largest of the first `count` (<= 128) keys of lds (0: fewer
// nonzero ones than that), by counting for each how many are larger.  Every
// wave has it; nonzero keys differ.
__device__ uint64_t nth_largest(const uint64_t* keys, int count, int want, Partial& partial) {
    const int lane = threadIdx.x & 63;
    uint64_t found = 0;
    for (int base = 0; base < count; base += 64) {
        const uint64_t mine = base + lane < count ? keys[base + lane] : 0;
        int above = 0;
        if (count <= 64) {
            above = count_above(keys, count, mine, partial);
        } else {
#pragma unroll 8
            for (int i = 0; i < count; i++) above += keys[i] > mine;
        }
        const unsigned long long hit = __ballot(mine != 0 && above == want - 1);
        if (hit) {
            const int src = __builtin_ctzll(hit);
            found = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(mine >> 32), src) << 32 |
                    (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)mine, src);
        }
    }
    return found;
}

// out[r] = the r-th largest of cand[0 .. count), r < top; 0 behind the last
__device__ void select_top(const uint64_t* cand, int count, int top, uint64_t* out, Partial& partial) {
    for (int i = count + (int)threadIdx.x; i < top; i += kThreads) out[i] = 0;
    if (count <= 64) {
        const int lane = threadIdx.x & 63;
        const uint64_t mine = lane < count ? cand[lane] : 0;
        const int above = count_above(cand, count, mine, partial);
        if ((int)threadIdx.x < count && above < top) out[above] = mine;
        return;
    }
    for (int i = threadIdx.x; i < count; i += kThreads) {
        const uint64_t mine = cand[i];
        int above = 0;
#pragma unroll 4
        for (int j = 0; j < count; j++) above += cand[j] > mine;
        if (above < top) out[above] = mine;
    }
}

// The row's results from its sums (m, s, t), its token's logit (thread 0) and its largest keys (LDS).
__device__ __forceinline__ void finish_row(const LogprobArgs& a, int row, int tok, float logit, float m, float s, float t, const uint64_t* keys) {
    const float log_s = __builtin_amdgcn_logf(s) * kLn2;
    // (m is -inf where nothing has probability, and s NaN where a logit was NaN or +inf)
    const bool none = !(s > 0.f) || m == -INFINITY;
    if (threadIdx.x == 0) {
        if (a.logprob) {
            float v = __builtin_nanf("");
            if (tok == -1) v = 0.f;
            else if (tok >= 0 && tok < a.vocab && !none) v = (logit - m) - log_s;
            a.logprob[row] = v;
        }
        if (a.entropy) a.entropy[row] = none ? __builtin_nanf("") : log_s - t / s;
    }
    if ((int)threadIdx.x < a.top) {
        const uint64_t k = keys[threadIdx.x];
        a.top_ids[(int64_t)row * a.top + threadIdx.x] = index_of(k);
        a.top_lp[(int64_t)row * a.top + threadIdx.x] = none ? __builtin_nanf("") : (value_of(k) - m) - log_s;
    }
}

// One block: a segment of a row, chunk by chunk, the next chunk's loads ahead
// of this one's arithmetic.  Each thread keeps, of its logits,
//
//   m = max x,  s = sum e^(x - m),  t = sum e^(x - m) (x - m)
//   ln p = x - m - ln s,  entropy = ln s - t / s   (no cancellation: both terms are >= 0)
//
// and the word of four or eight logits that its largest first came in.
// The largest `top`: 64 groups of four threads each give the largest (value,
// then lower word) of theirs; `top` groups reach the top-th largest of these,
// so `top` logits do at least.  The words of the threads that reach it are read
// again, by all threads, and the logits at or above it (some `top` more of
// ordinary rows) are ranked by counting.  A row of several segments is joined by the
// block that arrives last.  Logits are read in 16-byte words from the aligned
// address at or below the row's first, those of a row's edges one by one.
//
// 512 rows of 32768 in fp32 (67 MB) take 14.4 us, 61 rows of 130001 in bf16 (16
// MB) 13.4: eight instructions a logit, then about 5 us of dependent steps
// (the groups' keys, the words read again, the ranking, the join).  Segments
// of 8192 in registers with a selection for each took 27 and 18 us.
template <int DT>
__global__ void __launch_bounds__(kThreads) logprob_kernel(const LogprobArgs a) {
    constexpr int VEC = DT == GSDH_LOGITS_F32 ? 4 : 8, ES = DT == GSDH_LOGITS_F32 ? 4 : 2, kChunk = chunk_of(DT), kWavesOf = kThreads / 64;
    constexpr float kLowest = -3.40282347e38f;
    __shared__ float red[3 * kWavesOf];
    __shared__ uint64_t group[kMaxSeg], best[kMaxTop], cand[kMaxCand];
    __shared__ uint8_t owner[kThreads];
    __shared__ Partial partial;
    __shared__ int n_cand, n_owner, last;
    const int row = blockIdx.x / a.nseg, seg = blockIdx.x % a.nseg, tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
    const unsigned char* base = static_cast<const unsigned char*>(a.logits) + row * a.stride * ES;
    const int off = (int)(reinterpret_cast<uintptr_t>(base) % 16) / ES;   // logits between the aligned address and the row
    base -= off * ES;
    const int end = off + a.vocab;   // places off .. end - 1 are the row's
    const int c0 = seg * a.chunks, c1 = min(c0 + a.chunks, (end + kChunk - 1) / kChunk);

    // (the token's logit comes with the others, not after them)
    int tok = -1;
    float logit = 0.f;
    if (tid == 0 && a.logprob) {
        tok = a.tokens[row];
        if (tok >= 0 && tok < a.vocab) logit = logit_at<DT>(a.logits, row * a.stride + tok);
    }
    if (tid == 0) n_cand = n_owner = 0;

    auto place = [&](int c, int j) { return c * kChunk + (j * kThreads + tid) * VEC; };   // of the thread's j-th word in a chunk
    // the word at place `at`, -inf for what is not the row's
    auto word = [&](int at) {
        u32x4v w;
        if (at >= off && at + VEC <= end) {
            w = *reinterpret_cast<const u32x4v*>(base + (size_t)at * ES);
        } else {
            uint32_t e[VEC];
#pragma unroll
            for (int i = 0; i < VEC; i++) {
                e[i] = ES == 4 ? 0xFF800000u : DT == GSDH_LOGITS_F16 ? 0xFC00u : 0xFF80u;
                if (at + i >= off && at + i < end) {
                    if constexpr (ES == 4) e[i] = reinterpret_cast<const uint32_t*>(base)[at + i];
                    else e[i] = reinterpret_cast<const uint16_t*>(base)[at + i];
                }
            }
#pragma unroll
            for (int i = 0; i < 4; i++) w[i] = ES == 4 ? e[i] : e[2 * i % VEC] | e[(2 * i + 1) % VEC] << 16;
        }
        return w;
    };
    auto load = [&](int c, u32x4v (&w)[kNV]) {
        if (c * kChunk >= off && (c + 1) * kChunk <= end) {
#pragma unroll
            for (int j = 0; j < kNV; j++) w[j] = *reinterpret_cast<const u32x4v*>(base + (size_t)place(c, j) * ES);
        } else {
#pragma unroll
            for (int j = 0; j < kNV; j++) w[j] = word(place(c, j));
        }
    };
    auto values = [](const u32x4v w, float (&x)[VEC]) {
#pragma unroll
        for (int i = 0; i < VEC; i++) {
            if constexpr (DT == GSDH_LOGITS_F32) x[i] = __uint_as_float(w[i]);
            else if constexpr (DT == GSDH_LOGITS_F16) x[i] = h2f((uint16_t)(w[i >> 1] >> (16 * (i & 1))));
            else x[i] = __uint_as_float(i & 1 ? w[i >> 1] & 0xFFFF0000u : w[i >> 1] << 16);
        }
    };

    float mx = -INFINITY, m = kLowest, s = 0.f, t = 0.f;
    int first = c0 < c1 ? place(c0, 0) : end;   // the word that mx first came in
    u32x4v next[kNV];
    if (c0 < c1) load(c0, next);
    for (int c = c0; c < c1; c++) {
        u32x4v w[kNV];
#pragma unroll
        for (int j = 0; j < kNV; j++) w[j] = next[j];
        if (c + 1 < c1) load(c + 1, next);
#pragma unroll
        for (int j = 0; j < kNV; j++) {
            float x[VEC];
            values(w[j], x);
            float top = x[0];
#pragma unroll
            for (int i = 1; i < VEC; i++) top = fmaxf(top, x[i]);
            first = top > mx ? place(c, j) : first;
            mx = fmaxf(mx, top);
        }
        const float to = fmaxf(mx, kLowest);
        if (__any(to > m)) {
            const float d = fmaxf(m - to, -1e30f), f = __builtin_amdgcn_exp2f(d * kLog2e);
            t = f * fmaf(d, s, t);
            s *= f;
            m = to;
        }
#pragma unroll
        for (int j = 0; j < kNV; j++) {
            float x[VEC];
            values(w[j], x);
#pragma unroll
            for (int i = 0; i < VEC; i++) {
                const float d = x[i] - m, p = __builtin_amdgcn_exp2f(d * kLog2e);
                s += p;
                t = fmaf(p, fmaxf(d, -1e30f), t);
            }
        }
    }

    // the segment's largest, the groups' keys
    float sm = wave_max(m);
    if (lane == 0) red[wid] = sm;
    uint64_t mine = 0;
    if (a.top) {
        // (a thread whose first word lies behind the row has none)
        if (first + VEC > off && first < end) mine = key_of(mx, first);
        const uint64_t of = quad_max(mine);
        if ((lane & 3) == 0) group[tid >> 2] = of;
    }
    __syncthreads();
    sm = red[0];
#pragma unroll
    for (int w = 1; w < kWavesOf; w++) sm = fmaxf(sm, red[w]);
    const float d = fmaxf(m - sm, -1e30f), f = __builtin_amdgcn_exp2f(d * kLog2e);
    t = wave_sum(f * fmaf(d, s, t));
    s = wave_sum(s * f);
    if (lane == 0) {
        red[kWavesOf + wid] = s;
        red[2 * kWavesOf + wid] = t;
    }
    if (a.top) {
        const uint64_t least = nth_largest(group, kGroups, a.top, partial);
        const float lv = value_of(least);
        const int li = least ? index_of(least) : end;   // (0: fewer groups than that have logits: all of them)
        if (mine >= least && mine) owner[atomicAdd(&n_owner, 1)] = (uint8_t)tid;
        __syncthreads();
        // their words, dealt to all threads
        const int owners = n_owner, words = owners * (c1 - c0) * kNV;
        for (int k = tid; k < words; k += kThreads) {
            const int j = k / owners, at = (c0 + j / kNV) * kChunk + (j % kNV * kThreads + owner[k % owners]) * VEC;
            float x[VEC];
            values(word(at), x);
#pragma unroll
            for (int i = 0; i < VEC; i++) {
                const float y = fmaxf(x[i], -INFINITY);
                if ((!least || y > lv || (y == lv && at <= li)) && at + i >= off && at + i < end) {
                    const int p = atomicAdd(&n_cand, 1);
                    if (p < kMaxCand) cand[p] = key_of(x[i], at + i - off);
                }
            }
        }
    }
    __syncthreads();
    m = sm;
    s = t = 0.f;
#pragma unroll
    for (int w = 0; w < kWavesOf; w++) {
        s += red[kWavesOf + w];
        t += red[2 * kWavesOf + w];
    }
    if (a.top) {
        if (n_cand <= kMaxCand) {
            select_top(cand, n_cand, a.top, best, partial);
        } else {
            // (more than are ranked at once, as where a few threads' logits outweigh
            // all others': the largest one by one, each below the one before.  61 rows of
            // 130001 in fp32, the largest at 8 threads of the 256, top 20: 71 us, not 14)
            uint64_t before = ~0ull;
            for (int r = 0; r < a.top; r++) {
                uint64_t most = 0;
                for (int c = c0; c < c1; c++)
                    for (int j = 0; j < kNV; j++)
                        for (int i = 0; i < VEC; i++) {
                            const int at = place(c, j) + i;
                            const uint64_t k = at >= off && at < end ? key_of(logit_at<DT>(base, at), at - off) : 0;
                            if (k < before && k > most) most = k;
                        }
#pragma unroll
                for (int d = 32; d >= 1; d >>= 1) most = shfl_max(most, d);
                if (lane == 0) group[wid] = most;
                __syncthreads();
                before = group[0];
                for (int w = 1; w < kWavesOf; w++) before = group[w] > before ? group[w] : before;
                if (tid == 0) best[r] = before;
                __syncthreads();
            }
        }
        __syncthreads();
    }
    if (a.nseg == 1) {
        finish_row(a, row, tok, logit, m, s, t, best);
        return;
    }

    // this segment's part; the block that arrives last has all of them
    const int64_t slot = (int64_t)row * a.nseg + seg;
    if (tid == 0) {
        put2(a.part + 4 * slot, m, s);
        put2(a.part + 4 * slot + 2, t, 0.f);
    }
    if (tid < a.top) __hip_atomic_store(&a.part_keys[slot * a.top + tid], best[tid], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    published();
    __syncthreads();
    if (tid == 0) {
        last = arrive(&a.counters[row], (unsigned)a.nseg);
        n_cand = 0;
    }
    __syncthreads();
    if (!last) return;
    // its segments' sums, and each one's k-th largest key, k = ceil(top / nseg):
    // ceil(top / k) of these have k keys each that are as large
    const float* part = a.part + (int64_t)row * a.nseg * 4;
    const uint64_t* keys = a.part_keys + (int64_t)row * a.nseg * a.top;
    const auto get = [&](int i) { return __hip_atomic_load(&keys[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); };
    const int k = (a.top + a.nseg - 1) / a.nseg;
    __shared__ float4 sums[kMaxSeg];
    // (all that is read here in one go: each of these loads takes a microsecond)
    const int own = min(tid, a.nseg - 1), all = a.nseg * a.top;
    uint64_t y[kHeld], kth = 0;
    const float2 p = get2(part + 4 * own), q = get2(part + 4 * own + 2);
    if (a.top) {
        kth = get(own * a.top + k - 1);
#pragma unroll
        for (int j = 0; j < kHeld; j++) y[j] = get(min(tid + j * kThreads, all - 1));
    }
    if (tid < a.nseg) {
        group[tid] = kth;
        sums[tid] = make_float4(p.x, p.y, q.x, 0.f);
    }
    __syncthreads();
    if (a.top) {
        const uint64_t least = nth_largest(group, a.nseg, (a.top + k - 1) / k, partial);
        const auto keep = [&](uint64_t x) {
            if (x != 0 && x >= least) cand[atomicAdd(&n_cand, 1)] = x;   // (at most top^2)
        };
#pragma unroll
        for (int j = 0; j < kHeld; j++)
            if (tid + j * kThreads < all) keep(y[j]);
        for (int i = tid + kHeld * kThreads; i < all; i += kThreads) keep(get(i));
    }
    float top = -INFINITY;
    for (int i = 0; i < a.nseg; i++) top = fmaxf(top, sums[i].x);
    s = t = 0.f;
    const float cm = top == -INFINITY ? 0.f : top;
    for (int i = 0; i < a.nseg; i++) {
        const float4 p = sums[i];
        const float d = fmaxf(p.x - cm, -1e30f), f = __builtin_amdgcn_exp2f(d * kLog2e);
        s += f * p.y;
        t += f * (p.z + d * p.y);
    }
    if (a.top) {
        __syncthreads();
        select_top(cand, n_cand, a.top, best, partial);
        __syncthreads();
    }
    finish_row(a, row, tok, logit, top, s, t, best);
}

// Segments of a row, and their chunks; `extra`: places ahead of a row that
// does not start at a 16-byte address.
struct Plan {
    int nseg, chunks;
};
Plan plan_of(int n, int vocab, int dtype, int extra) {
    const int chunks = (vocab + extra + chunk_of(dtype) - 1) / chunk_of(dtype);
    const int want = std::min(std::min((kBlocks + n - 1) / n, chunks), kMaxSeg), each = (chunks + want - 1) / want;
    return {(chunks + each - 1) / each, each};
}
// Partial results: of n rows of (kBlocks + n - 1) / n segments, which is the
// most that fewer rows have too, in rows of at least two chunks.
uint64_t logprob_space(int n, int vocab, int top) {
    if (vocab + 3 <= chunk_of(GSDH_LOGITS_F32)) return 0;
    const uint64_t rows = (uint64_t)std::min(n, kBlocks - 1);
    return counted_workspace(rows, (rows + kBlocks) * (16 + 8 * (uint64_t)top));
}

template <int DT>
hipError_t launch_logprobs(const LogprobArgs& a, int n, hipStream_t st) {
    hipLaunchKernelGGL(logprob_kernel<DT>, dim3((unsigned)(n * a.nseg)), dim3(kThreads), 0, st, a);
    return hipGetLastError();
}

bool logprob_shape(int n, int vocab, int top) {
    return n >= 0 && n <= (1 << 22) && vocab > 0 && vocab <= kMaxVocab && top >= 0 && top <= kMaxTop && top <= vocab;
}

}  // namespace

extern "C" {

uint64_t gsdh_token_logprobs_workspace_bytes(int n, int vocab, int top_n) {
    return logprob_shape(n, vocab, top_n) ? logprob_space(n, vocab, top_n) : 0;
}

int gsdh_token_logprobs(void* stream, const void* logits, int dtype, int64_t row_stride, int n, int vocab, const int* tokens,
                        int top_n, float* logprob, float* entropy, int* top_ids, float* top_logprobs, void* workspace,
                        uint64_t workspace_bytes) {
    const char* who = "token_logprobs";
    if (dtype < GSDH_LOGITS_F32 || dtype > GSDH_LOGITS_BF16) return fail(-1, "%s: logits type %d", who, dtype);
    if (!logprob_shape(n, vocab, top_n))
        return fail(-1, "%s: %d rows of %d logits, %d alternatives (at most 2^20 - 8 logits, 32 alternatives)", who, n, vocab, top_n);
    if (n > 1 && row_stride < vocab) return fail(-1, "%s: rows of %d logits %lld apart", who, vocab, (long long)row_stride);
    if (!tokens != !logprob) return fail(-1, "%s: tokens and logprob go together", who);
    if (top_n && (!top_ids || !top_logprobs)) return fail(-1, "%s: no buffers for %d alternatives", who, top_n);
    if (n == 0) return 0;
    if (!logits || reinterpret_cast<uintptr_t>(logits) % (dtype == GSDH_LOGITS_F32 ? 4 : 2))
        return fail(-1, "%s: logits null or not aligned to their type", who);
    const int es = dtype == GSDH_LOGITS_F32 ? 4 : 2;
    const bool aligned = reinterpret_cast<uintptr_t>(logits) % 16 == 0 && (n == 1 || row_stride * es % 16 == 0);
    const Plan p = plan_of(n, vocab, dtype, aligned ? 0 : 16 / es - 1);
    const int rc = check_workspace(workspace, workspace_bytes, logprob_space(n, vocab, top_n), who);
    if (rc) return rc;
    LogprobArgs a{};
    a.logits = logits; a.stride = row_stride; a.tokens = tokens; a.vocab = vocab; a.top = top_n; a.nseg = p.nseg; a.chunks = p.chunks;
    a.logprob = logprob; a.entropy = entropy; a.top_ids = top_ids; a.top_lp = top_logprobs;
    unsigned char* w = static_cast<unsigned char*>(workspace);
    a.counters = reinterpret_cast<unsigned*>(w);
    a.part = reinterpret_cast<float*>(w + counter_bytes(workspace_bytes));
    a.part_keys = reinterpret_cast<uint64_t*>(a.part + 4 * (size_t)n * p.nseg);
    if ((int64_t)n * p.nseg > 0x7FFFFFFF) return fail(-1, "%s: %d rows of %d logits in one call", who, n, vocab);
    hipStream_t st = static_cast<hipStream_t>(stream);
    GSD_PAGED_CHK(dtype == GSDH_LOGITS_F32 ? launch_logprobs<GSDH_LOGITS_F32>(a, n, st)
                  : dtype == GSDH_LOGITS_F16 ? launch_logprobs<GSDH_LOGITS_F16>(a, n, st)
                                             : launch_logprobs<GSDH_LOGITS_BF16>(a, n, st), who);
    return 0;
}

}  // extern "C"
