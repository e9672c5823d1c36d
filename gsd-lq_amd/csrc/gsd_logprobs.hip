// gsd_logprobs.hip -- log probabilities of given tokens, entropy and the
// largest alternatives of rows of logits, each logit read once.
#include <algorithm>

#include "gsd_device.h"
#include "gsd_paged.h"

using namespace gsd;

namespace {

constexpr int kThreads = 256;
constexpr int kGroups = 64;         // of four threads; a row has at most twice as many segments
constexpr int kMaxTop = 32;
constexpr int kMaxVocab = (1 << 20) - 8;   // 128 segments of 8192 at most, wherever the row starts
constexpr int kMaxCand = 4096;      // keys that may reach a threshold (below)
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
    int vocab, top, nseg;
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

// The `want`-th largest of the first `count` (<= 128) keys of lds (0: fewer
// nonzero ones than that), by counting for each how many are larger.  Each
// wave computes it for itself; nonzero keys differ.
__device__ uint64_t nth_largest(const uint64_t* keys, int count, int want) {
    const int lane = threadIdx.x & 63;
    uint64_t found = 0;
    for (int base = 0; base < count; base += 64) {
        const uint64_t mine = base + lane < count ? keys[base + lane] : 0;
        int above = 0;
        for (int i = 0; i < count; i++) above += keys[i] > mine;
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
__device__ void select_top(const uint64_t* cand, int count, int top, uint64_t* out) {
    for (int i = count + (int)threadIdx.x; i < top; i += kThreads) out[i] = 0;
    for (int i = threadIdx.x; i < count; i += kThreads) {
        const uint64_t mine = cand[i];
        int above = 0;
        for (int j = 0; j < count; j++) above += cand[j] > mine;
        if (above < top) out[above] = mine;
    }
}

// The row's results from its sums (m, s, t) and its largest keys (LDS).
template <int DT>
__device__ void finish_row(const LogprobArgs& a, int row, float m, float s, float t, const uint64_t* keys) {
    const float log_s = __builtin_amdgcn_logf(s) * kLn2;
    // (m is -inf where nothing has probability, and s NaN where a logit was NaN or +inf)
    const bool none = !(s > 0.f) || m == -INFINITY;
    if (threadIdx.x == 0) {
        if (a.logprob) {
            const int tok = a.tokens[row];
            float v = __builtin_nanf("");
            if (tok == -1) v = 0.f;
            else if (tok >= 0 && tok < a.vocab && !none) v = (logit_at<DT>(a.logits, row * a.stride + tok) - m) - log_s;
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

// One block: a segment of kThreads * E logits of a row, held in registers.
//
//   m = max x,  s = sum e^(x - m),  t = sum e^(x - m) (x - m)
//   ln p = x - m - ln s,  entropy = ln s - t / s   (no cancellation: both terms are >= 0)
//
// The largest `top`: 64 groups of four threads each take the largest key of
// theirs; `top` groups reach the top-th largest of these 64, so at most
// 4 E top logits do (some `top` more of ordinary rows), and these are ranked
// by counting.  A row of several segments is joined by the block that arrives
// last.  Logits are read in 16-byte words from the aligned address at or
// below the row's first, those of a row's edges one by one.
template <int DT, int E>
__global__ void __launch_bounds__(kThreads) logprob_kernel(const LogprobArgs a) {
    constexpr int VEC = DT == GSDH_LOGITS_F32 ? 4 : 8, NV = E / VEC, ES = DT == GSDH_LOGITS_F32 ? 4 : 2;
    __shared__ float red[3 * (kThreads / 64)];
    __shared__ uint64_t group[2 * kGroups], best[kMaxTop], cand[kMaxCand];
    __shared__ int n_cand, last;
    const int row = blockIdx.x / a.nseg, seg = blockIdx.x % a.nseg, tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
    const unsigned char* base = static_cast<const unsigned char*>(a.logits) + row * a.stride * ES;
    const int off = (int)(reinterpret_cast<uintptr_t>(base) % 16) / ES;   // logits between the aligned address and the row
    base -= off * ES;
    const int end = off + a.vocab;   // places off .. end - 1 are the row's

    float x[E];
#pragma unroll
    for (int j = 0; j < NV; j++) {
        const int at = seg * kThreads * E + (j * kThreads + tid) * VEC;
        if (at >= off && at + VEC <= end) {
            const uint4 w = *reinterpret_cast<const uint4*>(base + (size_t)at * ES);
            const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int e = 0; e < VEC; e++) {
                if constexpr (DT == GSDH_LOGITS_F32) x[j * VEC + e] = __uint_as_float(u[e]);
                else if constexpr (DT == GSDH_LOGITS_F16) x[j * VEC + e] = h2f((uint16_t)(u[e >> 1] >> (16 * (e & 1))));
                else x[j * VEC + e] = __uint_as_float(e & 1 ? u[e >> 1] & 0xFFFF0000u : u[e >> 1] << 16);
            }
        } else {
#pragma unroll
            for (int e = 0; e < VEC; e++)
                x[j * VEC + e] = at + e >= off && at + e < end ? logit_at<DT>(base, at + e) : -INFINITY;
        }
    }

    float mx = -INFINITY;
#pragma unroll
    for (int e = 0; e < E; e++) mx = fmaxf(mx, x[e]);
    const float wmx = wave_max(mx);
    if (lane == 0) red[wid] = wmx;
    if (tid == 0) n_cand = 0;

    // the largest key of the thread, then of its group
    if (a.top) {
        uint64_t mine = 0;
        auto place = [&](int e) { return seg * kThreads * E + ((e / VEC) * kThreads + tid) * VEC + e % VEC; };
        if (mx > -INFINITY) {
            int at = 0;
#pragma unroll
            for (int e = E - 1; e >= 0; e--) at = x[e] == mx ? place(e) : at;
            mine = key_of(mx, at - off);
        } else {
            // nothing above -inf: the first place that is the row's
            for (int e = E - 1; e >= 0; e--)
                if (place(e) >= off && place(e) < end) mine = key_of(-INFINITY, place(e) - off);
        }
        mine = shfl_max(mine, 1);
        mine = shfl_max(mine, 2);
        if ((lane & 3) == 0) group[tid >> 2] = mine;
    }
    __syncthreads();
    float m = red[0];
#pragma unroll
    for (int w = 1; w < kThreads / 64; w++) m = fmaxf(m, red[w]);
    __syncthreads();

    if (a.top) {
        const uint64_t least = nth_largest(group, kGroups, a.top);
        const float lv = value_of(least);
#pragma unroll
        for (int e = 0; e < E; e++) {
            if (least == 0 || fmaxf(x[e], -INFINITY) >= lv) {
                const int at = seg * kThreads * E + ((e / VEC) * kThreads + tid) * VEC + e % VEC;
                const uint64_t k = key_of(x[e], at - off);
                if (k >= least && at >= off && at < end) {
                    const int p = atomicAdd(&n_cand, 1);
                    if (p < kMaxCand) cand[p] = k;
                }
            }
        }
    }

    float s = 0.f, t = 0.f;
    const float c = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int e = 0; e < E; e++) {
        const float d = x[e] - c, p = __builtin_amdgcn_exp2f(d * kLog2e);
        s += p;
        t = fmaf(p, fmaxf(d, -1e30f), t);
    }
    s = wave_sum(s);
    t = wave_sum(t);
    if (lane == 0) {
        red[(kThreads / 64) + wid] = s;
        red[2 * (kThreads / 64) + wid] = t;
    }
    __syncthreads();
    s = t = 0.f;
#pragma unroll
    for (int w = 0; w < kThreads / 64; w++) {
        s += red[(kThreads / 64) + w];
        t += red[2 * (kThreads / 64) + w];
    }
    if (a.top) {
        select_top(cand, min(n_cand, kMaxCand), a.top, best);
        __syncthreads();
    }
    if (a.nseg == 1) {
        finish_row<DT>(a, row, m, s, t, best);
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
    const float* part = a.part + (int64_t)row * a.nseg * 4;
    __shared__ float4 sums[2 * kGroups];
    for (int i = tid; i < a.nseg; i += kThreads) {
        const float2 p = get2(part + 4 * i), q = get2(part + 4 * i + 2);
        sums[i] = make_float4(p.x, p.y, q.x, 0.f);
    }
    __syncthreads();
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
        // each segment's k-th largest, k = ceil(top / nseg): k times the ceil(top / k)
        // largest of these are `top` at least
        const uint64_t* keys = a.part_keys + (int64_t)row * a.nseg * a.top;
        const int k = (a.top + a.nseg - 1) / a.nseg;
        const auto get = [&](int i) { return __hip_atomic_load(&keys[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); };
        for (int i = tid; i < a.nseg; i += kThreads) group[i] = get(i * a.top + k - 1);
        __syncthreads();
        const uint64_t least = nth_largest(group, a.nseg, (a.top + k - 1) / k);
        for (int i = tid; i < a.nseg * a.top; i += kThreads) {
            const uint64_t y = get(i);
            if (y != 0 && y >= least) {
                const int p = atomicAdd(&n_cand, 1);
                if (p < kMaxCand) cand[p] = y;
            }
        }
        __syncthreads();
        select_top(cand, min(n_cand, kMaxCand), a.top, best);
        __syncthreads();
    }
    finish_row<DT>(a, row, top, s, t, best);
}

// Logits of a thread: 32 where the rows fill the chip, else 8, as long as the
// join of a row's segments stays within its candidates.
struct Plan {
    int e, nseg;
};
Plan plan_of(int n, int vocab, int top) {
    Plan p{32, (vocab + 7 + kThreads * 32 - 1) / (kThreads * 32)};
    const int small = (vocab + 7 + kThreads * 8 - 1) / (kThreads * 8);
    if ((int64_t)n * p.nseg < 512 && small * top <= kMaxCand && small <= 2 * kGroups) p = {8, small};
    return p;
}
// bytes of the partial results of n rows, and of a workspace that holds them
size_t parts_of(int n, const Plan& p, int top) { return p.nseg == 1 ? 0 : (size_t)n * p.nseg * (16 + 8 * (size_t)top); }
uint64_t space_for(int n, const Plan& p, int top) { return p.nseg == 1 ? 0 : counted_workspace((uint64_t)n, parts_of(n, p, top)); }

template <int DT>
hipError_t launch_logprobs(const LogprobArgs& a, int n, int e, hipStream_t st) {
    const dim3 grid((unsigned)(n * a.nseg)), block(kThreads);
    if (e == 32) hipLaunchKernelGGL((logprob_kernel<DT, 32>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((logprob_kernel<DT, 8>), grid, block, 0, st, a);
    return hipGetLastError();
}

bool logprob_shape(int n, int vocab, int top) {
    return n >= 0 && n <= (1 << 22) && vocab > 0 && vocab <= kMaxVocab && top >= 0 && top <= kMaxTop && top <= vocab;
}

}  // namespace

extern "C" {

uint64_t gsdh_token_logprobs_workspace_bytes(int n, int vocab, int top_n) {
    if (!logprob_shape(n, vocab, top_n)) return 0;
    // (fewer rows may take more segments each)
    uint64_t most = space_for(n, plan_of(n, vocab, top_n), top_n);
    const Plan few = plan_of(1, vocab, top_n), many = plan_of(1 << 20, vocab, top_n);
    if (few.nseg != many.nseg) {
        const int rows = std::min(n, 511 / many.nseg);
        if (rows > 0) most = std::max(most, space_for(rows, few, top_n));
    }
    return most;
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
    const Plan p = plan_of(n, vocab, top_n);
    const int rc = check_workspace(workspace, workspace_bytes, space_for(n, p, top_n), who);
    if (rc) return rc;
    LogprobArgs a{};
    a.logits = logits; a.stride = row_stride; a.tokens = tokens; a.vocab = vocab; a.top = top_n; a.nseg = p.nseg;
    a.logprob = logprob; a.entropy = entropy; a.top_ids = top_ids; a.top_lp = top_logprobs;
    unsigned char* w = static_cast<unsigned char*>(workspace);
    a.counters = reinterpret_cast<unsigned*>(w);
    a.part = reinterpret_cast<float*>(w + counter_bytes(workspace_bytes));
    a.part_keys = reinterpret_cast<uint64_t*>(a.part + 4 * (size_t)n * p.nseg);
    if ((int64_t)n * p.nseg > 0x7FFFFFFF) return fail(-1, "%s: %d rows of %d logits in one call", who, n, vocab);
    hipStream_t st = static_cast<hipStream_t>(stream);
    GSD_PAGED_CHK(dtype == GSDH_LOGITS_F32 ? launch_logprobs<GSDH_LOGITS_F32>(a, n, p.e, st)
                  : dtype == GSDH_LOGITS_F16 ? launch_logprobs<GSDH_LOGITS_F16>(a, n, p.e, st)
                                             : launch_logprobs<GSDH_LOGITS_BF16>(a, n, p.e, st), who);
    return 0;
}

}  // extern "C"
