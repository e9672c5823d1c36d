// gsd_logits.hip -- what is done to rows of logits before a token is chosen:
// penalties for repeated tokens, biases, grammar masks.
#include "gsd_device.h"
#include "gsd_paged.h"

using namespace gsd;

namespace {

constexpr int kThreads = 256;
constexpr int kSeg = 4096;               // logits of a block, a word of LDS each
constexpr int kMaxVocab = 1 << 24;
constexpr int kMaxList = 1 << 30;         // tokens of a row's history; biases
constexpr int kHeld = 2;                 // times four tokens of the history that a thread has on their way
constexpr uint32_t kInPrompt = 1u << 31;   // in a logit's word, beside how often the answer has it

struct RulesArgs {
    gsdh_logit_rules r;
    const void* x;
    void* out;
    int64_t x_stride, out_stride;
    int vocab, nseg, in_place;
};

// Rows of logits start at any element: words of 16 bytes, aligned to the element.
template <typename T>
struct Word {
    static constexpr int N = 16 / sizeof(T);
    typedef T type __attribute__((ext_vector_type(16 / sizeof(T)), aligned(sizeof(T))));
};

// A logit x of token v becomes
//   x / r where x > 0, else x r        if v occurs in the history (r: repetition)
//   - frequency * count - presence     if it occurs in the answer, count times
//   + bias
//   -inf                               if the mask forbids it
//
// A block has 4096 logits of a row and a word of LDS for each: it goes through
// the whole history and counts what lies in its range by LDS atomics (integers:
// no order changes them), then through the biases, of which a token's last one
// counts (the greatest place in the list wins).  The lists are asked for first, then a
// thread's logits, 16 bytes at a time; those that a mask forbids are not read at all.
//
// Bound by the chain lengths -> lists -> LDS -> logits: one row of 32768 fp32 logits with
// a history of 900 6.6 us, 61 rows of 130001 bf16 logits with histories of up to 8000
// (23 MB) 13.5 us; then by memory: 256 rows of 32768 fp32 logits (48 MB) 16.0 us, 3.0
// TB/s.  (A token of the history per load, after the logits: 19.0 and 17.0 us; counts and
// places in LDS of their own leave room for 5 blocks per CU in place of 8: 16.3 and 21.4;
// 16 tokens of a thread on their way in place of 8: 13.8 and 18.7; blocks of 1024 threads
// and 16384 logits, which read a history less often: 12.5, but 16.4 and 7.3 for one row.)
template <typename T>
__global__ void __launch_bounds__(kThreads, 8) rules_kernel(const RulesArgs a) {
    typedef Word<T> W;
    constexpr int N = W::N, NW = kSeg / kThreads / N;   // logits of a word, words of a thread
    __shared__ __attribute__((aligned(16))) uint32_t lds[kSeg];   // counts, then places among the biases
    const int row = (int)(blockIdx.x / (unsigned)a.nseg), v0 = (int)(blockIdx.x % (unsigned)a.nseg) * kSeg, tid = threadIdx.x;
    const T* const x = static_cast<const T*>(a.x) + (int64_t)row * a.x_stride;
    T* const out = static_cast<T*>(a.out) + (int64_t)row * a.out_stride;

    int seen = a.r.history ? a.r.history_lens[row] : 0, prompt = a.r.history && a.r.prompt_lens ? a.r.prompt_lens[row] : 0;
    int b0 = a.r.bias_starts ? a.r.bias_starts[row] : 0, b1 = a.r.bias_starts ? a.r.bias_starts[row + 1] : 0;
    const int mask = a.r.masks ? a.r.mask_rows[row] : -1;
    const bool bad = seen < 0 || seen > a.r.history_width || b0 < 0 || b1 < b0 || b1 > a.r.n_bias || mask < -1 || (mask >= 0 && mask >= a.r.n_masks);
    if (bad) seen = b0 = b1 = 0;

    // the history, four tokens at a time: kHeld of them are on their way at once
    typedef int int4u __attribute__((ext_vector_type(4), aligned(4)));
    const int* const history = a.r.history + (int64_t)row * a.r.history_width;
    int4u held[kHeld];
    auto load_history = [&](int from) {
#pragma unroll
        for (int k = 0; k < kHeld; k++) {
            const int i = from + 4 * (k * kThreads + tid);
            held[k] = int4u{-1, -1, -1, -1};
            if (i + 4 <= seen) {
                held[k] = *reinterpret_cast<const int4u*>(history + i);
            } else {
#pragma unroll
                for (int e = 0; e < 3; e++)
                    if (i + e < seen) held[k][e] = history[i + e];
            }
        }
    };
    load_history(0);
    const int bias_id = b0 + tid < b1 ? a.r.bias_ids[b0 + tid] : -1;

    // what the mask allows of a thread's words, and these words
    uint32_t allowed[NW];
    float y[NW][N];
    auto at = [&](int i) { return v0 + (i * kThreads + tid) * N; };
#pragma unroll
    for (int i = 0; i < NW; i++) {
        const int left = a.vocab - at(i);
        allowed[i] = left >= N ? (1u << N) - 1 : left > 0 ? (1u << left) - 1 : 0;
        if (mask >= 0 && !bad && allowed[i]) allowed[i] &= a.r.masks[(int64_t)mask * a.r.mask_words + at(i) / 32] >> (at(i) % 32);
    }
    auto load = [&](int i) {
        if (at(i) + N <= a.vocab) {
            const typename W::type w = *reinterpret_cast<const typename W::type*>(x + at(i));
#pragma unroll
            for (int e = 0; e < N; e++) y[i][e] = (float)w[e];
        } else {
#pragma unroll
            for (int e = 0; e < N; e++) y[i][e] = allowed[i] >> e & 1 ? (float)x[at(i) + e] : 0.f;
        }
    };
    if (!a.in_place)
#pragma unroll
        for (int i = 0; i < NW; i++)
            if (allowed[i]) load(i);

    uint32_t came[NW] = {};   // in place: words that came in
    auto clear = [&] {
#pragma unroll
        for (int i = 0; i < kSeg / kThreads / 4; i++) *reinterpret_cast<uint4*>(lds + 4 * (i * kThreads + tid)) = make_uint4(0u, 0u, 0u, 0u);
    };
    auto word_of = [&](int i, uint32_t (&w)[N]) {   // of LDS; whether any is not 0
        uint32_t any = 0;
#pragma unroll
        for (int e = 0; e < N; e += 4) {
            const uint4 u = *reinterpret_cast<const uint4*>(lds + (i * kThreads + tid) * N + e);
            w[e] = u.x; w[e + 1] = u.y; w[e + 2] = u.z; w[e + 3] = u.w;
            any |= u.x | u.y | u.z | u.w;
        }
        return any != 0;
    };
    if (seen) {
        clear();
        lds_barrier();
        for (int from = 0; from < seen; from += 4 * kHeld * kThreads) {
            if (from) load_history(from);
#pragma unroll
            for (int k = 0; k < kHeld; k++) {
                const int i = from + 4 * (k * kThreads + tid);
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const unsigned v = (unsigned)held[k][e] - (unsigned)v0;   // (-1 is no token of any range)
                    if (v < (unsigned)kSeg) {
                        if (i + e < prompt) atomicOr(&lds[v], kInPrompt);
                        else atomicAdd(&lds[v], 1u);
                    }
                }
            }
        }
        const float rep = a.r.repetition ? a.r.repetition[row] : 1.f, freq = a.r.frequency ? a.r.frequency[row] : 0.f,
                    pres = a.r.presence ? a.r.presence[row] : 0.f;
        lds_barrier();
#pragma unroll
        for (int i = 0; i < NW; i++) {
            uint32_t w[N];
            if (!allowed[i] || !word_of(i, w)) continue;
            if (a.in_place) {
                load(i);
                came[i] = 1;
            }
#pragma unroll
            for (int e = 0; e < N; e++) {
                if (!w[e]) continue;
                float z = y[i][e];
                if (a.r.repetition) z = z > 0.f ? z / rep : z * rep;
                const uint32_t count = w[e] & ~kInPrompt;
                if (count) {
                    if (a.r.frequency) z -= freq * (float)count;
                    if (a.r.presence) z -= pres;
                }
                y[i][e] = z;
            }
        }
        if (b1 > b0) lds_barrier();   // (the counts are read)
    }
    if (b1 > b0) {
        clear();
        lds_barrier();
        for (int i = b0 + tid; i < b1; i += kThreads) {
            const unsigned v = (unsigned)(i < b0 + kThreads ? bias_id : a.r.bias_ids[i]) - (unsigned)v0;
            if (v < (unsigned)kSeg) atomicMax(&lds[v], (uint32_t)(i - b0) + 1u);
        }
        lds_barrier();
#pragma unroll
        for (int i = 0; i < NW; i++) {
            uint32_t w[N];
            if (!allowed[i] || !word_of(i, w)) continue;
            if (a.in_place && !came[i]) {
                load(i);
                came[i] = 1;
            }
#pragma unroll
            for (int e = 0; e < N; e++)
                if (w[e] && at(i) + e < a.vocab) y[i][e] += a.r.bias[b0 + (int)w[e] - 1];
        }
    }
#pragma unroll
    for (int i = 0; i < NW; i++) {
        const int left = a.vocab - at(i);
        if (left <= 0) continue;
        const uint32_t whole = left >= N ? (1u << N) - 1 : (1u << left) - 1;
        if (a.in_place && !bad && !came[i]) {
            if ((allowed[i] & whole) == whole) continue;   // nothing of it changes
            if (allowed[i] & whole) load(i);
        }
        float z[N];
#pragma unroll
        for (int e = 0; e < N; e++) z[e] = bad ? __builtin_nanf("") : allowed[i] >> e & 1 ? y[i][e] : -INFINITY;
        if (left >= N) {
            typename W::type w;
#pragma unroll
            for (int e = 0; e < N; e++) w[e] = (T)z[e];
            *reinterpret_cast<typename W::type*>(out + at(i)) = w;
        } else {
#pragma unroll
            for (int e = 0; e < N; e++)
                if (e < left) out[at(i) + e] = (T)z[e];
        }
    }
}

}  // namespace

extern "C" {

int gsdh_logits_adjust(void* stream, const gsdh_logit_rules* r, const void* x, int dtype, int64_t x_stride, int n, int vocab, void* out,
                       int64_t out_stride) {
    const char* who = "logits_adjust";
    if (!r) return fail(-1, "%s: null rules", who);
    if (dtype < GSDH_LOGITS_F32 || dtype > GSDH_LOGITS_BF16) return fail(-1, "%s: type %d", who, dtype);
    if (n < 0) return fail(-1, "%s: %d rows", who, n);
    if (vocab <= 0 || vocab > kMaxVocab) return fail(-1, "%s: rows of %d logits (at most %d)", who, vocab, kMaxVocab);
    if (out_stride < vocab || x_stride < 0 || (x == out && x_stride != out_stride))
        return fail(-1, "%s: rows %lld and %lld apart, of %d logits", who, (long long)x_stride, (long long)out_stride, vocab);
    if (r->history && (!r->history_lens || r->history_width < 0))
        return fail(-1, "%s: a history needs lengths and a width, has %d", who, r->history_width);
    if (!r->history && (r->repetition || r->frequency || r->presence)) return fail(-1, "%s: penalties need a history", who);
    if (r->history && r->history_width > kMaxList) return fail(-1, "%s: a history of %d tokens (at most 2^30)", who, r->history_width);
    if (r->bias_starts && r->n_bias > kMaxList) return fail(-1, "%s: %d biases (at most 2^30)", who, r->n_bias);
    if (r->bias_starts ? !r->bias_ids || !r->bias || r->n_bias < 0 : r->bias_ids || r->bias)
        return fail(-1, "%s: bias_starts, bias_ids and bias go together", who);
    if (r->masks ? !r->mask_rows || r->n_masks < 0 || (int64_t)r->mask_words * 32 < vocab : r->mask_rows != nullptr)
        return fail(-1, "%s: masks need mask_rows and words for %d logits, have %d", who, vocab, r->mask_words);
    if (n == 0) return 0;
    const uintptr_t es = dtype == GSDH_LOGITS_F32 ? 4 : 2;
    if (!x || !out || reinterpret_cast<uintptr_t>(x) % es || reinterpret_cast<uintptr_t>(out) % es)
        return fail(-1, "%s: logits null or not aligned to their type", who);
    RulesArgs a{};
    a.r = *r;
    a.x = x; a.x_stride = x_stride; a.out = out; a.out_stride = out_stride; a.vocab = vocab; a.in_place = x == out;
    a.nseg = (vocab + kSeg - 1) / kSeg;
    if ((int64_t)n * a.nseg > 0x7FFFFFFF) return fail(-1, "%s: %d rows of %d logits in one call", who, n, vocab);
    const dim3 grid((unsigned)(n * a.nseg)), block(kThreads);
    hipStream_t st = static_cast<hipStream_t>(stream);
    switch (dtype) {
        case GSDH_LOGITS_F32: hipLaunchKernelGGL(rules_kernel<float>, grid, block, 0, st, a); break;
        case GSDH_LOGITS_F16: hipLaunchKernelGGL(rules_kernel<_Float16>, grid, block, 0, st, a); break;
        default: hipLaunchKernelGGL(rules_kernel<__bf16>, grid, block, 0, st, a); break;
    }
    GSD_PAGED_CHK(hipGetLastError(), who);
    return 0;
}

}  // extern "C"
