// gsd_pages.hip -- pages of the paged KV cache: taken, forked, freed,
// compacted and copied, all on the device.
//
// The bookkeeping (refs, tables, lens: a few hundred KB at most) is one
// block's work: its order decides which page a sequence gets, and a block
// can keep that order with barriers instead of launches: a chain of loads of
// 3 us (take) to 6 (fork, compact) on pools of 216 and 372 pages.  Counts are
// looked at 8192 pages a step, about 1 us, one step after another: take on 131072
// pages of which the lowest nine tenths are in use 18 us, compact's two passes with
// 11700 pages freed 110 us.  What moves rows runs over the whole chip and is bound by
// memory (5 TB/s read and written; 200 pages of 2 MB copied, 839 MB moved: 149 us).
#include <algorithm>

#include "gsd_device.h"
#include "gsd_paged.h"

using namespace gsd;

namespace {

constexpr int kPlan = 1024;         // threads of a planning block
constexpr int kRun = 8;             // words of refs a thread looks at per step
constexpr int kPlanWaves = kPlan / 64;

// workspace words: header, then lists
constexpr int kMoves = 0, kUsed = 1, kFirst = 2, kHead = 4;   // moves, pages in use, the first source in its list

struct Space {
    size_t src, dst, map, plan, words;   // offsets in ints
};
Space space_of(const gsdh_paged_cache& c) {
    Space s;
    const size_t np = ((size_t)c.n_pages + 3) / 4 * 4;
    s.src = kHead;
    s.dst = s.src + np;
    s.map = s.dst + np;
    s.plan = s.map + np;
    s.words = s.plan + 4 * (size_t)c.n_seqs;
    return s;
}

// Exclusive sum over the block in thread order; *total gets the sum.
// lds: kPlanWaves ints.  All threads take part.
__device__ int block_scan(int v, int* lds, int* total) {
    const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
    int incl = v;
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) {
        const int b = __shfl_up(incl, s, 64);
        if (lane >= s) incl += b;
    }
    __syncthreads();
    if (lane == 63) lds[wid] = incl;
    __syncthreads();
    int before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kPlanWaves; w++) {
        before += w < wid ? lds[w] : 0;
        all += lds[w];
    }
    *total = all;
    return before + incl - v;
}

// Every page i in rising order of i: f(i, whether pred(refs[i]), how many
// before it have pred) until `stop` of them were seen (a whole step of pages
// more may be looked at); returns how many.  Order and counts come from
// ballots, a step is kPlan * kRun pages.  lds: kRun * kPlanWaves ints.
template <typename Pred, typename F>
__device__ int scan_pages(const int* refs, int n, int stop, int* lds, Pred pred, F f) {
    const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
    int seen = 0;
    for (int base = 0; base < n && seen < stop; base += kPlan * kRun) {
        unsigned long long mask[kRun];
        int ref[kRun];
#pragma unroll
        for (int j = 0; j < kRun; j++) {
            const int i = base + j * kPlan + (int)threadIdx.x;
            ref[j] = i < n ? refs[i] : -1;
        }
#pragma unroll
        for (int j = 0; j < kRun; j++) {
            const int i = base + j * kPlan + (int)threadIdx.x;
            mask[j] = __ballot(i < n && pred(ref[j], i));
            if (lane == 0) lds[j * kPlanWaves + wid] = __popcll(mask[j]);
        }
        __syncthreads();
        // the counts' sums up to each, two to a lane, by every wave for itself
        static_assert(kRun * kPlanWaves == 128, "two counts a lane");
        const int2 two = reinterpret_cast<const int2*>(lds)[lane];
        int incl = two.x + two.y;
#pragma unroll
        for (int s = 1; s < 64; s <<= 1) {
            const int b = __shfl_up(incl, s, 64);
            if (lane >= s) incl += b;
        }
        const int sum = __builtin_amdgcn_readlane(incl, 63);
        int before[kRun];
#pragma unroll
        for (int j = 0; j < kRun; j++) {
            const int at = j * kPlanWaves + wid;   // (the pair of counts that this one is in)
            const int upto = __shfl(incl, at >> 1, 64), lo = __shfl(two.x, at >> 1, 64), hi = __shfl(two.y, at >> 1, 64);
            before[j] = at & 1 ? upto - hi : upto - hi - lo;
        }
        __syncthreads();   // (the counts are read)
        const unsigned long long below = (1ull << lane) - 1ull;
#pragma unroll
        for (int j = 0; j < kRun; j++) {
            const int i = base + j * kPlan + (int)threadIdx.x;
            if (i < n) f(i, ((mask[j] >> lane) & 1ull) != 0, seen + before[j] + __popcll(mask[j] & below));
        }
        seen += sum;
    }
    __syncthreads();
    return seen;
}

__device__ __forceinline__ int pages_for(const gsdh_paged_cache& c, int len) { return (len + c.page_size - 1) / c.page_size; }
// a length that the tables can hold
__device__ __forceinline__ bool len_ok(const gsdh_paged_cache& c, int len) { return len >= 0 && len <= c.table_width * c.page_size; }

// The last index of off[0 .. n) (not falling, off[0] <= k) whose value is at most k
__device__ __forceinline__ int owner_of(const int* off, int n, int k) {
    int lo = 0, hi = n - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (off[mid] <= k) lo = mid; else hi = mid - 1;
    }
    return lo;
}

// first[s] = the first place in the list that names sequence s; `own`: list[threadIdx.x]
__device__ __forceinline__ void first_of(const gsdh_paged_cache& c, const int* list, int own, int n, int* first) {
    for (int s = threadIdx.x; s < c.n_seqs; s += kPlan) first[s] = 0x7FFFFFFF;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kPlan) {
        const int s = i < kPlan ? own : list[i];
        if (s >= 0 && s < c.n_seqs) atomicMin(&first[s], i);
    }
    __syncthreads();
}

// dynamic LDS of a planning block: the scans' words, first[n_seqs], off[n]
size_t plan_lds(const gsdh_paged_cache& c, int n) { return 4 * ((size_t)c.n_seqs + n + kRun * kPlanWaves + kPlanWaves); }

__global__ void __launch_bounds__(kPlan) pages_take_kernel(const gsdh_paged_cache c, const int* seqs, const int* counts, int n) {
    extern __shared__ __align__(16) int lds[];
    int *words = lds, *scan = words + kRun * kPlanWaves, *first = scan + kPlanWaves, *off = first + c.n_seqs;
    // (the thread's own entry, all there is of lists up to kPlan, is read ahead:
    // the launch is a chain of dependent loads)
    const int tid = threadIdx.x, s0 = tid < n ? seqs[tid] : -1, k0 = tid < n ? counts[tid] : 0;
    const int len0 = s0 >= 0 && s0 < c.n_seqs ? c.lens[s0] : 0;
    first_of(c, seqs, s0, n, first);
    // how many pages each wants: -1 in the list's place of one that is left out
    auto want = [&](int i, uint32_t* bad) {
        const int s = i < kPlan ? s0 : seqs[i], k = i < kPlan ? k0 : counts[i];
        if (s < 0 || s >= c.n_seqs || k < 0) { *bad |= GSDH_PAGES_BAD_INDEX; return -1; }
        if (first[s] != i) { *bad |= GSDH_PAGES_TWICE; return -1; }
        const int len = i < kPlan ? len0 : c.lens[s];
        if (!len_ok(c, len) || k > c.table_width * c.page_size - len) { *bad |= GSDH_PAGES_BAD_INDEX; return -1; }
        return pages_for(c, len + k) - pages_for(c, len);   // (beyond the pool: cannot be met)
    };
    uint32_t bad = 0;
    int total = 0;
    for (int base = 0; base < n; base += kPlan) {
        const int i = base + (int)threadIdx.x;
        const int k = i < n ? min(max(want(i, &bad), 0), c.n_pages + 1) : 0;
        int sum;
        const int at = block_scan(k, scan, &sum);
        // (a sum beyond the pool's pages cannot be met, and stays there: what
        // kPlan entries add, at most 2^20 + 1 each, would pass 32 bits in the end)
        if (i < n) off[i] = (int)min((unsigned)total + (unsigned)at, 0x3FFFFFFFu);
        total = (int)min((unsigned)total + (unsigned)sum, 0x3FFFFFFFu);
    }
    __syncthreads();
    const int found = scan_pages(c.refs, c.n_pages, total, words, [](int r, int) { return r == 0; },
        [&](int page, bool free_, int rank) {
            if (!free_ || rank >= total) return;
            const int i = owner_of(off, n, rank), s = seqs[i];
            c.tables[(size_t)s * c.table_width + pages_for(c, c.lens[s]) + rank - off[i]] = page;
            c.refs[page] = 1;
        });
    for (int i = threadIdx.x; i < n; i += kPlan) {
        uint32_t none = 0;
        const int k = want(i, &none);
        if (k < 0) continue;
        const int s = i < kPlan ? s0 : seqs[i], len = i < kPlan ? len0 : c.lens[s];
        if (k > 0 && off[i] + k > found) {
            bad |= GSDH_PAGES_EXHAUSTED;
            // the pages there were for the first one that does not fit
            int* t = c.tables + (size_t)s * c.table_width + pages_for(c, len);
            for (int j = 0; j < min(found - off[i], k); j++) {
                c.refs[t[j]] = 0;
                t[j] = -1;
            }
        } else {
            c.lens[s] = len + (i < kPlan ? k0 : counts[i]);
        }
    }
    if (bad) page_status(c, bad);
}

// A fork's plan per list entry, in the workspace: source, destination (-1:
// left out), positions, the page taken for the last partly filled one (-1: none)
__global__ void __launch_bounds__(kPlan) pages_fork_kernel(const gsdh_paged_cache c, const int* src, const int* dst, int n, int4* plan) {
    extern __shared__ __align__(16) int lds[];
    int *words = lds, *scan = words + kRun * kPlanWaves, *first = scan + kPlanWaves, *off = first + c.n_seqs;
    const int tid = threadIdx.x, a0 = tid < n ? src[tid] : -1, b0 = tid < n ? dst[tid] : -1;   // (as in pages_take_kernel)
    const int alen0 = a0 >= 0 && a0 < c.n_seqs ? c.lens[a0] : 0, blen0 = b0 >= 0 && b0 < c.n_seqs ? c.lens[b0] : 0;
    const int last0 = len_ok(c, alen0) && alen0 % c.page_size ? c.tables[(size_t)a0 * c.table_width + alen0 / c.page_size] : 0;
    first_of(c, dst, b0, n, first);
    uint32_t bad = 0;
    int total = 0;
    for (int base = 0; base < n; base += kPlan) {
        const int i = base + (int)threadIdx.x;
        int k = 0;
        if (i < n) {
            const bool own = i < kPlan;
            const int a = own ? a0 : src[i], b = own ? b0 : dst[i];
            int4 e = make_int4(a, -1, 0, -1);
            if (a < 0 || a >= c.n_seqs || b < 0 || b >= c.n_seqs) {
                bad |= GSDH_PAGES_BAD_INDEX;
            } else {
                const int len = own ? alen0 : c.lens[a];
                if (!len_ok(c, len)) bad |= GSDH_PAGES_BAD_INDEX;
                else if (first[b] != i || (own ? blen0 : c.lens[b]) != 0) bad |= GSDH_PAGES_TWICE;
                else e = make_int4(a, b, len, -1);
            }
            const int part = e.z % c.page_size;
            const int page = !part ? 0 : own ? last0 : c.tables[(size_t)a * c.table_width + e.z / c.page_size];
            if ((unsigned)page >= (unsigned)c.n_pages) {
                bad |= GSDH_PAGES_BAD_INDEX;
                e = make_int4(a, -1, 0, -1);
            } else {
                k = part != 0;
            }
            plan[i] = e;
        }
        int sum;
        const int at = block_scan(k, scan, &sum);
        if (i < n) off[i] = total + at;
        total += sum;
    }
    __syncthreads();
    const int found = scan_pages(c.refs, c.n_pages, total, words, [](int r, int) { return r == 0; },
        [&](int page, bool free_, int rank) {
            if (!free_ || rank >= total) return;
            const int i = owner_of(off, n, rank);
            plan[i].w = page;
            c.refs[page] = 1;
        });
    for (int i = threadIdx.x; i < n; i += kPlan) {
        const int4 e = plan[i];
        if (e.y < 0) continue;
        if (e.z % c.page_size && off[i] >= found) {
            plan[i].y = -1;
            bad |= GSDH_PAGES_EXHAUSTED;
        }
    }
    if (bad) page_status(c, bad);
}

// One block of a fork's rows: blockIdx.y = 0: the entry's table row, the shared
// pages' counts and the length, if all shared pages are the pool's (else the page
// taken goes back; a look at them in the plan would be 1 us more of its chain);
// else the filled rows of the last page in K or V of a layer.
__global__ void __launch_bounds__(256) pages_fork_rows_kernel(const gsdh_paged_cache c, const int4* plan, int es) {
    const int4 e = plan[blockIdx.x];
    if (e.y < 0) return;
    const int full = e.z / c.page_size, part = e.z % c.page_size;
    const int* from = c.tables + (size_t)e.x * c.table_width;
    if (blockIdx.y == 0) {
        int* to = c.tables + (size_t)e.y * c.table_width;
        bool out = false;
        for (int j = threadIdx.x; j < full; j += 256) out |= (unsigned)from[j] >= (unsigned)c.n_pages;
        out = __syncthreads_or(out);
        if (out) {
            if (threadIdx.x == 0) {
                if (part) c.refs[e.w] = 0;
                page_status(c, GSDH_PAGES_BAD_INDEX);
            }
            return;
        }
        for (int j = threadIdx.x; j < full; j += 256) {
            const int p = from[j];
            to[j] = p;
            atomicAdd(&c.refs[p], 1);
        }
        if (threadIdx.x == 0) {
            if (part) to[full] = e.w;
            c.lens[e.y] = e.z;
        }
        return;
    }
    if (!part) return;
    const int pool = blockIdx.y - 1;
    void *const k_pool = c.k, *const v_pool = c.v;
    // 16-byte words: the filled slots of all heads lie together, or each head's do
    const unsigned slot = (unsigned)c.head_dim * es / 16, runs = c.head_major ? c.n_kv_heads : 1;
    const unsigned run = slot * part * (c.head_major ? 1 : c.n_kv_heads), gap = c.head_major ? slot * c.page_size - run : 0;
    const size_t page = (size_t)slot * c.n_kv_heads * c.page_size;
    u32x4v* base = static_cast<u32x4v*>(pool & 1 ? v_pool : k_pool) + (size_t)(pool >> 1) * c.n_pages * page;
    const u32x4v* s = base + (size_t)from[full] * page;
    u32x4v* d = base + (size_t)e.w * page;
    const unsigned all = run * runs;
    for (unsigned k = threadIdx.x; k < all; k += 8 * 256) {
        u32x4v w[8];
        unsigned at[8];
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const unsigned i = min(k + 256 * j, all - 1);
            at[j] = gap ? i + i / run * gap : i;
            w[j] = s[at[j]];
        }
#pragma unroll
        for (int j = 0; j < 8; j++)
            if (k + 256 * j < all) d[at[j]] = w[j];
    }
}

__global__ void __launch_bounds__(256) pages_free_kernel(const gsdh_paged_cache c, const int* seqs) {
    const int s = seqs[blockIdx.x];
    __shared__ int len;
    const bool in = s >= 0 && s < c.n_seqs;
    if (threadIdx.x == 0) len = in ? atomicExch(&c.lens[s], 0) : -1;   // (one of two that name it gets the length)
    __syncthreads();
    if (!len_ok(c, len)) {
        if (threadIdx.x == 0) {
            // (back again; one that names it, too, and came in between found a free
            // sequence.  A load ahead of the exchange would be one more wait, 0.5 us.)
            if (in) atomicExch(&c.lens[s], len);
            page_status(c, GSDH_PAGES_BAD_INDEX);
        }
        return;
    }
    int* t = c.tables + (size_t)s * c.table_width;
    for (int j = threadIdx.x; j < pages_for(c, len); j += 256) {
        const int p = t[j];
        t[j] = -1;
        if ((unsigned)p >= (unsigned)c.n_pages) page_status(c, GSDH_PAGES_BAD_INDEX);
        else if (atomicSub(&c.refs[p], 1) <= 0) {   // (held by nobody: as it was)
            atomicAdd(&c.refs[p], 1);
            page_status(c, GSDH_PAGES_BAD_INDEX);
        }
    }
}

// Which page moves where: src[first + i] -> dst[i]; map[p] is the new place of a page
// p that moves, -1 for the free ones among those behind the last used place.
__global__ void __launch_bounds__(kPlan) pages_compact_kernel(const gsdh_paged_cache c, int* n_used, int* ws, Space s) {
    __shared__ __align__(8) int words[kRun * kPlanWaves];
    int *src = ws + s.src, *dst = ws + s.dst, *map = ws + s.map;
    const auto used = [](int r, int) { return r > 0; };
    const int n = scan_pages(c.refs, c.n_pages, c.n_pages + 1, words, used, [](int, bool, int) {});
    // holes below n in their order; behind them the used pages by their rank among all
    __shared__ int stay;   // used pages below n
    if (threadIdx.x == 0) stay = 0;
    scan_pages(c.refs, c.n_pages, c.n_pages + 1, words, used, [&](int page, bool in_use, int rank) {
        if (page < n) {
            if (!in_use) dst[page - rank] = page;
            if (page == n - 1) stay = rank + in_use;
        } else if (in_use) {
            src[rank] = page;
        } else {
            map[page] = -1;
        }
    });
    const int moves = n - stay;
    __threadfence_block();
    __syncthreads();
    for (int i = threadIdx.x; i < moves; i += kPlan) {
        const int a = src[stay + i], b = dst[i];
        map[a] = b;
        c.refs[b] = c.refs[a];
        c.refs[a] = 0;
    }
    if (threadIdx.x == 0) {
        ws[kMoves] = moves;
        ws[kFirst] = stay;
        ws[kUsed] = n;
        if (n_used) *n_used = n;
    }
}

// Whole pages, one after another in each block: page src[i] to page dst[i]
// in K or V of a layer (32 KB for 16 slots of 8 heads of 128 dims), eight
// 16-byte loads of a thread ahead of its stores.  The stores pass the caches
// by: a server's moves exceed them, and what they would push out is still to
// be read (294 MB moved: 74 us with ordinary stores, 59 so).  dst[i] < 0: left out.
__device__ __forceinline__ void move_pages(u32x4v* k_pool, u32x4v* v_pool, size_t n_pages, unsigned pools, const int* src, const int* dst,
                                           int n, size_t page, unsigned block, unsigned blocks) {
    for (size_t u = block; u < (size_t)n * pools; u += blocks) {
        const unsigned i = (unsigned)(u / pools), pool = (unsigned)(u % pools);
        const int a = src[i], b = dst[i];
        if (b < 0) continue;
        u32x4v* base = (pool & 1 ? v_pool : k_pool) + (pool >> 1) * n_pages * page;
        const u32x4v* s = base + (size_t)a * page;
        u32x4v* d = base + (size_t)b * page;
        size_t k = threadIdx.x;
        for (; k + 7 * 256 < page; k += 8 * 256) {
            u32x4v w[8];
#pragma unroll
            for (int j = 0; j < 8; j++) w[j] = s[k + 256 * j];
#pragma unroll
            for (int j = 0; j < 8; j++) __builtin_nontemporal_store(w[j], d + k + 256 * j);
        }
        for (; k < page; k += 256) d[k] = s[k];
    }
}

// The moves of a compaction, and the tables' entries after them.
__global__ void __launch_bounds__(256) pages_compact_rows_kernel(const gsdh_paged_cache c, const int* ws, Space s, size_t page, unsigned table_blocks) {
    const int moves = ws[kMoves], used = ws[kUsed], first = ws[kFirst];
    if (moves == 0) return;
    if (blockIdx.x >= table_blocks) {
        move_pages(static_cast<u32x4v*>(c.k), static_cast<u32x4v*>(c.v), (size_t)c.n_pages, 2u * c.n_layers, ws + s.src + first, ws + s.dst, moves, page,
                   blockIdx.x - table_blocks, gridDim.x - table_blocks);
        return;
    }
    for (int q = blockIdx.x; q < c.n_seqs; q += table_blocks) {
        const int len = c.lens[q];
        if (!len_ok(c, len)) continue;
        int* t = c.tables + (size_t)q * c.table_width;
        for (int j = threadIdx.x; j < pages_for(c, len); j += 256) {
            const int p = t[j];
            if ((unsigned)p < (unsigned)used) continue;
            const int to = (unsigned)p < (unsigned)c.n_pages ? ws[s.map + p] : -1;
            if (to >= 0) t[j] = to;
            else page_status(c, GSDH_PAGES_BAD_INDEX);   // (it names a page that nobody holds)
        }
    }
}

// A copy's plan: which entries are done (the first of each destination, no
// source that is one itself).
__global__ void __launch_bounds__(kPlan) pages_copy_kernel(const gsdh_paged_cache c, const int* src, const int* dst, int n, int* ws, Space s) {
    int *from = ws + s.src, *to = ws + s.dst, *first = ws + s.map;
    auto in = [&](int p) { return (unsigned)p < (unsigned)c.n_pages; };
    for (int i = threadIdx.x; i < n; i += kPlan) {
        if (in(src[i])) first[src[i]] = 0x7FFFFFFF;
        if (in(dst[i])) first[dst[i]] = 0x7FFFFFFF;
    }
    __threadfence_block();
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kPlan)
        if (in(src[i]) && in(dst[i])) atomicMin(&first[dst[i]], i);
    __threadfence_block();
    __syncthreads();
    uint32_t bad = 0;
    for (int i = threadIdx.x; i < n; i += kPlan) {
        const int a = src[i], b = dst[i];
        bool take = in(a) && in(b);
        if (!take && a >= 0 && b >= 0) bad |= GSDH_PAGES_BAD_INDEX;
        if (take && (first[b] != i || first[a] != 0x7FFFFFFF)) {
            take = false;
            bad |= GSDH_PAGES_TWICE;
        }
        from[i] = a;
        to[i] = take ? b : -1;
    }
    if (bad) page_status(c, bad);
}

__global__ void __launch_bounds__(256) pages_copy_rows_kernel(const gsdh_paged_cache c, const int* ws, Space s, int n, size_t page) {
    move_pages(static_cast<u32x4v*>(c.k), static_cast<u32x4v*>(c.v), (size_t)c.n_pages, 2u * c.n_layers, ws + s.src, ws + s.dst, n, page, blockIdx.x,
               gridDim.x);
}

unsigned move_blocks() { return 4u * (unsigned)std::max(1, device_cu_count()); }

int check_list(const gsdh_paged_cache* c, const int* a, const int* b, int n, int most, const char* who) {
    if (n < 0 || n > most) return fail(-1, "%s: a list of %d (at most %d)", who, n, most);
    if (n && (!a || !b)) return fail(-1, "%s: null list", who);
    return 0;
}

template <typename K>
hipError_t raise_plan_lds(LdsLimit& limit, K kernel, size_t lds) {
    return raise_lds_limit(limit, reinterpret_cast<const void*>(kernel), lds);
}

}  // namespace

extern "C" {

uint64_t gsdh_pages_workspace_bytes(const gsdh_paged_cache* c) {
    if (check_paged_cache(c, "pages_workspace_bytes", false)) return 0;
    return 4 * (uint64_t)space_of(*c).words;
}

int gsdh_pages_take(void* stream, const gsdh_paged_cache* c, const int* seqs, const int* counts, int n) {
    const char* who = "pages_take";
    int rc = check_paged_cache(c, who, true);
    if (!rc) rc = check_list(c, seqs, counts, n, c->n_seqs, who);
    if (rc || n == 0) return rc;
    static LdsLimit limit;
    const size_t lds = plan_lds(*c, n);
    GSD_PAGED_CHK(raise_plan_lds(limit, pages_take_kernel, lds), who);
    hipLaunchKernelGGL(pages_take_kernel, dim3(1), dim3(kPlan), lds, static_cast<hipStream_t>(stream), *c, seqs, counts, n);
    GSD_PAGED_CHK(hipGetLastError(), who);
    return 0;
}

int gsdh_pages_fork(void* stream, const gsdh_paged_cache* c, const int* src, const int* dst, int n, void* workspace,
                    uint64_t workspace_bytes) {
    const char* who = "pages_fork";
    int rc = check_paged_cache(c, who, true);
    if (!rc) rc = check_list(c, src, dst, n, c->n_seqs, who);
    if (rc || n == 0) return rc;
    const Space s = space_of(*c);
    rc = check_workspace(workspace, workspace_bytes, 4 * (uint64_t)s.words, who);
    if (rc) return rc;
    if (2 * (int64_t)c->n_layers + 1 > 65535) return fail(-1, "%s: %d layers", who, c->n_layers);
    static LdsLimit limit;
    const size_t lds = plan_lds(*c, n);
    hipStream_t st = static_cast<hipStream_t>(stream);
    int4* plan = reinterpret_cast<int4*>(static_cast<int*>(workspace) + s.plan);
    GSD_PAGED_CHK(raise_plan_lds(limit, pages_fork_kernel, lds), who);
    hipLaunchKernelGGL(pages_fork_kernel, dim3(1), dim3(kPlan), lds, st, *c, src, dst, n, plan);
    GSD_PAGED_CHK(hipGetLastError(), who);
    hipLaunchKernelGGL(pages_fork_rows_kernel, dim3((unsigned)n, 2u * (unsigned)c->n_layers + 1u), dim3(256), 0, st, *c, plan,
                       kv_type_bytes(c->dtype));
    GSD_PAGED_CHK(hipGetLastError(), who);
    return 0;
}

int gsdh_pages_free(void* stream, const gsdh_paged_cache* c, const int* seqs, int n) {
    const char* who = "pages_free";
    int rc = check_paged_cache(c, who, true);
    if (!rc) rc = check_list(c, seqs, seqs, n, c->n_seqs, who);
    if (rc || n == 0) return rc;
    hipLaunchKernelGGL(pages_free_kernel, dim3((unsigned)n), dim3(256), 0, static_cast<hipStream_t>(stream), *c, seqs);
    GSD_PAGED_CHK(hipGetLastError(), who);
    return 0;
}

int gsdh_pages_compact(void* stream, const gsdh_paged_cache* c, int* n_used, void* workspace, uint64_t workspace_bytes) {
    const char* who = "pages_compact";
    int rc = check_paged_cache(c, who, true);
    if (rc) return rc;
    const Space s = space_of(*c);
    rc = check_workspace(workspace, workspace_bytes, 4 * (uint64_t)s.words, who);
    if (rc) return rc;
    hipStream_t st = static_cast<hipStream_t>(stream);
    int* ws = static_cast<int*>(workspace);
    hipLaunchKernelGGL(pages_compact_kernel, dim3(1), dim3(kPlan), 0, st, *c, n_used, ws, s);
    GSD_PAGED_CHK(hipGetLastError(), who);
    const unsigned tables = (unsigned)std::min(c->n_seqs, 256);
    hipLaunchKernelGGL(pages_compact_rows_kernel, dim3(tables + move_blocks()), dim3(256), 0, st, *c, ws, s, page_bytes(*c) / 16, tables);
    GSD_PAGED_CHK(hipGetLastError(), who);
    return 0;
}

int gsdh_pages_copy(void* stream, const gsdh_paged_cache* c, const int* src, const int* dst, int n, void* workspace,
                    uint64_t workspace_bytes) {
    const char* who = "pages_copy";
    int rc = check_paged_cache(c, who, false);
    if (!rc) rc = check_list(c, src, dst, n, c->n_pages, who);
    if (rc || n == 0) return rc;
    const Space s = space_of(*c);
    rc = check_workspace(workspace, workspace_bytes, 4 * (uint64_t)s.words, who);
    if (rc) return rc;
    hipStream_t st = static_cast<hipStream_t>(stream);
    int* ws = static_cast<int*>(workspace);
    hipLaunchKernelGGL(pages_copy_kernel, dim3(1), dim3(kPlan), 0, st, *c, src, dst, n, ws, s);
    GSD_PAGED_CHK(hipGetLastError(), who);
    const size_t units = (size_t)n * 2 * c->n_layers;
    hipLaunchKernelGGL(pages_copy_rows_kernel, dim3((unsigned)std::min<size_t>(units, move_blocks())), dim3(256), 0, st, *c, ws, s, n,
                       page_bytes(*c) / 16);
    GSD_PAGED_CHK(hipGetLastError(), who);
    return 0;
}

}  // extern "C"
