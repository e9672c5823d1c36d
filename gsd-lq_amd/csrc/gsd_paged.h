// gsd_paged.h -- what the paged cache's kernels share: the check of a cache's
// descriptor and the addressing of its pages.  Internal to libgsdhip.so.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/gsdhip.h"
#include "gsd_internal.h"

namespace gsd {

// 0, or fail() with the reason (who: the entry point's name)
int check_paged_cache(const gsdh_paged_cache* c, const char* who, bool needs_refs);
// a caller's workspace: 16-byte aligned and at least `need` bytes
int check_workspace(const void* ws, uint64_t have, uint64_t need, const char* who);

inline int kv_type_bytes(int dtype) { return dtype == GSDH_KV_E4M3 ? 1 : 2; }
// bytes of one page of K (or V) of one layer
inline size_t page_bytes(const gsdh_paged_cache& c) {
    return (size_t)c.page_size * c.n_kv_heads * c.head_dim * kv_type_bytes(c.dtype);
}

// A workspace whose launches count arrivals: the first sixteenth of it holds
// the counters, zero between launches, whatever the sizes of a call are, so
// calls of different sizes never take one another's partial results for them.
inline size_t counter_bytes(uint64_t workspace_bytes) { return (size_t)(workspace_bytes / 256 * 16); }
inline uint64_t counted_workspace(uint64_t counters, uint64_t bytes) {
    const uint64_t n = counters * 4 > (bytes + 14) / 15 ? counters * 4 : (bytes + 14) / 15;   // the sixteenth
    return (n + 15) / 16 * 256;
}

#define GSD_PAGED_CHK(expr, who)                                                                  \
    do {                                                                                          \
        hipError_t e_ = (expr);                                                                   \
        if (e_ != hipSuccess) return ::gsd::fail((int)e_, "%s: %s", who, hipGetErrorString(e_)); \
    } while (0)

namespace {
__device__ __forceinline__ void page_status(const gsdh_paged_cache& c, uint32_t bits) {
    __hip_atomic_fetch_or(c.status, bits, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// Partial results that blocks on other XCDs read within the launch: 8-byte
// words stored and loaded past the XCD's own L2 (relaxed device-scope
// accesses).  arrive() after a barrier that every writer reached with its
// stores acknowledged (published()) counts the block in; the block that finds
// the others counted may read all words.  A release fence in place of this
// writes back the whole L2 of the XCD, once per block: 512 rows of 32768
// logits took 140 us with it and 30 without.
__device__ __forceinline__ void put2(float* p, float a, float b) {
    __hip_atomic_store(reinterpret_cast<unsigned long long*>(p),
                       (unsigned long long)__float_as_uint(b) << 32 | __float_as_uint(a), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float2 get2(const float* p) {
    const unsigned long long w =
        __hip_atomic_load(reinterpret_cast<const unsigned long long*>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return make_float2(__uint_as_float((unsigned)w), __uint_as_float((unsigned)(w >> 32)));
}
__device__ __forceinline__ void published() { __asm__ volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
// whether this block is the last of `of`; the counter is zero again then
__device__ __forceinline__ bool arrive(unsigned* counter, unsigned of) {
    const bool last = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == of - 1u;
    if (last) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return last;
}

}  // namespace

}  // namespace gsd
