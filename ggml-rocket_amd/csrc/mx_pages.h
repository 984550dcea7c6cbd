// SPDX-License-Identifier: MIT
// A KV cache in pages, on the device: a step's numbers, a tree's ancestors and the row of a position.
#pragma once

#include "mx_common.h"
#include "mx_kernels_impl.h"

namespace mx {

// A value that every lane of the wave reads, through the scalar cache: no vector load, which the waits of a kernel
// that counts them would have to count as well.
typedef const int32_t __attribute__((address_space(4))) * const_i32_t;
__device__ __forceinline__ int uniform_i32(const int32_t * p, int64_t i) {
    return ((const_i32_t)(uintptr_t)p)[i];
}

// What sequence s holds and adds. bad: n_past lies outside [0, cap] (nothing is added then), n_new outside [0, T] (held to
// it), or the new rows pass cap.
struct StepOf {
    int past, fresh;
    bool bad;
};
__device__ __forceinline__ StepOf step_of(const KvStepArgs & a, int s) {
    const int p = uniform_i32(a.n_past, s), n = a.n_new ? uniform_i32(a.n_new, s) : a.T;
    StepOf r;
    r.past = min(max(p, 0), a.cap);
    r.fresh = r.past == p ? min(max(n, 0), a.T) : 0;
    r.bad = r.past != p || r.fresh != n || n > a.cap - p;
    return r;
}

// The cache row where page `entry` of a table begins, or -1 if the cache has no such page.
__device__ __forceinline__ int64_t page_row(const KvStepArgs & a, int entry) {
    return entry >= 0 && entry < a.n_pages ? (int64_t)entry * a.page : -1;
}

// The ancestors of tree node `lane`, itself among them, as bits, from its parent's number (`up`: -1 the root); 0 for a
// node whose way up meets a number that is neither -1 nor a node before its own. By doubling: after
// round r a node has its next 2^r ancestors and knows the one above them. Lanes past the T nodes pass -1.
__device__ __forceinline__ uint64_t tree_ancestors(int up, int lane) {
    if (up < -1 || up >= lane) up = -2;
    uint32_t lo = lane < 32 ? 1u << lane : 0u, hi = lane < 32 ? 0u : 1u << (lane - 32);
#pragma unroll
    for (int r = 0; r < 6; r++) {
        const int from = up >= 0 ? up : lane;
        const uint32_t lo2 = (uint32_t)__shfl((int)lo, from, WAVE), hi2 = (uint32_t)__shfl((int)hi, from, WAVE);
        const int up2 = __shfl(up, from, WAVE);
        if (up >= 0) {
            lo |= lo2;
            hi |= hi2;
            up = up2;
        }
    }
    return up == -2 ? 0 : (uint64_t)hi << 32 | lo;
}

}  // namespace mx
