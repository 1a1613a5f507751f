// pages.h -- which sequence a row of a ragged batch belongs to, and where a
// position lies in the pages.
#pragma once
#include <algorithm>

#include "device_common.h"
#include "kernels.h"

namespace vai_dev {

// The last of `n` increasing numbers that is <= x, as its index; n if the first
// is larger (no such number). The whole wave calls with one x: 64 numbers are
// compared at a time, so 4096 of them take two loads.
__device__ __forceinline__ uint32_t wave_last_le(const uint32_t* a, uint32_t n, uint32_t x)
{
    const uint32_t lane = threadIdx.x & 63;
    uint32_t lo = 0, step = n > 64 ? (n + 63) / 64 : 1;   // (n <= 4096: step <= 64)
    uint64_t hit = __ballot(lane * step < n && a[min(lane * step, n - 1)] <= x);
    if (hit == 0) return n;
    lo = (63 - __builtin_clzll(hit)) * step;
    if (step > 1) {
        hit = __ballot(lane < step && lo + lane < n && a[min(lo + lane, n - 1)] <= x);
        lo += hit ? 63 - __builtin_clzll(hit) : 0;
    }
    return __builtin_amdgcn_readfirstlane(lo);
}

// A sequence of a ragged batch: its rows, and the positions held before them.
struct Sequence {
    uint32_t first, n;        // rows first .. first + n - 1
    uint32_t held;            // positions before the call, as counts has them: row t is at held + t
    uint32_t live;            // positions with its rows, as far as the table can hold them
};
__device__ __forceinline__ Sequence sequence_of(const KvPages& p, uint32_t s, uint32_t rows)
{
    Sequence q;
    const uint32_t a = min(p.start[s], rows), b = min(p.start[s + 1], rows);
    const uint32_t room = p.max_pages * p.page_size;      // (at most 2^30)
    q.first = a;
    q.n = b > a ? b - a : 0u;
    q.held = p.counts[s];
    q.live = (uint32_t)std::min<uint64_t>((uint64_t)q.held + q.n, room);
    return q;
}

// The same in every lane, in scalar registers.
__device__ __forceinline__ Sequence uniform(Sequence q)
{
    q.first = __builtin_amdgcn_readfirstlane(q.first);
    q.n = __builtin_amdgcn_readfirstlane(q.n);
    q.held = __builtin_amdgcn_readfirstlane(q.held);
    q.live = __builtin_amdgcn_readfirstlane(q.live);
    return q;
}

}   // namespace vai_dev
