// decode_range.h -- how the attention kernels for few query rows deal keys out:
// shared by their launches and the merge of their partial results.
#pragma once
#include <algorithm>

#include "kernels.h"

namespace vai_dev {
namespace fd {
constexpr int NW = 4, KT = 32;   // waves per workgroup; keys per wave tile

// The launch's key range: [tb, te) are the 32-key tiles some row sees. They
// are dealt out in turn, tile tb + i to wave i % NW of unit (i / NW) % units,
// so that which tiles a wave reads first does not wait for the live count
// unless a window moves tb.
struct Range {
    uint32_t cached, live;
    int64_t tb, te;
    uint32_t used;   // units with work (at least 1)
};
__device__ __forceinline__ Range range_of(const AttnDecodeParams& p)
{
    Range r;
    r.cached = p.cache_count ? __builtin_amdgcn_readfirstlane(*p.cache_count) : 0u;
    r.live = p.ring ? r.cached + p.tkv : std::min(r.cached + p.tkv, p.kv_rows);
    const int64_t kend = std::min<int64_t>(p.mask.key_end_cached(p.tq - 1, r.cached), r.live);
    const int64_t kbeg = p.mask.key_start_cached(0, r.cached);
    r.tb = kbeg / KT;
    r.te = kend <= kbeg ? r.tb : (kend + KT - 1) / KT;
    const uint32_t n = __builtin_amdgcn_readfirstlane((uint32_t)(r.te - r.tb));
    r.used = std::min(p.units, std::max<uint32_t>((n + NW - 1) / NW, 1u));
    return r;
}

}   // namespace fd
}   // namespace vai_dev
