#include "moe_mm.h"

namespace moe {

// The tiles of the 16-bit products on MXFP4 operands: a step of the same bytes holds four times as much of r.
static int grouped(const MmArgs& a) {
    const int64_t live = a.E < a.M ? a.E : a.M;
    if (a.M / live <= 32) return MM_64;
    return (live / 2 + a.M / 128) * ((a.J + 127) / 128) <= 256 ? MM_128_DEEP : MM_128x256;
}

template <bool F16>
static int launch(const MmArgs& a, hipStream_t st) {
    switch (a.offsets ? grouped(a) : mm_plan(MM_FWD, a.M, a.J, a.R, a.part != 0).shape) {
        case MM_128x256: return launch_mm_cfg<MM_FWD, F16, 4, 4, 4, 3, 1, 4, true>(a, st);
        case MM_128_DEEP: return launch_mm_cfg<MM_FWD, F16, 4, 4, 2, 4, 1, 4, true>(a, st);
        default: return launch_mm_cfg<MM_FWD, F16, 2, 2, 2, 4, 2, 4, true>(a, st);
    }
}
int launch_mm_mx4(const MmArgs& a, hipStream_t st) { return a.f16 ? launch<true>(a, st) : launch<false>(a, st); }

}  // namespace moe
