#include "moe_mm.h"

namespace moe {

// Grouped, as the forward product; few slots per group have 128 x 128 here, where a wider tile reads longer runs of w's rows
// (64 experts x 8 slots, [2048, 2048]: 97 us, 64 x 64 113, 128 x 256 96; x 4.6, [2048, 1024] 44.9, 51.5 and 46.0; from 16 on
// 128 x 256: 128 x 32, [1536, 2048] 144 and 153).
static int grouped(const MmArgs& a) {
    const int64_t live = a.E < a.M ? a.E : a.M, avg = a.M / live;
    if (avg <= 8) return MM_128;
    return (live / 2 + a.M / 128) * ((a.J + 127) / 128) <= 256 ? MM_128_DEEP : MM_128x256;
}

template <bool F16>
static int launch(const MmArgs& a, hipStream_t st) {
    const int s = a.offsets ? grouped(a) : mm_plan(MM_DX, a.M, a.J, a.R, a.part != 0).shape;
    switch (s) {
        case MM_128x256: return launch_mm_cfg<MM_DX, F16, 4, 4, 4, 3, 1, 4>(a, st);
        case MM_128_DEEP: return launch_mm_cfg<MM_DX, F16, 4, 4, 2, 4, 1, 4>(a, st);
        case MM_128: return launch_mm_cfg<MM_DX, F16, 4, 4, 2, 2, 2>(a, st);
        default: return launch_mm_cfg<MM_DX, F16, 2, 2, 2, 4, 2, 4>(a, st);
    }
}
int launch_mm_dx(const MmArgs& a, hipStream_t st) { return a.f16 ? launch<true>(a, st) : launch<false>(a, st); }

}  // namespace moe
