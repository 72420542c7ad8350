#include "moe_mm.h"

namespace moe {

// Grouped, as the forward product; up to 32 slots per group 128 x 128 is the better one here, where a wider tile reads longer
// runs of w's rows (64 experts x 8 slots, [2048, 2048]: 95 us, 64 x 64 109, 128 x 256 105). 256 x 256 needs the tiles
// (16 x 187, dx of 2048 columns, 128 tiles: 114 us, 128 x 256 77; 64 x 175 138 and 164).
static int grouped(const MmArgs& a) {
    const int64_t live = a.E < a.M ? a.E : a.M, avg = a.M / live;
    if (avg <= 32) return MM_128;
    if ((live / 2 + a.M / 128) * ((a.J + 127) / 128) <= 256) return MM_128_DEEP;
    const bool many = (live / 2 + a.M / 256) * ((a.J + 255) / 256) >= 192;
    return avg >= 384 || (avg > 128 && avg <= 192 && many) ? MM_256 : MM_128x256;
}

template <bool F16>
static int launch(const MmArgs& a, hipStream_t st) {
    const int s = a.offsets ? grouped(a) : mm_plan(a.M, a.J, a.R, a.part != 0).shape;
    switch (s) {
        case MM_256: return launch_mm_cfg<MM_DX, F16, 8, 8, 2, 2, 1>(a, st);
        case MM_128x256: return launch_mm_cfg<MM_DX, F16, 4, 4, 4, 3, 1>(a, st);
        case MM_128: return launch_mm_cfg<MM_DX, F16, 4, 4, 2, 2, 2>(a, st);
        case MM_128_DEEP: return launch_mm_cfg<MM_DX, F16, 4, 4, 2, 4, 1>(a, st);
        default: return launch_mm_cfg<MM_DX, F16, 2, 2, 2, 4, 2>(a, st);
    }
}
int launch_mm_dx(const MmArgs& a, hipStream_t st) { return a.f16 ? launch<true>(a, st) : launch<false>(a, st); }

}  // namespace moe
