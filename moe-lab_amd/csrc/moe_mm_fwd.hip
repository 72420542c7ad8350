#include "moe_mm.h"

namespace moe {

// Grouped, by the slots per group that can hold any. One: the weights' bytes are all there is, and the dot products have the
// most loads in flight (64 experts x 1 slot, [2048, 2048]: 51.7 us, 64 x 64 57.5; x 2 slots 92.0 and 84.7). Up to 32: 64 x 64
// (64 x 8: 107 us, 128 x 256 126; 32 uneven ones on average 119 and 143). Too few tiles for all CUs: 128 x 128 (8 x 128,
// [2048, 2048]: 27.4 us, 128 x 256 32.4). Else 128 x 256 (128 x 256 uneven, [1536, 2048]: 286 us, 128 x 128 319; 32 x 139,
// [5760, 2880]: 274 and 321).
static int grouped(const MmArgs& a) {
    const int64_t live = a.E < a.M ? a.E : a.M, avg = a.M / live, J = a.kind == EPI_GLU ? 2 * (int64_t)a.J : a.J;
    // the dot products have no block of 32 columns for the 8-bit form, and write no gate/up rows
    if (avg <= 1 && !(a.kind == EPI_GLU && (a.epi.gu || a.epi.codes))) return MM_ROWS;
    if (avg <= 32) return MM_64;
    return (live / 2 + a.M / 128) * ((J + 127) / 128) <= 256 ? MM_128_DEEP : MM_128x256;
}

template <bool F16>
static int launch(const MmArgs& a, hipStream_t st) {
    const int s = a.offsets ? grouped(a) : a.M <= MM_FEW && !a.part ? MM_ROWS : mm_plan(MM_FWD, a.M, a.J, a.R, a.part != 0).shape;
    switch (s) {
        case MM_128x256: return launch_mm_cfg<MM_FWD, F16, 4, 4, 4, 3, 1, 4>(a, st);
        case MM_128_DEEP: return launch_mm_cfg<MM_FWD, F16, 4, 4, 2, 4, 1, 4>(a, st);
        case MM_64:   // (a wave of 64 x 64 tiles has too few columns for a block of gate and one of up)
            if (a.kind == EPI_GLU) return launch_mm_cfg<MM_FWD, F16, 2, 4, 2, 3, 2>(a, st);
            return launch_mm_cfg<MM_FWD, F16, 2, 2, 2, 4, 2, 4>(a, st);
        default: return launch_mm_rows(a, st);
    }
}
int launch_mm_fwd(const MmArgs& a, hipStream_t st) {
    if (a.sa) return launch_mm_mx4(a, st);
    return a.f16 ? launch<true>(a, st) : launch<false>(a, st);
}

}  // namespace moe
