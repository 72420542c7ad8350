#include "moe_mm.h"

namespace moe {

template <bool F16>
static int launch(const MmArgs& a, hipStream_t st) {
    const int force = env_int("MM_CFG", -1);
    const int64_t live = a.offsets ? (a.E < a.M ? a.E : a.M) : 1;   // groups that can hold a slot
    const int64_t avg = a.M / live;
    auto tiles = [&](int bi, int bj) { return (live + a.M / bi) * ((a.J + bj - 1) / bj); };
    int c = avg > 64 && tiles(256, 256) >= 192 ? 0 : avg > 32 && tiles(128, 128) >= 192 ? 1 : 2;
    if (force >= 0) c = force;
    switch (c) {
        case 0: return launch_mm_cfg<MM_DX, F16, 8, 8, 2, 2, 1>(a, st);
        case 5: return launch_mm_cfg<MM_DX, F16, 8, 4, 4, 2, 1>(a, st);
        case 6: return launch_mm_cfg<MM_DX, F16, 4, 4, 4, 3, 1>(a, st);
        case 1: return launch_mm_cfg<MM_DX, F16, 4, 4, 2, 2, 2>(a, st);
        case 2: return launch_mm_cfg<MM_DX, F16, 2, 2, 2, 4, 2>(a, st);
        case 7: return launch_mm_cfg<MM_DX, F16, 4, 4, 2, 4, 1>(a, st);
        case 8: return launch_mm_cfg<MM_DX, F16, 2, 2, 2, 8, 1>(a, st);
        default: return MOE_ERR_ARG;
    }
}
int launch_mm_dx(const MmArgs& a, hipStream_t st) { return a.f16 ? launch<true>(a, st) : launch<false>(a, st); }

}  // namespace moe
