#include "moe_mm.h"

namespace moe {

template <bool F16>
static int launch(const MmArgs& a, hipStream_t st) {
    const int force = env_int("MM_CFG", -1);
    auto tiles = [&](int bi, int bj) { return (int64_t)a.E * ((a.I + bi - 1) / bi) * ((a.J + bj - 1) / bj); };
    int c = tiles(256, 256) >= 192 ? 0 : tiles(128, 128) >= 192 ? 1 : 2;
    if (force >= 0) c = force;
    switch (c) {
        case 0: return launch_mm_cfg<MM_DW, F16, 8, 8, 2, 2, 1>(a, st);
        case 5: return launch_mm_cfg<MM_DW, F16, 8, 4, 4, 2, 1>(a, st);
        case 1: return launch_mm_cfg<MM_DW, F16, 4, 4, 2, 2, 2>(a, st);
        case 4: return launch_mm_cfg<MM_DW, F16, 4, 8, 2, 3, 1>(a, st);
        default: return launch_mm_cfg<MM_DW, F16, 2, 2, 2, 4, 2>(a, st);
    }
}
int launch_mm_dw(const MmArgs& a, hipStream_t st) { return a.f16 ? launch<true>(a, st) : launch<false>(a, st); }

}  // namespace moe
