#include "moe_mm.h"

namespace moe {

int launch_mm_dw(const MmArgs& a, hipStream_t st) {
    const int force = env_int("MM_CFG", -1);
    auto tiles = [&](int b) { return (int64_t)a.E * ((a.I + b - 1) / b) * ((a.J + b - 1) / b); };
    int c = tiles(256) >= 192 ? 0 : tiles(128) >= 192 ? 1 : 2;
    if (force >= 0 && force < 3) c = force;
    if (c == 0) return a.f16 ? launch_mm_cfg<MM_DW, true, 8, 8, 2, 1>(a, st) : launch_mm_cfg<MM_DW, false, 8, 8, 2, 1>(a, st);
    if (c == 1) return a.f16 ? launch_mm_cfg<MM_DW, true, 4, 4, 2, 2>(a, st) : launch_mm_cfg<MM_DW, false, 4, 4, 2, 2>(a, st);
    return a.f16 ? launch_mm_cfg<MM_DW, true, 2, 2, 4, 2>(a, st) : launch_mm_cfg<MM_DW, false, 2, 2, 4, 2>(a, st);
}

}  // namespace moe
