#include "moe_mm.h"

namespace moe {

int launch_mm_dx(const MmArgs& a, hipStream_t st) {
    const int force = env_int("MM_CFG", -1);
    const int64_t live = a.offsets ? (a.E < a.M ? a.E : a.M) : 1;   // groups that can hold a slot
    const int64_t avg = a.M / live;
    auto tiles = [&](int b) { return (live + a.M / b) * ((a.J + b - 1) / b); };
    int c = avg > 64 && tiles(256) >= 192 ? 0 : avg > 32 && tiles(128) >= 192 ? 1 : 2;
    if (force >= 0) c = force;
    if (c == 0) return a.f16 ? launch_mm_cfg<MM_DX, true, 8, 8, 2, 1>(a, st) : launch_mm_cfg<MM_DX, false, 8, 8, 2, 1>(a, st);
    if (c == 1) return a.f16 ? launch_mm_cfg<MM_DX, true, 4, 4, 2, 2>(a, st) : launch_mm_cfg<MM_DX, false, 4, 4, 2, 2>(a, st);
    return a.f16 ? launch_mm_cfg<MM_DX, true, 2, 2, 4, 2>(a, st) : launch_mm_cfg<MM_DX, false, 2, 2, 4, 2>(a, st);
}

}  // namespace moe
