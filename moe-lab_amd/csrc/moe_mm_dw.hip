#include "moe_mm.h"

namespace moe {

// Tiles of 128 x 128, two workgroups on a CU: while one stores its sums the other multiplies, and with sums over the slots of
// one expert (often three steps of 64) stores are most of the traffic. With long sums and enough tiles, 128 x 256. Measured,
// 128 x 128 against 128 x 256: 32 experts x 139 slots, [5760, 2880] 330 and 410 us; 64 x 128, [2048, 2048] 162 and 229;
// 8 x 1024, [4096, 4096] 314 and 305; one group of 8192, [8192, 2048] 272 and 240; 4096, [4096, 4096] 141 and 129.
static int grouped(const MmArgs& a) {
    const int64_t big = (int64_t)a.E * ((a.I + 127) / 128) * ((a.J + 255) / 256);
    return a.M / a.E >= 1024 && big >= 192 ? MM_128x256 : MM_128;
}

// One group: by the plan, but not with the larger tile for short sums (237 slots, [2048, 2816]: 128 x 256 11.4 us, 128 x 128
// 9.3).
static int dense(const MmArgs& a) {
    const int s = mm_plan(MM_DW, a.I, a.J, a.M, a.part != 0).shape;
    return !a.part && a.M < 1024 && s == MM_128x256 ? MM_128 : s;
}

template <bool F16>
static int launch(const MmArgs& args, hipStream_t st) {
    MmArgs a = args;
    const int s = a.offsets ? grouped(a) : dense(a);
    // operands up to half of the memory cache, in groups of a few steps
    const int64_t ra = a.arows ? a.a_n : a.M, rb = a.brows ? a.b_n : a.M;
    a.touch = a.offsets && a.M > 0 && ra * a.lda + rb * a.ldb <= (64 << 20) && a.M / a.E <= 256;
    switch (s) {
        case MM_128x256: return launch_mm_cfg<MM_DW, F16, 4, 4, 4, 3, 1, 4>(a, st);
        case MM_128_DEEP: return launch_mm_cfg<MM_DW, F16, 4, 4, 2, 4, 1, 4>(a, st);
        case MM_64: return launch_mm_cfg<MM_DW, F16, 2, 2, 2, 4, 2>(a, st);
        default: return launch_mm_cfg<MM_DW, F16, 4, 4, 2, 2, 2>(a, st);
    }
}
int launch_mm_dw(const MmArgs& a, hipStream_t st) { return a.f16 ? launch<true>(a, st) : launch<false>(a, st); }

}  // namespace moe
