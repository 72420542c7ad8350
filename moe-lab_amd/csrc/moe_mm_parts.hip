// Dense products with few output tiles: split over the sums, joined by a second kernel.
#include "moe_mm.h"

namespace moe {

// Which of the shapes, and into how many parts: the shortest of estimates that take a step of 64 r at its measured time with
// every CU busy, workgroups in rounds over the 256 CUs, a tile's start and stores as a few more, and the join as a launch and one
// pass over the parts at 4.5 TB/s. Measured, parts against one whole:
//   T 64, w [4096, 4096] 16.2 us, whole 24.5      T 512, w [4096, 4096] 31.3, whole 36.7
//   dx, T 1024, w [14336, 4096] 116, whole 157
//   dw of 16384 slots, [512, 512] 22.0, whole 107      dw of 65536 slots, [1024, 1024] 133, whole 426
MmPlan mm_plan(int mode, int64_t rows, int64_t J, int64_t R, bool split) {
    // us of a step: with two workgroups on each CU that takes two, and with one; steps that a tile's start and stores take
    static const struct { int shape, bi, bj, slots; float busy, alone; int more; } S[] = {
        {MM_128x256, 128, 256, 256, 0.83f, 0.83f, 3}, {MM_128_DEEP, 128, 128, 256, 0.52f, 0.52f, 6},
        {MM_128, 128, 128, 512, 1.05f, 0.92f, 2}, {MM_64, 64, 64, 512, 0.55f, 0.41f, 3}};
    MmPlan best{MM_128x256, 1};
    float least = 3e38f;
    for (const auto& c : S) {
        if (c.shape == MM_128 && mode != MM_DW) continue;
        const int64_t tiles = ((rows + c.bi - 1) / c.bi) * ((J + c.bj - 1) / c.bj), steps = (R + 63) / 64;
        for (int parts = 1; parts <= 64 && parts <= steps; parts *= 2) {
            const int64_t n = tiles * parts;
            if (parts > 1 && (!split || n > c.slots)) break;
            const float rounds = (float)((n + c.slots - 1) / c.slots);
            float us = rounds * (float)((steps + parts - 1) / parts + c.more) * (n <= 256 ? c.alone : c.busy);
            if (parts > 1) us += 3.5f + (float)parts * rows * J * 8.f / 4.5e6f;
            if (us < least) {
                least = us;
                best = {c.shape, parts};
            }
        }
    }
    return best;
}

template <bool F16>
__global__ void __launch_bounds__(256) k_join(const float* ws, int parts, int64_t n, uint32_t per_row, MmEpi epi, void* y, int ydt,
                                              const float* bias_parts, int bias_n, uint16_t* dbias) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;   // 8 columns
    if (dbias && i < bias_n) {
        float v = 0.f;
        for (int s = 0; s < parts; ++s) v += bias_parts[(int64_t)s * bias_n + i];
        dbias[i] = (uint16_t)pack16<F16>(v, 0.f);
    }
    if (i * 8 >= n) return;
    f32x4 v[2] = {};
#pragma unroll 4
    for (int s = 0; s < parts; ++s) {
        const f32x4* p = (const f32x4*)(ws + s * n + i * 8);
        v[0] += p[0];
        v[1] += p[1];
    }
    const auto words = [&]() {
        return (u32x4){pack16<F16>(v[0][0], v[0][1]), pack16<F16>(v[0][2], v[0][3]), pack16<F16>(v[1][0], v[1][1]),
                       pack16<F16>(v[1][2], v[1][3])};
    };
    if (epi.bias) {
        const int c = (int)(i % per_row) * 8;
        v[0] += load4<F16>(epi.bias, c);
        v[1] += load4<F16>(epi.bias, c + 4);
    }
    if (epi.z) ((u32x4*)epi.z)[i] = words();
#pragma unroll
    for (int u = 0; u < 2; ++u) {
#pragma unroll
        for (int c = 0; c < 4; ++c) v[u][c] = lin_act(epi.act, v[u][c]);
        if (epi.residual) v[u] += load4<F16>(epi.residual, i * 8 + 4 * u);
    }
    if (ydt == MOE_DTYPE_F32) {
        ((f32x4*)y)[2 * i] = v[0];
        ((f32x4*)y)[2 * i + 1] = v[1];
    } else {
        ((u32x4*)y)[i] = words();
    }
}

int launch_mm_parts(int mode, const MmArgs& a, int parts, float* ws, hipStream_t st) {
    MmArgs p = a;
    const int64_t sum = mode == MM_DW ? a.M : a.R, rows = mode == MM_DW ? a.I : a.M, n = rows * a.J;
    p.part = (int)((sum + 64 * parts - 1) / (64 * parts) * 64);
    p.E = (int)((sum + p.part - 1) / p.part);
    p.y = ws;
    p.ydt = MOE_DTYPE_F32;
    p.kind = EPI_PLAIN;
    p.epi = MmEpi{};
    float* bias_parts = ws + parts * n;
    if (a.dbias) p.dbias = bias_parts;
    const int rc = mode == MM_FWD ? launch_mm_fwd(p, st) : mode == MM_DX ? launch_mm_dx(p, st) : launch_mm_dw(p, st);
    if (rc) return rc;
    const unsigned grid = (unsigned)((n / 8 + 255) / 256);
    auto go = [&](auto kernel) {
        kernel<<<grid, 256, 0, st>>>(ws, p.E, n, (uint32_t)(a.J / 8), a.epi, a.y, a.ydt, bias_parts, a.I, (uint16_t*)a.dbias);
    };
    if (a.f16) go(k_join<true>);
    else go(k_join<false>);
    return hipGetLastError() == hipSuccess ? MOE_OK : MOE_ERR_LAUNCH;
}

}  // namespace moe
