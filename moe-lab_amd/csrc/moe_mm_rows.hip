// Forward products of few rows: one wave per R rows of the weights, dot products on the vector unit.
#include "moe_mm.h"

namespace moe {

template <bool F16>
__device__ __forceinline__ float dot2(uint32_t a, uint32_t b, float c) {
    return F16 ? dot2_f16(a, b, c) : dot2_bf16(a, b, c);
}

// A group's rows are multiplied MR at a time; the weights come from HBM once and, for the further passes of a group with more
// rows, from the caches. Bound by the weights' bytes: every 16-byte load of a wave is a contiguous 1 KiB of a weight row
// (traced: w [14336, 4096], one row: 19.6 us, 6.0 TB/s; 8 experts' [1536, 2048]: 10.6 us, 4.7 TB/s).
// GLU: a wave takes R rows of gate and the same R of up, and writes h.
// Workgroups go by slot, not by group: with few slots most groups are empty. The one at a group's first slot does the group.
template <bool F16, int R, int MR, bool GLU>
__global__ void __launch_bounds__(256) k_mm_rows(const MmArgs g) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int n0 = (blockIdx.x * 4 + wave) * R;
    const int p = blockIdx.y;
    int e = 0, lo = 0, hi = g.M;
    if (g.offsets) {
        // the group whose first slot is p (none: p lies inside a group, or behind the last)
        e = -1;
        for (int base = 0; base < g.E && e < 0; base += 64) {
            int l = -1, h = -1;
            if (base + lane < g.E) group_of<MM_FWD>(g, base + lane, l, h);
            const uint64_t hit = __ballot(l == p && h > l);
            if (hit) {
                const int at = __builtin_ctzll(hit);
                e = base + at;
                group_of<MM_FWD>(g, e, lo, hi);
            }
        }
        if (e < 0) {
            if (!g.fill) return;
            int l, h;
            group_of<MM_FWD>(g, g.E - 1, l, h);
            if (p < h) return;
            if (lane < R && n0 + lane < g.J) {
                if (g.ydt == MOE_DTYPE_F32) ((float*)g.y)[(int64_t)p * g.J + n0 + lane] = 0.f;
                else ((uint16_t*)g.y)[(int64_t)p * g.J + n0 + lane] = 0;
            }
            return;
        }
    }
    if (n0 >= g.J) return;
    constexpr int S = GLU ? 2 : 1;
    const uint16_t* w = (const uint16_t*)g.b + ((int64_t)e * S * g.J + n0) * g.ldb;
    const int64_t up = (int64_t)g.J * g.ldb;
    for (int m0 = lo; m0 < hi; m0 += MR) {
        const uint16_t* x[MR];
        bool live[MR];
#pragma unroll
        for (int m = 0; m < MR; ++m) {
            int s = m0 + m < hi ? m0 + m : lo;
            if (g.arows) s = g.arows[s];
            live[m] = s >= 0 && s < g.a_n;
            x[m] = (const uint16_t*)g.a + (int64_t)(live[m] ? s : 0) * g.lda;
        }
        float acc[S * R][MR] = {};
        auto chunk = [&](int c) {
            const int k = c * 512 + lane * 8;
            const bool in = k < g.R;
            u32x4 wv[S * R], xv[MR];
#pragma unroll
            for (int r = 0; r < S * R; ++r)
                wv[r] = in && n0 + r % R < g.J ? *(const u32x4*)(w + (r < R ? 0 : up) + (int64_t)(r % R) * g.ldb + k)
                                               : (u32x4){0, 0, 0, 0};
#pragma unroll
            for (int m = 0; m < MR; ++m) xv[m] = in ? *(const u32x4*)(x[m] + k) : (u32x4){0, 0, 0, 0};
#pragma unroll
            for (int r = 0; r < S * R; ++r)
#pragma unroll
                for (int m = 0; m < MR; ++m)
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[r][m] = dot2<F16>(wv[r][i], xv[m][i], acc[r][m]);
        };
        const int chunks = (g.R + 511) / 512;
#pragma unroll 4
        for (int c = 0; c < chunks; ++c) chunk(c);
#pragma unroll
        for (int r = 0; r < S * R; ++r)
#pragma unroll
            for (int m = 0; m < MR; ++m) acc[r][m] = wave_sum_dpp(acc[r][m]);
#pragma unroll
        for (int m = 0; m < MR; ++m) {
            if (m0 + m >= hi) break;
            float v = 0.f, u = 0.f;
#pragma unroll
            for (int r = 0; r < R; ++r)
                if (lane == r) {
                    v = acc[r][m];
                    if constexpr (GLU) u = acc[R + r][m];
                }
            const int n = n0 + lane;
            if (lane < R && n < g.J) {
                if (!live[m]) v = 0.f;
                const int64_t at = (int64_t)(m0 + m) * g.J + n;
                if constexpr (GLU) {
                    float f, up1, df, du;
                    glu_parts(g.epi.act, v, live[m] ? u : 0.f, f, up1, df, du);
                    ((uint16_t*)g.y)[at] = (uint16_t)pack16<F16>(f * up1, 0.f);
                    continue;
                }
                if (g.epi.bias) v += un16<F16>(((const uint16_t*)g.epi.bias)[(int64_t)e * g.J + n]);
                if (g.epi.z) ((uint16_t*)g.epi.z)[at] = (uint16_t)pack16<F16>(v, 0.f);
                v = lin_act(g.epi.act, v);
                if (g.epi.residual) v += un16<F16>(((const uint16_t*)g.epi.residual)[at]);
                if (g.ydt == MOE_DTYPE_F32) ((float*)g.y)[at] = v;
                else ((uint16_t*)g.y)[at] = (uint16_t)pack16<F16>(v, 0.f);
            }
        }
    }
}

template <bool F16, int R, bool GLU>
static int launch_r(const MmArgs& a, hipStream_t st) {
    const dim3 grid((unsigned)((a.J + 4 * R - 1) / (4 * R)), a.offsets ? (unsigned)a.M : 1);
    if (a.M == 1 || (a.offsets && a.M <= a.E)) k_mm_rows<F16, R, 1, GLU><<<grid, 256, 0, st>>>(a);
    else k_mm_rows<F16, R, 4, GLU><<<grid, 256, 0, st>>>(a);
    return hipGetLastError() == hipSuccess ? MOE_OK : MOE_ERR_LAUNCH;
}
template <bool F16>
static int launch(const MmArgs& a, hipStream_t st) {
    // rows per wave: more share a load of x, fewer give a small product enough waves
    const int64_t waves = (int64_t)a.J * (a.offsets ? a.M : 1);
    if (a.kind == EPI_GLU) return waves >= 2 * 4096 ? launch_r<F16, 2, true>(a, st) : launch_r<F16, 1, true>(a, st);
    if (waves >= 4 * 4096) return launch_r<F16, 4, false>(a, st);
    if (waves >= 2 * 2048) return launch_r<F16, 2, false>(a, st);
    return launch_r<F16, 1, false>(a, st);
}

int launch_mm_rows(const MmArgs& a, hipStream_t st) { return a.f16 ? launch<true>(a, st) : launch<false>(a, st); }

}  // namespace moe
