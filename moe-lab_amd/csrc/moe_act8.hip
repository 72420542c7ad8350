// Elementwise passes of the 16-bit expert layer: the GLU with its input kept in 8 bits, its backward pass from those codes,
// the activation's backward pass of the linear layer, and the weighted sum of a token's slots. Each is one pass over its
// data, 16 bytes per lane and load, and bound by HBM (traced: GLU with codes, 32768 rows of F 768, 33 us for 203 MB; from codes
// back to 16 bits 24 us for 153 MB; backward, 16383 rows of F 1024, 30 us for 169 MB).
#include "moe_mm.h"
#include "moe_rows.h"

namespace moe {

__device__ __forceinline__ uint32_t max_block(uint32_t v) {   // over the 4 lanes of 8 values that make a block of 32
    v = dpp_umax<0xB1>(v);
    return dpp_umax<0x4E>(v);
}
template <bool F16>
__device__ __forceinline__ void unpack8(u32x4 w, float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[2 * i] = un16<F16>(w[i]);
        v[2 * i + 1] = un16<F16>(w[i] >> 16);
    }
}
template <bool F16>
__device__ __forceinline__ u32x4 pack8(const float (&v)[8]) {
    return (u32x4){pack16<F16>(v[0], v[1]), pack16<F16>(v[2], v[3]), pack16<F16>(v[4], v[5]), pack16<F16>(v[6], v[7])};
}
// this lane's 8 codes; s: the block's exponent byte. All four lanes of a block are here or none.
__device__ __forceinline__ u32x2 quantise8(const float (&v)[8], uint32_t& s) {
    uint32_t b = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t a = __float_as_uint(v[i]) & 0x7fffffffu;
        b = a > b ? a : b;
    }
    s = exponent8(max_block(b));
    u32x2 q = {0, 0};
    if (s < 255) {
#pragma unroll
        for (int i = 0; i < 8; ++i) q[i >> 2] |= code8(v[i], s) << (8 * (i & 3));
    }
    return q;
}
__device__ __forceinline__ void values8(u32x2 q, uint32_t s, float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = value8(q[i >> 2] >> (8 * (i & 3)), s);
}

// gu [M, 2 F] -> h [M, F], and (codes not null) the 8-bit form of gu. One item: 8 columns of gate and up.
template <bool F16>
__global__ void __launch_bounds__(256) k_glu_fwd(const uint16_t* gu, int64_t ldg, uint32_t items, uint32_t per_row, int F, int act,
                                                 uint16_t* h, uint8_t* codes, uint8_t* scales) {
    const uint32_t i = blockIdx.x * 256 + threadIdx.x;
    if (i >= items) return;   // items % 4 == 0: a block's four lanes leave together
    const uint32_t row = i / per_row, c = (i - row * per_row) * 8;
    const uint16_t* p = gu + row * ldg + c;
    float g[8], u[8], o[8];
    unpack8<F16>(*(const u32x4*)p, g);
    unpack8<F16>(*(const u32x4*)(p + F), u);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        float f, m, df, dm;
        glu_parts(act, g[j], u[j], f, m, df, dm);
        o[j] = f * m;
    }
    *(u32x4*)(h + (uint64_t)row * F + c) = pack8<F16>(o);
    if (codes) {
        uint32_t sg, su;
        const u32x2 qg = quantise8(g, sg), qu = quantise8(u, su);
        uint8_t* q = codes + (uint64_t)row * 2 * F + c;
        *(u32x2*)q = qg;
        *(u32x2*)(q + F) = qu;
        if ((threadIdx.x & 3) == 0) {
            uint8_t* s = scales + ((uint64_t)row * 2 * F + c) / 32;
            s[0] = (uint8_t)sg;
            s[F / 32] = (uint8_t)su;
        }
    }
}

// Backward: from the codes (or gu itself, codes null), dh and the rows' weights w
//   dgu = w dh h'(g, u),  hw = w h,  dw = sum_f dh h
// L lanes per row. Row r's weight is wts[idx ? idx[r] : r], and dw goes there too; rows from *count on are left alone.
template <bool F16, int L>
__global__ void __launch_bounds__(256) k_glu_bwd(const GluBwd a) {
    const int64_t row = (int64_t)blockIdx.x * (256 / L) + threadIdx.x / L;
    const int64_t n = a.count ? min((int64_t)*a.count, a.M) : a.M;
    if (row >= n) return;
    const int F = a.F;
    const int64_t slot = a.idx ? a.idx[row] : row;
    const float w = a.wts ? a.wts[slot] : 1.f;
    float dw = 0.f;
    for (int c = (threadIdx.x % L) * 8; c < F; c += 8 * L) {
        float g[8], u[8], d[8], og[8], ou[8], oh[8];
        if (a.codes) {
            const uint8_t* q = a.codes + row * 2 * F + c;
            const uint8_t* s = a.scales + (row * 2 * F + c) / 32;
            values8(*(const u32x2*)q, s[0], g);
            values8(*(const u32x2*)(q + F), s[F / 32], u);
        } else {
            const uint16_t* p = a.gu + row * a.ldg + c;
            unpack8<F16>(*(const u32x4*)p, g);
            unpack8<F16>(*(const u32x4*)(p + F), u);
        }
        if (a.dh32) {
            const f32x4* p = (const f32x4*)((const float*)a.dh + row * F + c);
            const f32x4 d0 = p[0], d1 = p[1];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                d[j] = d0[j];
                d[4 + j] = d1[j];
            }
        } else {
            unpack8<F16>(*(const u32x4*)((const uint16_t*)a.dh + row * F + c), d);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            float f, m, df, dm;
            glu_parts(a.act, g[j], u[j], f, m, df, dm);
            const float h = f * m, wd = w * d[j];
            dw += d[j] * h;
            og[j] = wd * (df * m);
            ou[j] = wd * (f * dm);
            oh[j] = w * h;
        }
        uint16_t* o = a.dgu + row * 2 * F + c;
        *(u32x4*)o = pack8<F16>(og);
        *(u32x4*)(o + F) = pack8<F16>(ou);
        if (a.hw) *(u32x4*)(a.hw + row * F + c) = pack8<F16>(oh);
    }
    if (a.dwts) {
#pragma unroll
        for (int o = 1; o < L; o *= 2) dw += __shfl_xor(dw, o);
        if (threadIdx.x % L == 0) a.dwts[slot] = dw;
    }
}

// x [M, C] <-> 8 bits, 8 columns per item
template <bool F16>
__global__ void __launch_bounds__(256) k_pack8(const uint16_t* x, int64_t ld, uint32_t items, uint32_t per_row, uint8_t* codes,
                                               uint8_t* scales) {
    const uint32_t i = blockIdx.x * 256 + threadIdx.x;
    if (i >= items) return;
    const uint32_t row = i / per_row, c = (i - row * per_row) * 8;
    float v[8];
    unpack8<F16>(*(const u32x4*)(x + row * ld + c), v);
    uint32_t s;
    const u32x2 q = quantise8(v, s);
    *(u32x2*)(codes + (uint64_t)i * 8) = q;
    if ((threadIdx.x & 3) == 0) scales[i / 4] = (uint8_t)s;
}
template <bool F16>
__global__ void __launch_bounds__(256) k_unpack8(const uint8_t* codes, const uint8_t* scales, uint32_t items, void* out, int f32) {
    const uint32_t i = blockIdx.x * 256 + threadIdx.x;
    if (i >= items) return;
    float v[8];
    values8(*(const u32x2*)(codes + (uint64_t)i * 8), scales[i / 4], v);
    // fp16 values from 65280 on are kept as 64 steps of 1024, past fp16's range by one rounding
    if constexpr (F16)
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = fabsf(v[j]) == 65536.f ? copysignf(65504.f, v[j]) : v[j];
    if (f32) {
        f32x4* o = (f32x4*)((float*)out + (uint64_t)i * 8);
        o[0] = (f32x4){v[0], v[1], v[2], v[3]};
        o[1] = (f32x4){v[4], v[5], v[6], v[7]};
    } else {
        *(u32x4*)((uint16_t*)out + (uint64_t)i * 8) = pack8<F16>(v);
    }
}

// dz = dy act'(z), z as 16-bit values or 8-bit codes
template <bool F16>
__global__ void __launch_bounds__(256) k_lin_act_bwd(const uint16_t* dy, int64_t ldy, const uint16_t* z, const uint8_t* codes,
                                                     const uint8_t* scales, uint32_t items, uint32_t per_row, int act,
                                                     uint16_t* dz) {
    const uint32_t i = blockIdx.x * 256 + threadIdx.x;
    if (i >= items) return;
    const uint32_t row = i / per_row, c = (i - row * per_row) * 8;
    float d[8], v[8], o[8];
    unpack8<F16>(*(const u32x4*)(dy + row * ldy + c), d);
    if (codes) values8(*(const u32x2*)(codes + (uint64_t)i * 8), scales[i / 4], v);
    else unpack8<F16>(*(const u32x4*)(z + (uint64_t)i * 8), v);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        float f, m, df, dm;
        glu_parts(act == MOE_LIN_GELU ? MOE_ACT_GEGLU : MOE_ACT_SWIGLU, v[j], 1.f, f, m, df, dm);
        o[j] = d[j] * df;
    }
    *(u32x4*)(dz + (uint64_t)i * 8) = pack8<F16>(o);
}

// Slots of a grouping: rows[p] = token of the slot at sorted position p, pos[slot] = its position, -1 for an id outside
// [0, E).
__global__ void __launch_bounds__(256) k_slots(const int32_t* idx, const int32_t* sorted, const int32_t* offsets, int n, int k,
                                               int E, int32_t* rows, int32_t* pos) {
    const int p = blockIdx.x * 256 + threadIdx.x;
    if (p >= n) return;
    if (p < offsets[E]) {
        const int s = sorted[p];
        rows[p] = s / k;
        pos[s] = p;
    }
    if ((uint32_t)idx[p] >= (uint32_t)E) pos[p] = -1;
}

// y[t] = residual[t] + sum_j w[t][j] ys[pos[t k + j]] in fp32, slots in ascending j; 8 columns per item
template <bool F16>
__global__ void __launch_bounds__(256) k_slot_sum(const float* ys, const int32_t* pos, const float* wts, const uint16_t* residual,
                                                  int64_t M, int k, int d, uint32_t items, uint32_t per_row, void* y, int ydt) {
    const uint32_t i = blockIdx.x * 256 + threadIdx.x;
    if (i >= items) return;
    const uint32_t t = i / per_row, c = (i - t * per_row) * 8;
    float acc[8] = {};
    if (residual) unpack8<F16>(*(const u32x4*)(residual + (uint64_t)t * d + c), acc);
    // eight slots' loads before their sums: a branch per slot would wait for each (5 tokens of 8 slots: 5.6 us)
    for (int j0 = 0; j0 < k; j0 += 8) {
        int p[8];
        float w[8], v[8][8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const uint64_t s = (uint64_t)t * k + min(j0 + j, k - 1);
            p[j] = pos[s];
            w[j] = wts ? wts[s] : 1.f;
            if (j0 + j >= k || p[j] >= M) p[j] = -1;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const uint64_t at = (uint64_t)max(p[j], 0) * d + c;
            const f32x4 lo = *(const f32x4*)(ys + at), hi = *(const f32x4*)(ys + at + 4);
#pragma unroll
            for (int q = 0; q < 4; ++q) v[j][q] = lo[q], v[j][4 + q] = hi[q];
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            if (p[j] < 0) continue;
#pragma unroll
            for (int q = 0; q < 8; ++q) acc[q] += w[j] * v[j][q];
        }
    }
    if (ydt == MOE_DTYPE_F32) {
        f32x4* o = (f32x4*)((float*)y + (uint64_t)i * 8);
        o[0] = (f32x4){acc[0], acc[1], acc[2], acc[3]};
        o[1] = (f32x4){acc[4], acc[5], acc[6], acc[7]};
    } else {
        *(u32x4*)((uint16_t*)y + (uint64_t)i * 8) = pack8<F16>(acc);
    }
}

static int done() { return hipGetLastError() == hipSuccess ? MOE_OK : MOE_ERR_LAUNCH; }

// A kernel indexes its items with 32 bits: rows go in parts of fewer than 2^31 items.
template <class Fn>
static int by_parts(int64_t M, int64_t per_row, Fn fn) {
    const int64_t most = ((1ll << 31) - 1024) / per_row;
    for (int64_t r = 0; r < M; r += most) {
        const int64_t rows = M - r < most ? M - r : most;
        fn(r, (uint32_t)(rows * per_row), (unsigned)((rows * per_row + 255) / 256));
        const int rc = done();
        if (rc) return rc;
    }
    return MOE_OK;
}

int launch_glu_fwd(const void* gu, int64_t ldg, int64_t M, int F, int act, bool f16, void* h, uint8_t* codes, uint8_t* scales,
                   hipStream_t st) {
    return by_parts(M, F / 8, [&](int64_t r, uint32_t items, unsigned grid) {
        const uint16_t* p = (const uint16_t*)gu + r * ldg;
        uint16_t* o = (uint16_t*)h + r * F;
        uint8_t *q = codes ? codes + r * 2 * F : nullptr, *s = codes ? scales + r * (2 * F / 32) : nullptr;
        if (f16) k_glu_fwd<true><<<grid, 256, 0, st>>>(p, ldg, items, F / 8, F, act, o, q, s);
        else k_glu_fwd<false><<<grid, 256, 0, st>>>(p, ldg, items, F / 8, F, act, o, q, s);
    });
}

template <bool F16>
static void glu_bwd(const GluBwd& a, hipStream_t st) {
    // lanes per row: the most that leave no more than an eighth of them idle over the row's 16-byte pieces
    const int c = a.F / 8;
    auto fits = [&](int L) { return (c + L - 1) / L * L * 7 <= c * 8; };
    auto grid = [&](int L) { return (unsigned)((a.M + 256 / L - 1) / (256 / L)); };
    if (fits(64)) k_glu_bwd<F16, 64><<<grid(64), 256, 0, st>>>(a);
    else if (fits(32)) k_glu_bwd<F16, 32><<<grid(32), 256, 0, st>>>(a);
    else if (fits(16)) k_glu_bwd<F16, 16><<<grid(16), 256, 0, st>>>(a);
    else if (fits(8)) k_glu_bwd<F16, 8><<<grid(8), 256, 0, st>>>(a);
    else k_glu_bwd<F16, 4><<<grid(4), 256, 0, st>>>(a);
}
int launch_glu_bwd(const GluBwd& a, bool f16, hipStream_t st) {
    if (a.M == 0) return MOE_OK;
    if (f16) glu_bwd<true>(a, st);
    else glu_bwd<false>(a, st);
    return done();
}

int launch_pack8(const void* x, int64_t ld, int64_t M, int64_t C, bool f16, uint8_t* codes, uint8_t* scales, hipStream_t st) {
    return by_parts(M, C / 8, [&](int64_t r, uint32_t items, unsigned grid) {
        const uint16_t* p = (const uint16_t*)x + r * ld;
        if (f16) k_pack8<true><<<grid, 256, 0, st>>>(p, ld, items, (uint32_t)(C / 8), codes + r * C, scales + r * (C / 32));
        else k_pack8<false><<<grid, 256, 0, st>>>(p, ld, items, (uint32_t)(C / 8), codes + r * C, scales + r * (C / 32));
    });
}
int launch_unpack8(const uint8_t* codes, const uint8_t* scales, int64_t M, int64_t C, int dtype, void* out, hipStream_t st) {
    const int es = dtype == MOE_DTYPE_F32 ? 4 : 2;
    return by_parts(M, C / 8, [&](int64_t r, uint32_t items, unsigned grid) {
        void* o = (char*)out + r * C * es;
        if (dtype == MOE_DTYPE_F16) k_unpack8<true><<<grid, 256, 0, st>>>(codes + r * C, scales + r * (C / 32), items, o, 0);
        else k_unpack8<false><<<grid, 256, 0, st>>>(codes + r * C, scales + r * (C / 32), items, o, dtype == MOE_DTYPE_F32);
    });
}
int launch_lin_act_bwd(const void* dy, int64_t ldy, const void* z, const uint8_t* codes, const uint8_t* scales, int64_t M,
                       int64_t N, int act, bool f16, void* dz, hipStream_t st) {
    return by_parts(M, N / 8, [&](int64_t r, uint32_t items, unsigned grid) {
        const uint16_t *d = (const uint16_t*)dy + r * ldy, *v = z ? (const uint16_t*)z + r * N : nullptr;
        const uint8_t *q = codes ? codes + r * N : nullptr, *s = codes ? scales + r * (N / 32) : nullptr;
        uint16_t* o = (uint16_t*)dz + r * N;
        if (f16) k_lin_act_bwd<true><<<grid, 256, 0, st>>>(d, ldy, v, q, s, items, (uint32_t)(N / 8), act, o);
        else k_lin_act_bwd<false><<<grid, 256, 0, st>>>(d, ldy, v, q, s, items, (uint32_t)(N / 8), act, o);
    });
}
int launch_slots(const int32_t* idx, const int32_t* sorted, const int32_t* offsets, int n, int k, int E, int32_t* rows,
                 int32_t* pos, hipStream_t st) {
    if (n == 0) return MOE_OK;
    k_slots<<<(n + 255) / 256, 256, 0, st>>>(idx, sorted, offsets, n, k, E, rows, pos);
    return done();
}
int launch_slot_sum(const float* ys, const int32_t* pos, const float* wts, const void* residual, int64_t M, int64_t T, int k,
                    int d, bool f16, void* y, int ydt, hipStream_t st) {
    return by_parts(T, d / 8, [&](int64_t r, uint32_t items, unsigned grid) {
        const int32_t* p = pos + r * k;
        const float* w = wts ? wts + r * k : nullptr;
        const uint16_t* res = residual ? (const uint16_t*)residual + r * d : nullptr;
        void* o = (char*)y + r * d * (ydt == MOE_DTYPE_F32 ? 4 : 2);
        auto go = [&](auto kernel) { kernel<<<grid, 256, 0, st>>>(ys, p, w, res, M, k, d, items, d / 8, o, ydt); };
        f16 ? go(k_slot_sum<true>) : go(k_slot_sum<false>);
    });
}

}  // namespace moe
