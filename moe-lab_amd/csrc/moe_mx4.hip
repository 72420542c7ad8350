// MXFP4 quantisation and its inverse, and products of few rows.
#include "moe_mx4.h"

namespace moe {

typedef float f32x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ uint32_t max4(uint32_t v) {   // over the 4 lanes of 8 values that make a block of 32
    v = dpp_umax<0xB1>(v);
    return dpp_umax<0x4E>(v);
}
// The block's exponent byte from the bits of its largest magnitude (fp32): that of the largest power of two in it, less 2, so that
// the largest lies in [4, 8) of E2M1's 6. Below 2^-124 (a byte of 0) the block is zeros; 255: it holds an infinity or NaN.
__device__ __forceinline__ uint32_t exponent4(uint32_t top) {
    const uint32_t e = top >> 23;
    return e == 255 ? 255 : e > 2 ? e - 2 : 0;
}
// Eight values of type DT as a lane holds them: u32x4 of 16-bit pairs, or two f32x4.
template <int DT>
struct Eight {
    u32x4 w[DT == MOE_DTYPE_F32 ? 2 : 1];
    __device__ __forceinline__ void load(const char* p) {
#pragma unroll
        for (int i = 0; i < (DT == MOE_DTYPE_F32 ? 2 : 1); ++i) w[i] = ((const u32x4*)p)[i];
    }
    __device__ __forceinline__ uint32_t top() const {   // bits of the largest magnitude in fp32
        uint32_t m = 0;
        if constexpr (DT == MOE_DTYPE_F32) {
#pragma unroll
            for (int i = 0; i < 8; ++i) m = max(m, w[i >> 2][i & 3] & 0x7fffffffu);
            return m;
        } else {
            typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
            u16x2 p = {0, 0};   // magnitudes of 16-bit floats compare as integers
#pragma unroll
            for (int i = 0; i < 4; ++i) p = __builtin_elementwise_max(p, __builtin_bit_cast(u16x2, w[0][i] & 0x7fff7fffu));
            const uint32_t h = max((uint32_t)p[0], (uint32_t)p[1]);
            return DT == MOE_DTYPE_BF16 ? h << 16 : __float_as_uint(un16<true>(h));
        }
    }
    // Their codes at the scale of byte e in [1, 254]. The instruction rounds to nearest, ties to even, and saturates.
    __device__ __forceinline__ uint32_t codes(uint32_t e) const {
        const float s = __uint_as_float(e << 23);
        uint32_t q = 0;
        if constexpr (DT == MOE_DTYPE_F32) {
            const auto f = [&](int i) { return __uint_as_float(w[i >> 2][i & 3]); };
            q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, f(0), f(1), s, 0);
            q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, f(2), f(3), s, 1);
            q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, f(4), f(5), s, 2);
            q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, f(6), f(7), s, 3);
        } else if constexpr (DT == MOE_DTYPE_BF16) {
            const auto f = [&](int i) { return __builtin_bit_cast(moe_bf16x2, (uint32_t)w[0][i]); };
            q = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(q, f(0), s, 0);
            q = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(q, f(1), s, 1);
            q = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(q, f(2), s, 2);
            q = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(q, f(3), s, 3);
        } else {
            const auto f = [&](int i) { return __builtin_bit_cast(moe_f16x2, (uint32_t)w[0][i]); };
            q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(q, f(0), s, 0);
            q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(q, f(1), s, 1);
            q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(q, f(2), s, 2);
            q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(q, f(3), s, 3);
        }
        return q;
    }
};

// Bytes of the values in memory.
__host__ __device__ constexpr int size_of(int dt) { return dt == MOE_DTYPE_F32 ? 4 : 2; }

// Block b's byte of the eight of its row and step. With a row's last block also those that fill its step, with 1.0: they meet
// codes of zero in the products, whose product with a NaN would be one.
__device__ __forceinline__ void write_exponent(uint8_t* s, int b, uint32_t e, bool last) {
    s[mx4_byte(b)] = (uint8_t)e;
    if (last)
        for (int p = b + 1; p < 8; ++p) s[mx4_byte(p)] = 127;
}

// One item: 8 columns of a row, its 4-lane neighbours the rest of its block: a block's largest magnitude is two DPP steps away, loads
// are 16 bytes a lane (fp32: two of them), and nothing is read twice. Bound by memory: [14336, 4096] bf16 29 us (149 MB, 5.1 TB/s, the
// rate of a large copy), [5760, 2880] fp32 13 us (75 MB); 5 rows 2.5 us, the launch.
template <int DT>
__global__ void __launch_bounds__(256) k_mx4_quantize(const char* x, int64_t ld, uint32_t items, uint32_t per_row, uint32_t row0,
                                                      uint32_t rows, int64_t scale_stride, uint8_t* codes, uint8_t* scales) {
    const uint32_t i = blockIdx.x * 256 + threadIdx.x;
    if (i >= items) return;   // items % 4 == 0: a block's four lanes leave together
    const uint32_t r = i / per_row, c = i - r * per_row;
    const uint32_t row = row0 + r, g = row / rows, n = row - g * rows;
    Eight<DT> v;
    v.load(x + ((int64_t)row * ld + c * 8) * size_of(DT));
    const uint32_t e = exponent4(max4(v.top()));
    const uint32_t q = v.codes(e - 1 < 254 ? e : 127);
    *(uint32_t*)(codes + ((int64_t)row * per_row + c) * 4) = e - 1 < 254 ? q : 0;
    if ((c & 3) == 0) {
        const uint32_t b = c >> 2;
        uint8_t* s = scales + g * scale_stride + ((int64_t)(b >> 3) * rows + n) * 8;
        write_exponent(s, b & 7, e, c + 4 == per_row);
    }
}

// The same items. Bound by memory too: [14336, 4096] to bf16 23.5 us (149 MB; its writes go past 5.1 TB/s), [5760, 2880] to fp32 14.
template <int DT>
__global__ void __launch_bounds__(256) k_mx4_dequantize(const uint8_t* codes, const uint8_t* scales, uint32_t items,
                                                        uint32_t per_row, uint32_t row0, uint32_t rows, int64_t scale_stride,
                                                        char* out) {
    const uint32_t i = blockIdx.x * 256 + threadIdx.x;
    if (i >= items) return;
    const uint32_t r = i / per_row, c = i - r * per_row;
    const uint32_t row = row0 + r, g = row / rows, n = row - g * rows, b = c >> 2;
    const uint32_t e = scales[g * scale_stride + ((int64_t)(b >> 3) * rows + n) * 8 + mx4_byte(b & 7)];
    const int64_t at = (int64_t)row * per_row + c;
    const uint32_t q = *(const uint32_t*)(codes + at * 4);
    // codes as fp32 (exact), then the power of two: 2^-127 is subnormal, and 255 stands for NaN
    const float s = e == 255 ? __uint_as_float(0x7fc00000u) : ldexpf(1.f, (int)e - 127);
    f32x2 v[4];
    v[0] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, 1.f, 0);
    v[1] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, 1.f, 1);
    v[2] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, 1.f, 2);
    v[3] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, 1.f, 3);
    float f[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = v[j >> 1][j & 1] * s;
    if constexpr (DT == MOE_DTYPE_F32) {
        ((f32x4*)out)[2 * at] = (f32x4){f[0], f[1], f[2], f[3]};
        ((f32x4*)out)[2 * at + 1] = (f32x4){f[4], f[5], f[6], f[7]};
    } else {
        constexpr bool H = DT == MOE_DTYPE_F16;
        ((u32x4*)out)[at] = (u32x4){pack16<H>(f[0], f[1]), pack16<H>(f[2], f[3]), pack16<H>(f[4], f[5]), pack16<H>(f[6], f[7])};
    }
}

// Rows that a launch takes: its items are counted in 32 bits.
static int64_t rows_at_once(int64_t rows, int64_t per_row) {
    const int64_t fit = ((int64_t)1 << 31) / per_row;
    return rows < fit ? rows : fit;
}

int launch_mx4_quantize(const void* x, int64_t ld, int64_t G, int64_t rows, int64_t K, int dtype, Mx4 out, hipStream_t st) {
    const int64_t all = G * rows, per_row = K / 8, step = rows_at_once(all, per_row), stride = (int64_t)mx4_steps(K) * rows * 8;
    for (int64_t r = 0; r < all; r += step) {
        const uint32_t items = (uint32_t)((all - r < step ? all - r : step) * per_row);
        auto go = [&](auto kernel) {
            kernel<<<(items + 255) / 256, 256, 0, st>>>((const char*)x, ld, items, (uint32_t)per_row, (uint32_t)r, (uint32_t)rows, stride,
                                                        out.codes, out.scales);
        };
        if (dtype == MOE_DTYPE_F32) go(k_mx4_quantize<MOE_DTYPE_F32>);
        else if (dtype == MOE_DTYPE_F16) go(k_mx4_quantize<MOE_DTYPE_F16>);
        else go(k_mx4_quantize<MOE_DTYPE_BF16>);
        if (hipGetLastError() != hipSuccess) return MOE_ERR_LAUNCH;
    }
    return MOE_OK;
}

int launch_mx4_dequantize(const uint8_t* codes, const uint8_t* scales, int64_t G, int64_t rows, int64_t K, int dtype, void* out,
                          hipStream_t st) {
    const int64_t all = G * rows, per_row = K / 8, step = rows_at_once(all, per_row), stride = (int64_t)mx4_steps(K) * rows * 8;
    for (int64_t r = 0; r < all; r += step) {
        const uint32_t items = (uint32_t)((all - r < step ? all - r : step) * per_row);
        auto go = [&](auto kernel) {
            kernel<<<(items + 255) / 256, 256, 0, st>>>(codes, scales, items, (uint32_t)per_row, (uint32_t)r, (uint32_t)rows, stride,
                                                        (char*)out);
        };
        if (dtype == MOE_DTYPE_F32) go(k_mx4_dequantize<MOE_DTYPE_F32>);
        else if (dtype == MOE_DTYPE_F16) go(k_mx4_dequantize<MOE_DTYPE_F16>);
        else go(k_mx4_dequantize<MOE_DTYPE_BF16>);
        if (hipGetLastError() != hipSuccess) return MOE_ERR_LAUNCH;
    }
    return MOE_OK;
}

// Sums of 16-bit rows by group: a workgroup 256 columns (8 to a lane, 32 lanes a row) of a piece of a group's rows, 8 of them at a
// time, the 8 partial sums joined in LDS in order. Bound by the one read of dy: 4444 x 5760 of 32 groups 10.5 us (4.8 TB/s), 32768 x
// 1536 of 128 17 us (5.9), 4096 x 4096 of one 7.2 us. (The weight gradient's product with columns of zeros: 27, 37, 50.)
constexpr int SUM_COLS = 256, SUM_ROWS = 8;
template <bool F16>
__global__ void __launch_bounds__(256) k_mx4_sums(const MmArgs g, int parts, float* out) {
    __shared__ float sm[SUM_ROWS][SUM_COLS];
    const int e = blockIdx.y, z = blockIdx.z, c = threadIdx.x & 31, r = threadIdx.x >> 5, j = blockIdx.x * SUM_COLS + c * 8;
    int lo, hi;
    group_of<MM_FWD>(g, e, lo, hi);
    const int n = ((hi - lo) / parts + ((hi - lo) % parts > 0) + SUM_ROWS - 1) / SUM_ROWS * SUM_ROWS;   // rows of a piece
    const int64_t first = lo + (int64_t)z * n, end = min((int64_t)hi, first + n);
    float v[8] = {};
    if (j < g.J) {
        const uint16_t* p = (const uint16_t*)g.a + j;
        const auto add = [&](u32x4 w) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[2 * i] += un16<F16>(w[i]);
                v[2 * i + 1] += un16<F16>(w[i] >> 16);
            }
        };
        int64_t i = first + r;
        for (; i + 7 * SUM_ROWS < end; i += 8 * SUM_ROWS) {
            u32x4 w[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) w[u] = *(const u32x4*)(p + (i + u * SUM_ROWS) * g.lda);
#pragma unroll
            for (int u = 0; u < 8; ++u) add(w[u]);
        }
        for (; i < end; i += SUM_ROWS) add(*(const u32x4*)(p + i * g.lda));
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) *(f32x4*)(&sm[r][c * 8 + 4 * i]) = (f32x4){v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]};
    __syncthreads();
    const int col = blockIdx.x * SUM_COLS + threadIdx.x;
    if (col >= g.J) return;
    float s = 0.f;
#pragma unroll
    for (int u = 0; u < SUM_ROWS; ++u) s += sm[u][threadIdx.x];
    if (parts > 1) out[((int64_t)z * g.E + e) * g.J + col] = s;
    else ((uint16_t*)g.y)[(int64_t)e * g.J + col] = (uint16_t)pack16<F16>(s, 0.f);
}
template <bool F16>
__global__ void __launch_bounds__(256) k_mx4_join_sums(const float* sums, int parts, int64_t n, uint16_t* y) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    float s = 0.f;
#pragma unroll 8
    for (int z = 0; z < parts; ++z) s += sums[z * n + i];
    y[i] = (uint16_t)pack16<F16>(s, 0.f);
}

// Pieces so that about 512 workgroups have 64 rows or more each: one group of 4096 rows would have 16 workgroups of its columns.
// (About 1024: a join where 736 workgroups do without, 4444 x 5760 of 32 groups 12.3 us.)
int mx4_sum_parts(int64_t M, int64_t E, int64_t N) {
    const int64_t wgs = E * ((N + SUM_COLS - 1) / SUM_COLS), rows = M / E;
    int parts = 1;
    while (wgs * parts < 512 && rows >= 128 * parts) parts *= 2;
    return parts;
}

int launch_mx4_sums(const MmArgs& a, int parts, float* sums, hipStream_t st) {
    const dim3 grid((unsigned)((a.J + SUM_COLS - 1) / SUM_COLS), (unsigned)a.E, (unsigned)parts);
    auto go = [&](auto f16) {
        constexpr bool F16 = decltype(f16)::value;
        k_mx4_sums<F16><<<grid, 256, 0, st>>>(a, parts, sums);
        if (parts > 1) {
            const int64_t n = (int64_t)a.E * a.J;
            k_mx4_join_sums<F16><<<(unsigned)((n + 255) / 256), 256, 0, st>>>(sums, parts, n, (uint16_t*)a.y);
        }
    };
    if (a.f16) go(std::true_type{});
    else go(std::false_type{});
    return hipGetLastError() == hipSuccess ? MOE_OK : MOE_ERR_LAUNCH;
}

// Both operands MXFP4, 16 x 16 outputs and 128 of k: lane l holds 32 codes of row l & 15 (k from 32 (l >> 4) on), and in byte B of
// its word their exponent.
template <int B>
__device__ __forceinline__ f32x4 mma16(s16x8 a, uint32_t sa, s16x8 b, uint32_t sb, f32x4 c) {
    typedef int i32x4 __attribute__((ext_vector_type(4)));
    const auto wide = [](s16x8 v) {   // the upper half is not read
        const i32x4 w = __builtin_bit_cast(i32x4, v);
        return __builtin_shufflevector(w, w, 0, 1, 2, 3, -1, -1, -1, -1);
    };
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wide(a), wide(b), c, 4, 4, B, (int)sa, B, (int)sb);
}

// Few rows: a wave multiplies 16 rows of the weights by up to 16 NT rows of x, with the weights' codes straight from memory as the
// matrix instruction's first operand. ks waves of a workgroup share the steps of K, and their sums meet in LDS, in the waves'
// order. FUSE: x's rows are quantised here first, while the first weights are on their way; else their codes come from memory too.
// Bound by the weights' bytes and the latency of the first ones: AHEAD steps of a wave are loaded together. One row, [14336, 4096]
// 8.3 us (31 MB, 3.8 TB/s), [4096, 4096] 4.5; 8 of 128 experts, [1536, 2048], 7.6 (13 MB: a chain of index list, row, weights).
// FUSE: to quantise one row needs a launch of 2.5 us in front and its codes back from memory; with 4 rows every workgroup quantises
// 4 K numbers for itself while its weights come, with more that takes longer than the launch. Their codes have to fit LDS.
// Workgroups go by slot, not by group (as k_mm_rows): the one at a group's first slot does the group.
constexpr int MXR_WAVES = 8;
template <bool F16, bool FUSE, int NT>
__global__ void __launch_bounds__(64 * MXR_WAVES) k_mx4_rows(const MmArgs g, const uint16_t* x16, int64_t ldx, int ks) {
    static_assert(!FUSE || NT == 1, "");
    constexpr int ROWS = FUSE ? MX4_FUSE : 16 * NT, AHEAD = 4;
    extern __shared__ __attribute__((aligned(16))) uint8_t sx[];   // FUSE: codes [MX4_FUSE, K / 2], exponents [MX4_FUSE, steps, 8]
    __shared__ f32x4 sums[MXR_WAVES][NT][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), part = wave % ks;
    const int l = lane & 15, q = lane >> 4;
    const int wg0 = blockIdx.x * 16 * (MXR_WAVES / ks), n0 = wg0 + wave / ks * 16, p = blockIdx.y;
    int e = 0, lo = 0, hi = g.M;
    if (g.offsets) {
        e = -1;   // the group whose first slot is p; 256 groups' offsets at once
        for (int base = 0; base < g.E && e < 0; base += 256) {
            int a[4], b[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) group_of<MM_FWD>(g, min(base + 64 * u + lane, g.E - 1), a[u], b[u]);
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const uint64_t hit = __ballot(base + 64 * u + lane < g.E && a[u] == p && b[u] > a[u]);
                if (hit && e < 0) {
                    e = base + 64 * u + __builtin_ctzll(hit);
                    lo = p;
                    hi = __builtin_amdgcn_readlane(b[u], __builtin_ctzll(hit));
                }
            }
        }
        if (e < 0) {
            if (!g.fill) return;
            int a, b;
            group_of<MM_FWD>(g, g.E - 1, a, b);
            if (p < b) return;
            const int n = wg0 + threadIdx.x;
            if (threadIdx.x < 16 * (MXR_WAVES / ks) && n < g.J) {
                const int64_t at = (int64_t)p * g.J + n;
                if (g.ydt == MOE_DTYPE_F32) ((float*)g.y)[at] = 0.f;
                else ((uint16_t*)g.y)[at] = 0;
            }
            return;
        }
    }
    const int K = g.R * 4, KB = K / 2, steps = (K + 255) / 256;
    const int n = min(n0 + l, g.J - 1);   // rows past the last: multiplied, not stored
    const uint8_t* wc = (const uint8_t*)g.b + ((int64_t)e * g.J + n) * KB + q * 16;
    const uint8_t* ws = g.sb + ((int64_t)e * steps * g.J + n) * 8 + (q & 1) * 4;
    const int sh = (q >> 1) * 8;   // the first half step's exponent in byte 0, the second's in byte 2
    s16x8 w[AHEAD][2];
    uint32_t we[AHEAD];
    const s16x8 zero = {};
    auto load_w = [&](int s0) {
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            const int s = s0 + u * ks;
            if (s >= steps) break;
#pragma unroll
            for (int c = 0; c < 2; ++c)
                w[u][c] = s * 256 + c * 128 + q * 32 < K ? *(const s16x8*)(wc + (int64_t)s * 128 + c * 64) : zero;
            we[u] = *(const uint32_t*)(ws + (int64_t)s * g.J * 8) >> sh;
        }
    };
    if (n0 < g.J) load_w(part);
    for (int m0 = lo; m0 < hi; m0 += ROWS) {
        const int rows = min(hi - m0, ROWS);
        int src[NT];   // this lane's rows of x
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            src[i] = -1;
            if (16 * i + l < rows) {
                src[i] = g.arows ? g.arows[m0 + 16 * i + l] : m0 + 16 * i + l;
                if ((uint32_t)src[i] >= (uint32_t)g.a_n) src[i] = -1;
            }
        }
        if constexpr (FUSE) {
            if (m0 > lo) __syncthreads();   // the last rows are multiplied
            const int per_row = K / 8;
            for (int i = threadIdx.x; i < rows * per_row; i += 64 * MXR_WAVES) {   // a block's four lanes together: K % 32 == 0
                const int r = i / per_row, c = i - r * per_row, b = c >> 2;
                const int s = g.arows ? g.arows[m0 + r] : m0 + r;
                Eight<F16 ? MOE_DTYPE_F16 : MOE_DTYPE_BF16> v;
                const bool live = (uint32_t)s < (uint32_t)g.a_n;
                v.load((const char*)(x16 + (live ? s : 0) * ldx + c * 8));
                const uint32_t ex = exponent4(max4(v.top()));
                const uint32_t code = v.codes(ex - 1 < 254 ? ex : 127);
                *(uint32_t*)(sx + (r * per_row + c) * 4) = live && ex - 1 < 254 ? code : 0;
                if ((c & 3) == 0) write_exponent(sx + MX4_FUSE * KB + (r * steps + (b >> 3)) * 8, b & 7, live ? ex : 127, c + 4 == per_row);
            }
            __syncthreads();
        }
        f32x4 acc[NT] = {};
        if (n0 < g.J)
            for (int s0 = part; s0 < steps; s0 += AHEAD * ks) {
                if (s0 != part || m0 > lo) load_w(s0);
                s16x8 x[AHEAD][NT][2];
                uint32_t xe[AHEAD][NT];
#pragma unroll
                for (int u = 0; u < AHEAD; ++u) {
                    const int s = s0 + u * ks;
                    if (s >= steps) break;
#pragma unroll
                    for (int i = 0; i < NT; ++i) {
                        x[u][i][0] = x[u][i][1] = zero;
                        xe[u][i] = 0x7f7f7f7f;
                        if (src[i] < 0) continue;
                        const uint8_t* xc = FUSE ? sx + l * KB : (const uint8_t*)g.a + (int64_t)src[i] * KB;
                        const uint8_t* xs = FUSE ? sx + MX4_FUSE * KB + (l * steps + s) * 8 : g.sa + ((int64_t)s * g.a_n + src[i]) * 8;
#pragma unroll
                        for (int c = 0; c < 2; ++c)
                            if (s * 256 + c * 128 + q * 32 < K) x[u][i][c] = *(const s16x8*)(xc + s * 128 + c * 64 + q * 16);
                        xe[u][i] = *(const uint32_t*)(xs + (q & 1) * 4) >> sh;
                    }
                }
#pragma unroll
                for (int u = 0; u < AHEAD; ++u) {
                    if (s0 + u * ks >= steps) break;
#pragma unroll
                    for (int i = 0; i < NT; ++i) {
                        acc[i] = mma16<0>(w[u][0], we[u], x[u][i][0], xe[u][i], acc[i]);
                        acc[i] = mma16<2>(w[u][1], we[u], x[u][i][1], xe[u][i], acc[i]);
                    }
                }
            }
        if (ks > 1) {
#pragma unroll
            for (int i = 0; i < NT; ++i) sums[wave][i][lane] = acc[i];
            __syncthreads();
        }
        const int j = n0 + 4 * q;   // four neighbours of J (a multiple of 8)
        if (part == 0 && j < g.J) {
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                if (16 * i + l >= rows) continue;
                f32x4 v = acc[i];
                for (int k = 1; k < ks; ++k) v += sums[wave + k][i][lane];
                const int64_t at = (int64_t)(m0 + 16 * i + l) * g.J + j;
                if (g.epi.bias) v += load4<F16>(g.epi.bias, (int64_t)e * g.J + j);
                if (g.epi.z) *(u32x2*)((uint16_t*)g.epi.z + at) = (u32x2){pack16<F16>(v[0], v[1]), pack16<F16>(v[2], v[3])};
#pragma unroll
                for (int c = 0; c < 4; ++c) v[c] = lin_act(g.epi.act, v[c]);
                if (g.epi.residual) v += load4<F16>(g.epi.residual, at);
                if (g.ydt == MOE_DTYPE_F32) *(f32x4*)((float*)g.y + at) = v;
                else *(u32x2*)((uint16_t*)g.y + at) = (u32x2){pack16<F16>(v[0], v[1]), pack16<F16>(v[2], v[3])};
            }
        }
        if (ks > 1 && m0 + ROWS < hi) __syncthreads();   // the sums are read
    }
}

int launch_mx4_rows(const MmArgs& a, const void* x16, int64_t ldx, hipStream_t st) {
    const int64_t K = (int64_t)a.R * 4, steps = mx4_steps(K), blocks = (int64_t)((a.J + 15) / 16) * (a.offsets ? a.M : 1);
    // Waves that share K, until 2048 of them have work (us with 1024, 2048, 4096: one row, [4096, 4096], 6.3, 5.6, 5.6, [4096, 14336]
    // 13.4, 10.9, 11.0, [14336, 4096] 10.0, 9.4, 12.0; 8 of 128 experts, [1536, 2048], 6.0, 6.1, 7.6).
    int ks = 1;
    while (ks < MXR_WAVES && ks < steps && blocks * ks < 2048) ks *= 2;
    const int rows = 16 * (MXR_WAVES / ks);
    const dim3 grid((unsigned)((a.J + rows - 1) / rows), a.offsets ? (unsigned)a.M : 1);
    const size_t lds = x16 ? (size_t)MX4_FUSE * (K / 2 + steps * 8) : 0;
    auto go = [&](auto f16) {
        constexpr bool F16 = decltype(f16)::value;
        auto run = [&](auto kernel) { kernel<<<grid, 64 * MXR_WAVES, lds, st>>>(a, (const uint16_t*)x16, ldx, ks); };
        if (x16) run(k_mx4_rows<F16, true, 1>);
        else if (a.offsets || a.M <= 16) run(k_mx4_rows<F16, false, 1>);
        else run(k_mx4_rows<F16, false, 2>);
    };
    if (a.f16) go(std::true_type{});
    else go(std::false_type{});
    return hipGetLastError() == hipSuccess ? MOE_OK : MOE_ERR_LAUNCH;
}

}  // namespace moe
