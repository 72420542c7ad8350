// Products of 16-bit matrices on the matrix cores, by ragged groups of rows (one group per expert, or one in all):
//   forward  y[p][n]     = sum_k x[p][k] w[e][n][k]        p in group e
//   dx       dx[p][k]    = sum_n dy[p][n] w[e][n][k]
//   dw       dw[e][n][k] = sum_p dy[p][n] x[p][k]           p over group e
// One tile kernel computes C[i][j] = sum_r A[i][r] B[j][r] for all three; an operand is stored either with r contiguous
// (x and w in the forward pass, dy in dx) or with its own index contiguous (w in dx, both operands in dw).
#pragma once
#include "moe_common.h"
#include "moe_internal.h"

namespace moe {

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t srd_t __attribute__((ext_vector_type(4)));   // a raw buffer descriptor

enum MmMode { MM_FWD = 0, MM_DX = 1, MM_DW = 2 };

template <bool F16>
__device__ __forceinline__ f32x4 mma(s16x8 a, s16x8 b, f32x4 c) {
    if constexpr (F16)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
// The same with the sums held in the accumulation registers for good: the largest tile's 256 sums fill that half of the
// register file, and left to itself the compiler copies a third of them between the halves in every step. s_nop: a vector
// instruction may have written an operand just before (2 wait states; they pass while the last product still runs). The
// sums are read only after drain(), and added to again no sooner than 8 products later.
template <bool F16>
__device__ __forceinline__ void mma_acc(s16x8 a, s16x8 b, f32x4& c) {
    if constexpr (F16) asm("s_nop 1\n\tv_mfma_f32_16x16x32_f16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
    else asm("s_nop 1\n\tv_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
}
template <bool F16>
__device__ __forceinline__ void mma_vec(s16x8 a, s16x8 b, f32x4& c) {   // the same, sums in ordinary registers
    if constexpr (F16) asm("s_nop 1\n\tv_mfma_f32_16x16x32_f16 %0, %1, %2, %0" : "+v"(c) : "v"(a), "v"(b));
    else asm("s_nop 1\n\tv_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+v"(c) : "v"(a), "v"(b));
}
__device__ __forceinline__ void drain() { asm volatile("s_nop 15\n\ts_nop 15" ::: "memory"); }
template <bool F16>
__device__ __forceinline__ uint32_t pack16(float a, float b) {
    if constexpr (F16) {
        return (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)a) | (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)b) << 16;
    } else {
        const moe_bf16x2 v = {(__bf16)a, (__bf16)b};
        return __builtin_bit_cast(uint32_t, v);
    }
}
template <bool F16>
__device__ __forceinline__ float un16(uint32_t h) {   // the low half
    if constexpr (F16) return (float)__builtin_bit_cast(_Float16, (uint16_t)h);
    return __uint_as_float(h << 16);
}

// Buffer descriptor of `bytes` from p on; loads past the end deliver zeros. Offsets from MM_OOB on are always past it.
#define MM_OOB 0xC0000000u
__device__ __forceinline__ srd_t srd_of(const void* p, int64_t bytes) {
    const uint64_t a = (uint64_t)p;
    const uint32_t n = bytes < 0 ? 0u : bytes > (int64_t)MM_OOB ? MM_OOB : (uint32_t)bytes;
    srd_t s;
    s[0] = __builtin_amdgcn_readfirstlane((uint32_t)a);
    s[1] = __builtin_amdgcn_readfirstlane((uint32_t)(a >> 32) & 0xffffu);
    s[2] = __builtin_amdgcn_readfirstlane(n);
    s[3] = 0x00027000u;
    return s;
}
// 64 lanes x 16 bytes from buffer offset `off` of each lane to LDS at lds + 16 lane. Asynchronous: counted in vmcnt, which
// the compiler does not know of (its own waits for other loads can only become stricter). s_nop: M0 and scalar operands
// written just before.
__device__ __forceinline__ void dma16(srd_t s, uint32_t off, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(lds), "v"(off), "s"(s) : "memory", "m0");
}
template <int N>
__device__ __forceinline__ void wait_vm() {
    static_assert(N >= 0 && N < 64, "vmcnt has 6 bits");
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
__device__ __forceinline__ void wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }
__device__ __forceinline__ void barrier_raw() { asm volatile("s_barrier" ::: "memory"); }

// One operand's tile in LDS: X rows of the operand's own index x 64 of r, 128 X bytes, filled in units of 1024 bytes
// (one dma16 each, X / 8 units, unit i * 4 + wave by a wave's i-th load).
//   r contiguous:  row x at 128 x, its 16-byte pieces XORed with x & 7, so the 16 rows that a fragment read touches
//                  spread over the banks;
//   x contiguous:  r-row at 2 X r, its 32-byte granules (16 x) XORed with bits of r, so the 4 x 4 r-rows that a
//                  transposing read touches do.
template <int X>
__device__ __forceinline__ int gran_swz(int r) {
    if constexpr (X >= 256) return (r & 3) | ((r >> 3) & 3) << 2;
    if constexpr (X == 128) return (r & 3) | ((r >> 3) & 1) << 2;
    return ((r >> 1) & 1) | ((r >> 3) & 1) << 1;
}

template <bool XC, int X>   // XC: x contiguous
struct Operand {
    static constexpr int UNITS = X / 32;   // dma16 per wave and step
    static constexpr int BYTES = X * 128;
    // what lane `lane` fetches for unit u: its row (x or r) and first column (r or x) inside the tile
    static __device__ __forceinline__ void at(int u, int lane, int& row, int& col) {
        if constexpr (!XC) {
            row = 8 * u + (lane >> 3);
            col = ((lane & 7) ^ (row & 7)) * 8;
        } else {
            constexpr int PC = X / 8;   // 16-byte pieces per r-row
            row = u * (64 / PC) + lane / PC;
            const int c = lane % PC;
            col = (((c >> 1) ^ gran_swz<X>(row)) & (X / 16 - 1)) * 16 + (c & 1) * 8;
        }
    }
    // LDS byte offset of the fragment of x tile row block xb (16 rows), r half kk; !XC: one 16-byte read; XC: two
    // transposing 8-byte reads at addr and addr + 4 r-rows
    static __device__ __forceinline__ uint32_t frag(int xb, int lane) {
        const int l = lane & 15, q = lane >> 4;
        if constexpr (!XC) {
            return (uint32_t)((16 * xb + l) * 128 + ((q ^ (l & 7)) * 16));
        } else {
            const int r = 8 * q + (l >> 2);
            return (uint32_t)(r * 2 * X + ((xb ^ gran_swz<X>(r)) & (X / 16 - 1)) * 32 + (l & 3) * 8);
        }
    }
    static __device__ __forceinline__ s16x8 read(const char* sm, uint32_t f, int kk) {
        if constexpr (!XC) {
            return *(const s16x8*)(sm + (f ^ (kk * 64)));   // piece q + 4 kk, XORed
        } else {
            typedef __attribute__((address_space(3))) s16x4 lds4;
            const char* p = sm + f + kk * 32 * 2 * X;
            const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)p);
            const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(p + 4 * 2 * X));
            return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
        }
    }
};

struct MmEpi {
    const void* bias;        // [E, J] of the operands' type, or null
    const void* residual;    // [M, J] of the operands' type, or null
    void* z;                 // [M, J] of the operands' type: the sums with bias, before the activation; or null
    int act;                 // MOE_LIN_*
};

struct MmArgs {
    const void* a;           // forward: x; dx, dw: dy
    const void* b;           // forward, dx: w [E, N, K]; dw: x
    const int32_t* offsets;  // [E + 1], or null: one group of M rows
    const int32_t* arows;    // row of a of each slot, or null: the slot itself
    const int32_t* brows;    // dw: the same for b
    void* y;
    void* dbias;             // dw: [E, N] of the operands' type, or null
    int64_t M;               // slots
    int64_t a_n, b_n;        // rows of a and (dw) b
    int64_t lda, ldb;        // elements between rows; ldb of forward and dx: K
    int E, I, J, R;          // dw: I = N, J = K; forward: J = N, R = K; dx: J = K, R = N
    int f16, ydt, fill;      // ydt: MOE_DTYPE_*; fill: rows behind the last group are set to zero
    MmEpi epi;
};

// The slots of group e, inside [0, M) whatever offsets hold.
__device__ __forceinline__ void group_of(const MmArgs& a, int e, int64_t& lo, int64_t& hi) {
    if (!a.offsets) {
        lo = 0;
        hi = a.M;
        return;
    }
    const int64_t p = e ? a.offsets[e] : 0, q = a.offsets[e + 1];
    lo = p < 0 ? 0 : p > a.M ? a.M : p;
    hi = q < lo ? lo : q > a.M ? a.M : q;
}

struct MmTile {
    int e;          // group; E: the rows behind the last one
    int64_t lo;     // forward, dx: first slot of the tile; dw: of the group
    int64_t cnt;    // dw: slots of the group
    int i0, rows;   // dw: first output row; valid rows, <= BI
    int j0;
};

// Tile `id` of the contiguous runs that the 8 XCDs are dealt (workgroup b runs on XCD b % 8), or -1: tiles that share an
// expert's weights share an L2.
__device__ __forceinline__ int64_t xcd_tile(int64_t tiles, int b) {
    const int xcd = b & 7, at = b >> 3, rem = (int)(tiles & 7);
    const int64_t q = tiles >> 3;
    return at >= q + (xcd < rem) ? -1 : xcd * q + min(xcd, rem) + at;
}

// Which tile a workgroup computes. Every wave scans the groups' row counts, 64 at a time: the number of tiles is known
// only on the device, so the grid is an upper bound and surplus workgroups leave here. Inside a group tiles run down up to
// 4 row tiles before the next column tile.
template <int BI, int BJ>
__device__ __forceinline__ bool find_tile(const MmArgs& a, int b, MmTile& t) {
    const int lane = threadIdx.x & 63, nj = (a.J + BJ - 1) / BJ;
    const int G = a.E + (a.fill && a.offsets ? 1 : 0);   // the last pseudo group: rows to fill
    auto span = [&](int e, int64_t& lo, int64_t& hi) {
        group_of(a, min(e, a.E - 1), lo, hi);
        if (e == a.E) {
            lo = hi;
            hi = a.M;
        }
    };
    auto tiles_of = [&](int e) -> int {
        if (e >= G) return 0;
        int64_t lo, hi;
        span(e, lo, hi);
        return (int)((hi - lo + BI - 1) / BI);
    };
    const int t0 = tiles_of(lane), scan0 = wave_incl_scan(t0);
    int total = __builtin_amdgcn_readlane(scan0, 63);
    for (int base = 64; base < G; base += 64) total += __builtin_amdgcn_readlane(wave_incl_scan(tiles_of(base + lane)), 63);
    const int64_t id = xcd_tile((int64_t)total * nj, b);
    if (id < 0) return false;
    int before = 0;
    for (int base = 0; base < G; base += 64) {
        const int n = base ? tiles_of(base + lane) : t0, s = base ? wave_incl_scan(n) : scan0;
        const uint64_t hit = __ballot((int64_t)(before + s) * nj > id);
        if (hit) {
            const int l = __builtin_ctzll(hit);
            const int nr = __builtin_amdgcn_readlane(n, l), first = before + __builtin_amdgcn_readlane(s, l) - nr;
            const int64_t local = id - (int64_t)first * nj;
            const int sup = (int)(local / (4 * nj)), in = (int)(local - (int64_t)sup * 4 * nj), h = min(4, nr - 4 * sup);
            const int rt = 4 * sup + in % h;
            int64_t lo, hi;
            t.e = base + l;
            span(t.e, lo, hi);
            t.j0 = in / h * BJ;
            t.lo = lo + (int64_t)rt * BI;
            t.rows = (int)min((int64_t)BI, hi - t.lo);
            t.i0 = 0;
            t.cnt = 0;
            return true;
        }
        before += __builtin_amdgcn_readlane(s, 63);
    }
    return false;
}
// dw: group by group, 4 row tiles (n) down before the next column tile (k)
template <int BI, int BJ>
__device__ __forceinline__ bool find_tile_dw(const MmArgs& a, int b, MmTile& t) {
    const int ni = (a.I + BI - 1) / BI, nj = (a.J + BJ - 1) / BJ;
    const int64_t id = xcd_tile((int64_t)a.E * ni * nj, b);
    if (id < 0) return false;
    t.e = (int)(id / (ni * nj));
    const int local = (int)(id - (int64_t)t.e * ni * nj), sup = local / (4 * nj), in = local - sup * 4 * nj;
    const int h = min(4, ni - 4 * sup);
    int64_t hi;
    group_of(a, t.e, t.lo, hi);
    t.cnt = hi - t.lo;
    t.i0 = (4 * sup + in % h) * BI;
    t.j0 = in / h * BJ;
    t.rows = min(BI, a.I - t.i0);
    return true;
}

__device__ __forceinline__ float lin_act(int act, float z) {
    if (act == MOE_LIN_SILU) return z * sigmoid_fast(z);
    if (act == MOE_LIN_GELU) return z * sigmoid_fast(1.5957691216057308f * (z + 0.044715f * z * z * z));
    return z;
}
template <bool F16>
__device__ __forceinline__ f32x4 load4(const void* p, int64_t i) {
    const u32x2 w = *(const u32x2*)((const uint16_t*)p + i);
    return (f32x4){un16<F16>(w[0]), un16<F16>(w[0] >> 16), un16<F16>(w[1]), un16<F16>(w[1] >> 16)};
}

// A tile of 32 FA x 32 FB outputs, 4 waves as 2 x 2, each FA x FB fragments of 16 x 16 (wave (wi, wj): row blocks
// 2 f + wi, column blocks wj FB + h), r in steps of 64 through ST stages of LDS. The matrix instruction takes B's rows as
// its first operand, so a lane's four sums are neighbours in j, the output's contiguous index.
// A tile with few valid rows runs the same loop on NF = FA, FA / 2, .. 1 row blocks per wave (32 NF rows).
template <int MODE, bool F16, int FA, int FB, int ST, bool GATHER>
struct MmKernel {
    static constexpr bool ACC = FA * FB * 4 >= 256;   // sums pinned to the accumulation registers
    static constexpr bool AX = MODE == MM_DW, BX = MODE != MM_FWD;   // operand with its own index contiguous
    static constexpr int BI = 32 * FA, BJ = 32 * FB;
    using A = Operand<AX, BI>;
    using B = Operand<BX, BJ>;
    static constexpr int STAGE = A::BYTES + B::BYTES;

    template <int NF, bool FULL>   // FULL: bias, activation, residual and z
    static __device__ __forceinline__ void store(const MmArgs& g, const MmTile& t, f32x4 (&acc)[NF][FB], int lane, int wi, int wj) {
        const int l = lane & 15, q = lane >> 4;
        const int64_t row0 = MODE == MM_DW ? (int64_t)t.e * g.I + t.i0 : t.lo;
        const int jw = t.j0 + wj * FB * 16;
#pragma unroll
        for (int f = 0; f < NF; ++f) {
            const int i = 16 * (2 * f + wi) + l;
            const bool in = i < t.rows;
            const int64_t at = (row0 + i) * g.J;
#pragma unroll
            for (int h = 0; h < FB; h += 2) {
                f32x4 v[2] = {acc[f][h], acc[f][h + 1]};
                uint32_t zz[2][2];
                if constexpr (FULL) {
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        const int j = jw + 16 * (h + u) + 4 * q;
                        const bool ok = in && j < g.J;
                        if (g.epi.bias && ok) v[u] += load4<F16>(g.epi.bias, (int64_t)t.e * g.J + j);
                        if (g.epi.z) {
                            zz[u][0] = pack16<F16>(v[u][0], v[u][1]);
                            zz[u][1] = pack16<F16>(v[u][2], v[u][3]);
                        }
                        if (g.epi.act != MOE_LIN_NONE)
#pragma unroll
                            for (int c = 0; c < 4; ++c) v[u][c] = lin_act(g.epi.act, v[u][c]);
                        if (g.epi.residual && ok) v[u] += load4<F16>(g.epi.residual, at + j);
                    }
                }
                if (g.ydt == MOE_DTYPE_F32) {
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        const int j = jw + 16 * (h + u) + 4 * q;
                        if (in && j < g.J) *(f32x4*)((float*)g.y + at + j) = v[u];
                    }
                }
                // 16-bit rows: two column blocks change halves between neighbouring rows of lanes, so that a lane holds
                // eight neighbours and stores 16 bytes
                const int jj = jw + 16 * (h + (q & 1)) + 4 * (q & 2);
                auto put = [&](void* out, uint32_t a0, uint32_t a1, uint32_t b0, uint32_t b1) {
                    const auto s0 = __builtin_amdgcn_permlane16_swap(a0, b0, false, false);
                    const auto s1 = __builtin_amdgcn_permlane16_swap(a1, b1, false, false);
                    if (in && jj < g.J) *(u32x4*)((uint16_t*)out + at + jj) = (u32x4){s0[0], s1[0], s0[1], s1[1]};
                };
                if (g.ydt != MOE_DTYPE_F32)
                    put(g.y, pack16<F16>(v[0][0], v[0][1]), pack16<F16>(v[0][2], v[0][3]), pack16<F16>(v[1][0], v[1][1]),
                        pack16<F16>(v[1][2], v[1][3]));
                if constexpr (FULL)
                    if (g.epi.z) put(g.epi.z, zz[0][0], zz[0][1], zz[1][0], zz[1][1]);
            }
        }
    }

    template <int NF, bool DB>
    static __device__ __forceinline__ void run(const MmArgs& g, const MmTile& t, char* sm) {
        constexpr int LA = AX ? FA : NF, L = LA + FB;
        const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wi = wave & 1, wj = wave >> 1;
        const bool gath_a = MODE == MM_DW ? GATHER : g.arows != nullptr;
        constexpr bool gath_b = MODE == MM_DW && GATHER;
        const int64_t r_n = MODE == MM_DW ? t.cnt : g.R;
        const int steps = (int)((r_n + 63) / 64);
        const int64_t lda2 = g.lda * 2, ldb2 = g.ldb * 2;
        const int64_t step_a = AX ? (gath_a ? 0 : 64 * lda2) : 128, step_b = BX ? (gath_b ? 0 : 64 * ldb2) : 128;
        const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)sm;

        // where the operands begin, how many bytes may be read from there, and each lane's offsets
        const char *pa = (const char*)g.a, *pb = (const char*)g.b;
        int64_t na, nb;
        uint32_t offa[LA], offb[FB];
        int cola[LA], colb[FB], rowa[LA], rowb[FB];
#pragma unroll
        for (int i = 0; i < LA; ++i) A::at(i * 4 + wave, lane, rowa[i], cola[i]);
#pragma unroll
        for (int i = 0; i < FB; ++i) B::at(i * 4 + wave, lane, rowb[i], colb[i]);
        if constexpr (!AX) {
            if (gath_a) {
                na = (g.a_n - 1) * lda2 + (int64_t)g.R * 2;
            } else {
                pa += t.lo * lda2;
                na = (t.rows - 1) * lda2 + (int64_t)g.R * 2;
            }
#pragma unroll
            for (int i = 0; i < LA; ++i) {
                int64_t src = rowa[i];
                bool ok = src < t.rows;
                if (gath_a && ok) {
                    src = g.arows[t.lo + src];
                    ok = src >= 0 && src < g.a_n;
                }
                offa[i] = ok ? (uint32_t)(src * lda2 + cola[i] * 2) : MM_OOB;
            }
        } else {
            pa += (int64_t)t.i0 * 2 + (gath_a ? 0 : t.lo * lda2);
            na = ((gath_a ? g.a_n : t.cnt) - 1) * lda2 + (int64_t)(g.I - t.i0) * 2;
#pragma unroll
            for (int i = 0; i < LA; ++i)
                offa[i] = t.i0 + cola[i] < g.I ? (uint32_t)((gath_a ? 0 : rowa[i] * lda2) + cola[i] * 2) : MM_OOB;
        }
        if constexpr (!BX) {
            pb += ((int64_t)t.e * g.J + t.j0) * ldb2;
            nb = (int64_t)(min(BJ, g.J - t.j0) - 1) * ldb2 + (int64_t)g.R * 2;
#pragma unroll
            for (int i = 0; i < FB; ++i) offb[i] = t.j0 + rowb[i] < g.J ? (uint32_t)(rowb[i] * ldb2 + colb[i] * 2) : MM_OOB;
        } else {
            const int64_t base = MODE == MM_DX ? (int64_t)t.e * g.R : gath_b ? 0 : t.lo;
            pb += base * ldb2 + (int64_t)t.j0 * 2;
            nb = ((MODE == MM_DX ? g.R : gath_b ? g.b_n : t.cnt) - 1) * ldb2 + (int64_t)(g.J - t.j0) * 2;
#pragma unroll
            for (int i = 0; i < FB; ++i)
                offb[i] = t.j0 + colb[i] < g.J ? (uint32_t)((gath_b ? 0 : rowb[i] * ldb2) + colb[i] * 2) : MM_OOB;
        }

        f32x4 acc[NF][FB];
        f32x4 accb[DB ? NF : 1];
#pragma unroll
        for (int f = 0; f < NF; ++f)
#pragma unroll
            for (int h = 0; h < FB; ++h) acc[f][h] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int f = 0; f < (DB ? NF : 1); ++f) accb[f] = (f32x4){0.f, 0.f, 0.f, 0.f};

        uint32_t fra[NF], frb[FB];
#pragma unroll
        for (int f = 0; f < NF; ++f) fra[f] = A::frag(2 * f + wi, lane);
#pragma unroll
        for (int h = 0; h < FB; ++h) frb[h] = A::BYTES + B::frag(wj * FB + h, lane);

        // dw with gathered rows: the step's 64 source rows, one per lane
        int ia = -1, ib = -1;
        auto fetch_rows = [&](int s) {
            if constexpr (MODE == MM_DW) {
                const int64_t p = 64 * (int64_t)s + lane;
                if constexpr (GATHER) {
                    const bool in = p < r_n;
                    ia = !in ? -1 : g.arows ? g.arows[t.lo + p] : (int)(t.lo + p);
                    ib = !in ? -1 : g.brows ? g.brows[t.lo + p] : (int)(t.lo + p);
                }
            }
        };
        auto row_off = [&](int ids, int row, uint32_t off, int64_t n, int64_t ld2) -> uint32_t {
            const int src = __shfl(ids, row);
            return off < MM_OOB && (uint32_t)src < (uint64_t)n ? (uint32_t)(src * ld2) + off : MM_OOB;
        };
        auto load_a = [&](int s, srd_t d, int i) {
            uint32_t off = offa[i];
            if constexpr (!AX) {
                if (64 * s + cola[i] >= g.R) off = MM_OOB;
            } else {
                if (gath_a) off = row_off(ia, rowa[i], off, g.a_n, lda2);
            }
            dma16(d, off, lds0 + (uint32_t)((s % ST) * STAGE + (i * 4 + wave) * 1024));
        };
        auto load_b = [&](int s, srd_t d, int i) {
            uint32_t off = offb[i];
            if constexpr (!BX) {
                if (64 * s + colb[i] >= g.R) off = MM_OOB;
            } else {
                if (gath_b) off = row_off(ib, rowb[i], off, g.b_n, ldb2);
            }
            dma16(d, off, lds0 + (uint32_t)((s % ST) * STAGE + A::BYTES + (i * 4 + wave) * 1024));
        };
        auto srd_a = [&](int s) { return srd_of(pa + s * step_a, na - s * step_a); };
        auto srd_b = [&](int s) { return srd_of(pb + s * step_b, nb - s * step_b); };

        s16x8 ra[2][NF], rb[2][FB];
        auto read_a = [&](int set, int s, int kk, int f) { ra[set][f] = A::read(sm + (s % ST) * STAGE, fra[f], kk); };
        auto read_b = [&](int set, int s, int kk, int h) { rb[set][h] = B::read(sm + (s % ST) * STAGE, frb[h], kk); };
        auto mul = [&](int set, int f) {
#pragma unroll
            for (int h = 0; h < FB; ++h) {
                if constexpr (ACC) mma_acc<F16>(rb[set][h], ra[set][f], acc[f][h]);
                else acc[f][h] = mma<F16>(rb[set][h], ra[set][f], acc[f][h]);
            }
            if constexpr (DB) {
                const short one = F16 ? 0x3C00 : 0x3F80;
                const s16x8 ones = {one, one, one, one, one, one, one, one};
                if constexpr (ACC) mma_vec<F16>(ones, ra[set][f], accb[f]);
                else accb[f] = mma<F16>(ones, ra[set][f], accb[f]);
            }
        };

        // Steps past the last one are loaded too, as zeros (their descriptors or columns are past the end), and read but
        // not used: the loop has no branches and waits for the same number of loads in every step.
        if (steps > 0) {
#pragma unroll
            for (int s = 0; s < ST; ++s) {
                fetch_rows(s);
                const srd_t da = srd_a(s), db = srd_b(s);
#pragma unroll
                for (int i = 0; i < LA; ++i) load_a(s, da, i);
#pragma unroll
                for (int i = 0; i < FB; ++i) load_b(s, db, i);
            }
            wait_vm<(ST - 1) * L>();
            barrier_raw();
#pragma unroll
            for (int f = 0; f < NF; ++f) read_a(0, 0, 0, f);
#pragma unroll
            for (int h = 0; h < FB; ++h) read_b(0, 0, 0, h);
#pragma nounroll
            for (int s = 0; s < steps; ++s) {
                fetch_rows(s + ST);
                // first half of r: products of set 0, the second half's fragments on their way
#pragma unroll
                for (int f = 0; f < NF; ++f) {
#pragma unroll
                    for (int h = f * FB / NF; h < (f + 1) * FB / NF; ++h) read_b(1, s, 1, h);
                    read_a(1, s, 1, f);
                    mul(0, f);
                    __builtin_amdgcn_sched_barrier(0);
                }
                // every read of this stage is done, so once all waves are here it is free for step s + ST; and step s + 1
                // has landed for all waves
                wait_lds();
                wait_vm<(ST - 2) * L>();
                barrier_raw();
                const srd_t da = srd_a(s + ST), db = srd_b(s + ST);
#pragma unroll
                for (int f = 0; f < NF; ++f) {
#pragma unroll
                    for (int h = f * FB / NF; h < (f + 1) * FB / NF; ++h) read_b(0, s + 1, 0, h);
                    read_a(0, s + 1, 0, f);
#pragma unroll
                    for (int i = f * LA / NF; i < (f + 1) * LA / NF; ++i) load_a(s + ST, da, i);
#pragma unroll
                    for (int i = f * FB / NF; i < (f + 1) * FB / NF; ++i) load_b(s + ST, db, i);
                    mul(1, f);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            wait_vm<0>();   // no load may still write this workgroup's LDS when it ends
        }
        if constexpr (ACC) {
            drain();
#pragma unroll
            for (int f = 0; f < NF; ++f)
#pragma unroll
                for (int h = 0; h < FB; ++h) asm volatile("" : "+a"(acc[f][h]));
#pragma unroll
            for (int f = 0; f < (DB ? NF : 1); ++f) asm volatile("" : "+v"(accb[f]));
        }
        if constexpr (MODE == MM_FWD) {
            if (g.epi.bias || g.epi.residual || g.epi.z || g.epi.act != MOE_LIN_NONE) store<NF, true>(g, t, acc, lane, wi, wj);
            else store<NF, false>(g, t, acc, lane, wi, wj);
        } else {
            store<NF, false>(g, t, acc, lane, wi, wj);
        }
        if constexpr (DB) {
            if (wj == 0 && lane < 16) {
#pragma unroll
                for (int f = 0; f < NF; ++f) {
                    const int i = 16 * (2 * f + wi) + lane;
                    if (i < t.rows) ((uint16_t*)g.dbias)[(int64_t)t.e * g.I + t.i0 + i] = (uint16_t)pack16<F16>(accb[f][0], 0.f);
                }
            }
        }
    }

    template <int NF>
    static __device__ __forceinline__ void by_rows(const MmArgs& g, const MmTile& t, char* sm) {
        if constexpr (NF > 1) {
            if (t.rows <= 16 * NF) return by_rows<NF / 2>(g, t, sm);
        }
        if constexpr (MODE == MM_DW) {
            if (g.dbias && t.j0 == 0) return run<NF, true>(g, t, sm);
        }
        run<NF, false>(g, t, sm);
    }

    static __device__ __forceinline__ void block(const MmArgs& g, char* sm) {
        MmTile t;
        if constexpr (MODE == MM_DW) {
            if (!find_tile_dw<BI, BJ>(g, blockIdx.x, t)) return;
        } else {
            if (!find_tile<BI, BJ>(g, blockIdx.x, t)) return;
            if (t.e == g.E) {   // rows behind the last group
                const int es = g.ydt == MOE_DTYPE_F32 ? 4 : 2, w = min(BJ, g.J - t.j0) * es / 16;
                for (int i = threadIdx.x; i < t.rows * w; i += 256)
                    *(u32x4*)((char*)g.y + ((t.lo + i / w) * g.J + t.j0) * es + (i % w) * 16) = (u32x4){0, 0, 0, 0};
                return;
            }
        }
        by_rows<FA>(g, t, sm);
    }
};

template <int MODE, bool F16, int FA, int FB, int ST, int OCC, bool GATHER>
__global__ void __launch_bounds__(256, OCC) k_mm(const MmArgs g) {
    using K = MmKernel<MODE, F16, FA, FB, ST, GATHER>;
    __shared__ __attribute__((aligned(1024))) char sm[ST * K::STAGE];
    K::block(g, sm);
}

// Launches one mode's kernels (moe_mm_fwd.hip, moe_mm_dx.hip, moe_mm_dw.hip).
int launch_mm_fwd(const MmArgs& a, hipStream_t st);
int launch_mm_dx(const MmArgs& a, hipStream_t st);
int launch_mm_dw(const MmArgs& a, hipStream_t st);
int launch_mm_rows(const MmArgs& a, hipStream_t st);   // forward, few rows (moe_mm_rows.hip)

// Workgroups for tiles of BI rows when the groups' sizes are known on the device only: every group can add a part tile.
inline int64_t mm_row_tiles(const MmArgs& a, int BI) {
    if (!a.offsets) return (a.M + BI - 1) / BI;
    return a.M / BI + (a.E + 1 < a.M ? a.E + 1 : a.M);
}
inline int64_t round8(int64_t n) { return (n + 7) / 8 * 8; }

template <int MODE, bool F16, int FA, int FB, int ST, int OCC>
int launch_mm_cfg(const MmArgs& a, hipStream_t st) {
    const int64_t nj = (a.J + 32 * FB - 1) / (32 * FB);
    const int64_t ni = MODE == MM_DW ? (int64_t)a.E * ((a.I + 32 * FA - 1) / (32 * FA)) : mm_row_tiles(a, 32 * FA);
    const int64_t grid = round8(ni * nj);
    if (grid == 0) return MOE_OK;
    if (grid > 0x7fffffff) return MOE_ERR_ARG;
    if constexpr (MODE == MM_DW) {
        if (a.arows || a.brows) k_mm<MODE, F16, FA, FB, ST, OCC, true><<<(unsigned)grid, 256, 0, st>>>(a);
        else k_mm<MODE, F16, FA, FB, ST, OCC, false><<<(unsigned)grid, 256, 0, st>>>(a);
    } else {
        k_mm<MODE, F16, FA, FB, ST, OCC, false><<<(unsigned)grid, 256, 0, st>>>(a);
    }
    return hipGetLastError() == hipSuccess ? MOE_OK : MOE_ERR_LAUNCH;
}

}  // namespace moe
