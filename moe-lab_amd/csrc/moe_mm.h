// Products of 16-bit matrices on the matrix cores, by ragged groups of rows (one group per expert, or one in all):
//   forward  y[p][n]     = sum_k x[p][k] w[e][n][k]        p in group e
//   dx       dx[p][k]    = sum_n dy[p][n] w[e][n][k]
//   dw       dw[e][n][k] = sum_p dy[p][n] x[p][k]           p over group e
// One tile kernel computes C[i][j] = sum_r A[i][r] B[j][r] for all three; an operand is stored either with r contiguous
// (x and w in the forward pass, dy in dx) or with its own index contiguous (w in dx, both operands in dw).
#pragma once
#include "moe_common.h"
#include "moe_glu8.h"
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
__device__ __forceinline__ srd_t srd_of(const char* p, uint32_t bytes) {
    const uint64_t a = (uint64_t)p;
    srd_t s;
    s[0] = __builtin_amdgcn_readfirstlane((uint32_t)a);
    s[1] = __builtin_amdgcn_readfirstlane((uint32_t)(a >> 32) & 0xffffu);
    s[2] = __builtin_amdgcn_readfirstlane(bytes);
    s[3] = 0x00027000u;
    return s;
}
// N pieces of 64 lanes x 16 bytes, piece i from buffer offset off[i] of each lane to LDS at lds + STRIDE i + 16 lane.
// Asynchronous: counted in vmcnt, which the compiler does not know of (its own waits for other loads can only become
// stricter; told of them, it would wait for all before every LDS read). s_nop 4: the descriptor may have been written by a
// vector instruction just before; s_nop 0: M0.
template <int N, int STRIDE>
__device__ __forceinline__ void dma16(srd_t s, const uint32_t* off, uint32_t lds) {
    static_assert(N == 2 || N == 4, "");
    if constexpr (N == 4)
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %5, 0 offen lds\n\t"
                     "s_add_u32 m0, m0, %6\n\ts_nop 0\n\tbuffer_load_dwordx4 %2, %5, 0 offen lds\n\t"
                     "s_add_u32 m0, m0, %6\n\ts_nop 0\n\tbuffer_load_dwordx4 %3, %5, 0 offen lds\n\t"
                     "s_add_u32 m0, m0, %6\n\ts_nop 0\n\tbuffer_load_dwordx4 %4, %5, 0 offen lds"
                     ::"s"(lds), "v"(off[0]), "v"(off[1]), "v"(off[2]), "v"(off[3]), "s"(s), "n"(STRIDE) : "memory", "m0", "scc");
    else
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %3, 0 offen lds\n\t"
                     "s_add_u32 m0, m0, %4\n\ts_nop 0\n\tbuffer_load_dwordx4 %2, %3, 0 offen lds"
                     ::"s"(lds), "v"(off[0]), "v"(off[1]), "s"(s), "n"(STRIDE) : "memory", "m0", "scc");
}
// 4 bytes per lane, to LDS at lds + 4 lane
__device__ __forceinline__ void dma4(srd_t s, uint32_t off, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dword %1, %2, 0 offen lds"
                 ::"s"(lds), "v"(off), "s"(s) : "memory", "m0");
}
template <int N>
__device__ __forceinline__ void wait_vm() {
    static_assert(N >= 0 && N < 64, "vmcnt has 6 bits");
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
__device__ __forceinline__ void wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }
__device__ __forceinline__ void barrier_raw() { asm volatile("s_barrier" ::: "memory"); }

// One operand's tile in LDS: X rows of the operand's own index x 64 of r, 128 X bytes, filled in units of 1024 bytes
// (X / 8 units, unit i NW + wave by a wave's i-th load).
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

template <bool XC, int X, int NW>   // XC: x contiguous; NW: waves that share the loads
struct Operand {
    static constexpr int BYTES = X * 128;
    static constexpr int PC = X / 8;                      // XC: 16-byte pieces per r-row
    static constexpr int ROWS = XC ? 64 * NW / PC : 8 * NW;   // rows (r or x) between a wave's pieces i and i + 1
    static constexpr int PIECES = X / 8 / NW;             // of a wave and step
    // row and first column that `lane` fetches for its wave's piece 0; piece i: row + ROWS i, column col_of(col, i)
    static __device__ __forceinline__ void at(int wave, int lane, int& row, int& col) {
        if constexpr (!XC) {
            row = 8 * wave + (lane >> 3);
            col = ((lane & 7) ^ (row & 7)) * 8;
        } else {
            row = wave * (64 / PC) + lane / PC;
            const int c = lane % PC;
            col = (((c >> 1) ^ gran_swz<X>(row)) & (X / 16 - 1)) * 16 + (c & 1) * 8;
        }
    }
    static __device__ __forceinline__ int col_of(int col, int i) { return XC && X == 256 ? col ^ ((ROWS * i / 8 & 3) * 64) : col; }
    // LDS byte offset of the fragment of row block xb (16 x), and the fragment at a multiple n of xstep row blocks from one:
    // one 16-byte read, or (XC) two transposing 8-byte reads, which need the offset of each row block
    static __device__ __forceinline__ uint32_t frag(int xb, int lane) {
        const int l = lane & 15, q = lane >> 4;
        if constexpr (!XC) {
            return (uint32_t)((16 * xb + l) * 128 + ((q ^ (l & 7)) * 16));
        } else {
            const int r = 8 * q + (l >> 2);
            return (uint32_t)(r * 2 * X + ((xb ^ gran_swz<X>(r)) & (X / 16 - 1)) * 32 + (l & 3) * 8);
        }
    }
    template <int N>
    static __device__ __forceinline__ s16x8 read(const char* sm, const uint32_t (&f)[N], int n, int xstep, int kk) {
        if constexpr (!XC) {
            return *(const s16x8*)(sm + (f[0] ^ (kk * 64)) + n * xstep * 2048);   // piece q + 4 kk, XORed
        } else {
            typedef __attribute__((address_space(3))) s16x4 lds4;
            const char* p = sm + f[n] + kk * 32 * 2 * X;
            const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)p);
            const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(p + 4 * 2 * X));
            return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
        }
    }
};

// What the forward product's epilogue does with a tile's sums.
enum MmEpiKind {
    EPI_PLAIN = 0,
    EPI_LIN = 1,    // bias, activation, residual, z (moe_linear; bias alone: moe_grouped_mm)
    EPI_GLU = 2     // w is [E, 2 F, K], gate rows then up: y = act(gate, up) [M, F], and optionally the gate/up rows themselves
                    // in 16 bits or in 8 (moe_glu8.h)
};
struct MmEpi {
    const void* bias;        // [E, J] of the operands' type, or null
    const void* residual;    // [M, J] of the operands' type, or null
    void* z;                 // [M, J] of the operands' type: the sums with bias, before the activation; or null
    int act;                 // MOE_LIN_*; EPI_GLU: MOE_ACT_*
    void* gu;                // EPI_GLU: [M, 2 F] of the operands' type, or null
    uint8_t* codes;          // EPI_GLU: [M, 2 F] and scales [M, F / 16], or null
    uint8_t* scales;
};

struct MmArgs {
    const void* a;           // forward: x; dx, dw: dy
    const void* b;           // forward, dx: w [E, N, K]; dw: x
    const int32_t* offsets;  // [E + 1], or null: one group of M rows
    const int32_t* arows;    // row of a of each slot, or null: the slot itself
    const int32_t* brows;    // dw: the same for b
    void* y;
    void* dbias;             // dw: [E, N] of the operands' type (parts: fp32), or null
    int M;                   // slots
    // Without offsets: E = 1 group of all slots, or E parts of one product (split over r; y: the parts' fp32 sums, [E, rows, J]).
    int part;                // slots (dw) or r (forward, dx) of a part, a multiple of 64; 0: no parts
    int a_n, b_n;            // rows of a and (dw) b
    int lda, ldb;            // elements between rows; ldb of forward and dx: K
    int E, I, J, R;          // dw: I = N, J = K; forward: J = N (EPI_GLU: F), R = K; dx: J = K, R = N
    int kind;                // forward: MmEpiKind
    int touch;               // dw: read the operands through once at the start (set by the launcher)
    int f16, ydt, fill;      // ydt: MOE_DTYPE_*; fill: rows behind the last group are set to zero
    MmEpi epi;
};

// The slots of group e, inside [0, M) whatever offsets hold.
template <int MODE>
__device__ __forceinline__ void group_of(const MmArgs& a, int e, int& lo, int& hi) {
    if (!a.offsets) {
        lo = MODE == MM_DW ? e * a.part : 0;
        hi = MODE == MM_DW && a.part && a.M - lo > a.part ? lo + a.part : a.M;
        return;
    }
    const int p = e ? a.offsets[e] : 0, q = a.offsets[e + 1];
    lo = p < 0 ? 0 : p > a.M ? a.M : p;
    hi = q < lo ? lo : q > a.M ? a.M : q;
}

struct MmTile {
    int e;          // group
    int lo;         // forward, dx: first slot of the tile; dw: of the group
    int cnt;        // dw: slots of the group
    int i0, rows;   // dw: first output row; valid rows, <= BI
    int j0;
};

// Workgroup b runs on XCD b % 8. The tiles go round by round, in each to the XCDs one after the other, as many as an XCD has
// workgroups: neighbouring tiles, which share an expert's weights, share an L2, and a busy expert's tiles spread over all XCDs.
// The tiles left after whole rounds are dealt evenly, in the forward and dx products cut into 2 or 4 pieces of their rows while
// that leaves a piece or none to a CU: a piece's weights are read by its neighbours on the XCD too, its products are its own
// (dx of 8 experts x 256, w [14336, 4096]: 442 -> 398 us, 16 x 64, [8192, 5120]: 313 -> 294).
struct MmRun {
    static constexpr int NONE = 0x7fffffff;
    int first, step, whole, last, cut;   // cut: log2 of the pieces
    __device__ __forceinline__ int next(int id) const { return id >= whole ? NONE : id + step < whole ? id + step : last; }
    __device__ __forceinline__ int tile(int id) const { return id < whole ? id : whole + ((id - whole) >> cut); }
};
template <int MAX_CUT>
__device__ __forceinline__ MmRun xcd_run(int tiles) {
    const int xcd = blockIdx.x & 7, w = blockIdx.x >> 3, per = gridDim.x >> 3;
    MmRun r;
    r.step = gridDim.x;
    r.whole = tiles / r.step * r.step;
    int left = tiles - r.whole;
    r.cut = 0;
    while (r.cut < MAX_CUT && left * 2 <= min(r.step, 256)) left *= 2, ++r.cut;
    const int q = left >> 3, rem = left & 7;
    r.last = w < q + (xcd < rem) ? r.whole + xcd * q + min(xcd, rem) + w : MmRun::NONE;
    r.first = r.whole ? xcd * per + w : r.last;
    return r;
}

// Row tiles of the groups, counted on the device: pre[e] = tiles of the groups before e. Wave 0 scans 64 groups at a time.
#define MM_MAX_E 1024
// most: offsets that overlap (which the caller should not pass) could count past 32 bits.
template <int MODE, int BI>
__device__ __forceinline__ void count_tiles(const MmArgs& a, int* pre, int most) {
    if (threadIdx.x < 64) {
        const int lane = threadIdx.x;
        int before = 0;
        if (lane == 0) pre[0] = 0;
        for (int base = 0; base < a.E; base += 64) {
            int n = 0;
            if (base + lane < a.E) {
                int lo, hi;
                group_of<MODE>(a, base + lane, lo, hi);
                n = (hi - lo) / BI + ((hi - lo) % BI > 0);
            }
            const int s = min(wave_incl_scan(n) + before, most);
            if (base + lane < a.E) pre[base + lane + 1] = s;
            before = __builtin_amdgcn_readlane(s, 63);
        }
    }
    __syncthreads();
}
// Zeros into the rows behind the last group, 16 bytes a thread over the whole grid.
template <int MODE>
__device__ __forceinline__ void fill_rest(const MmArgs& a) {
    int lo, hi;
    group_of<MODE>(a, a.E - 1, lo, hi);
    const int64_t row16 = (int64_t)a.J * (a.ydt == MOE_DTYPE_F32 ? 4 : 2) / 16, n = (a.M - hi) * row16;
    u32x4* y = (u32x4*)a.y + hi * row16;
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (int64_t)gridDim.x * blockDim.x)
        y[i] = (u32x4){0, 0, 0, 0};
}
// Tile id of the forward or dx product: its group by two 64-way searches in pre; inside a group down up to 4 row tiles before
// the next column tile.
template <int MODE, int BI, int BJ>
__device__ __forceinline__ void tile_at(const MmArgs& a, const int* pre, int id, MmTile& t) {
    const int lane = threadIdx.x & 63, nj = (a.J + BJ - 1) / BJ;
    constexpr int C = (MM_MAX_E + 63) / 64;
    int e = 0;
    if (a.E > 1) {
        const int c = __builtin_ctzll(__ballot(pre[min(C * (lane + 1), a.E)] * nj > id));
        e = C * c + __builtin_ctzll(__ballot(lane >= C || pre[min(C * c + lane + 1, a.E)] * nj > id));
    }
    const int first = __builtin_amdgcn_readfirstlane(pre[e]), nr = __builtin_amdgcn_readfirstlane(pre[e + 1]) - first;
    const int local = id - first * nj, sup = local / (4 * nj), in = local - sup * 4 * nj, h = min(4, nr - 4 * sup);
    int lo, hi;
    group_of<MODE>(a, e, lo, hi);
    t.e = e;
    t.j0 = in / h * BJ;
    t.lo = lo + (4 * sup + in % h) * BI;
    t.rows = min(BI, hi - t.lo);
    t.i0 = 0;
    t.cnt = 0;
}
// dw: group by group, 4 row tiles (n) down before the next column tile (k)
template <int BI, int BJ>
__device__ __forceinline__ void tile_at_dw(const MmArgs& a, int id, MmTile& t) {
    const int ni = (a.I + BI - 1) / BI, nj = (a.J + BJ - 1) / BJ;
    t.e = id / (ni * nj);
    const int local = id - t.e * ni * nj, sup = local / (4 * nj), in = local - sup * 4 * nj, h = min(4, ni - 4 * sup);
    int hi;
    group_of<MM_DW>(a, t.e, t.lo, hi);
    t.cnt = hi - t.lo;
    t.i0 = (4 * sup + in % h) * BI;
    t.j0 = in / h * BJ;
    t.rows = min(BI, a.I - t.i0);
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

// Tiles of 32 FA x 16 NWJ FB outputs, 2 x NWJ waves, each FA x FB fragments of 16 x 16 (wave (wi, wj): row blocks 2 f + wi,
// column blocks wj FB + h), r in steps of 64 through ST stages of LDS. The matrix instruction takes B's rows as its first
// operand, so a lane's four sums are neighbours in j, the output's contiguous index. Row blocks past a tile's valid rows are
// neither multiplied nor stored.
// A workgroup goes through its tiles with two streams: loads run ST steps ahead of the products and pass from one tile into the
// next, so a tile's first stages arrive during the last one's products and stores. Every step loads the same number of pieces
// (past the last tile from empty descriptors: zeros, no traffic), so the waits are constants.
// NL > 0: as many waves beside the others only load. A wave's loads wait for their turn to be issued, and the products behind
// them with it (4096^3 without any loads: 84 us of 117): 128 x 256 went from 131 to 109 us for 4096^3, 197 to 178 for dx of
// 64 experts x 256 slots, 128 x 128 from 48 to 40 for 1024 x 4096 x 4096. 12 waves leave 168 registers each, enough for 64 x 64
// outputs of a wave; 256 x 256 tiles with 4 waves of all registers are no faster and are gone. With two workgroups of 6 waves on a
// CU they do not pay (128 x 128: the second one does not fit).
// What bounds it: dense, LDS reads and loads into LDS beside the matrix cores (4096^3: 1.17-1.26 PFLOP/s, a library product
// 1.3-1.5); ragged groups, loads, at 3.6-5.8 TB/s of weights.
// EPI_GLU: the tile's columns are BJ / 2 of gate and the same of up, half by half for each wave, so that a lane holds both.
// GATHER: operands that are read through index lists, bit 0: a, bit 1 (dw): b. Such an operand is addressed with 32 bits from its
// start; one in slot order from its group's first slot, in 64 bits, so that its own size has no bound (one flag for both made
// weight gradients of slot-ordered rows past 4 GiB wrong).
template <int MODE, bool F16, int FA, int FB, int NWJ, int ST, int GATHER, int EPI, bool LDS_OUT, int NL>
struct MmKernel {
    static constexpr bool GLU = EPI == EPI_GLU;
    static constexpr bool AX = MODE == MM_DW, BX = MODE != MM_FWD;   // operand with its own index contiguous
    static constexpr int NWC = 2 * NWJ, NW = NL ? NL : NWC;   // waves that multiply, waves that load
    static constexpr int BI = 32 * FA, BJ = 16 * NWJ * FB;
    static constexpr int TJ = GLU ? BJ / 2 : BJ;   // output columns of a tile
    using A = Operand<AX, BI, NW>;
    using B = Operand<BX, BJ, NW>;
    static constexpr int PA = A::PIECES, PB = B::PIECES;
    static constexpr int STAGE = A::BYTES + B::BYTES;
    static constexpr bool LINES = MODE == MM_DW && LDS_OUT;

    // Stores (and the loads of bias and residual) go through buffer descriptors: lanes and columns past the tile's valid ones
    // get an offset past the end, absent operands an empty descriptor, so that the epilogue has no branches per element.
    // 16-bit results without an epilogue go through LDS, 16 rows of a wave's columns at a time (private to the wave), so that
    // every store instruction writes whole cache lines: from the matrix instruction's layout it would write half lines.
    static constexpr int OUT_LD = 32 * FB + 16, OUT_BYTES = 16 * OUT_LD;   // of a wave
    static __device__ __forceinline__ void store_lines(const MmArgs& g, const MmTile& t, f32x4 (&acc)[FA][FB], char* so, int lane,
                                                       int wi, int wj) {
        const int l = lane & 15, q = lane >> 4, jw = t.j0 + wj * FB * 16;
        const int64_t row0 = MODE == MM_DW ? (int64_t)t.e * g.I + t.i0 : (g.part ? (int64_t)t.e * g.M : 0) + t.lo;
        const auto yb = __builtin_amdgcn_make_buffer_rsrc((char*)g.y + row0 * g.J * 2, 0, (uint32_t)t.rows * (uint32_t)g.J * 2,
                                                          0x00027000);
        constexpr int LPR = 2 * FB, RPI = 64 / LPR;   // lanes per row, rows per store
        const int r = lane / LPR, c = lane % LPR * 8;
        const bool ok = jw + c < g.J;
        char *in = so + l * OUT_LD + q * 8, *out = so + r * OUT_LD + c * 2;
#pragma unroll
        for (int f = 0; f < FA; ++f) {
            if (32 * f >= t.rows) break;
#pragma unroll
            for (int h = 0; h < FB; ++h)
                *(u32x2*)(in + h * 32) = (u32x2){pack16<F16>(acc[f][h][0], acc[f][h][1]), pack16<F16>(acc[f][h][2], acc[f][h][3])};
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int k = 0; k < 16 / RPI; ++k) {
                const int i = 16 * (2 * f + wi) + k * RPI + r;
                const uint32_t to = ok && i < t.rows ? ((uint32_t)i * (uint32_t)g.J + jw + c) * 2 : MM_OOB;
                __builtin_amdgcn_raw_buffer_store_b128(*(const u32x4*)(out + k * RPI * OUT_LD), yb, to, 0, 2);
            }
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    static __device__ __forceinline__ void store(const MmArgs& g, const MmTile& t, f32x4 (&acc)[FA][FB], int lane, int wi, int wj) {
        const bool f32 = g.ydt == MOE_DTYPE_F32;
        const int ES = f32 ? 4 : 2;
        const int l = lane & 15, q = lane >> 4, jw = t.j0 + wj * FB * 16;
        const int64_t row0 = MODE == MM_DW ? (int64_t)t.e * g.I + t.i0 : (g.part ? (int64_t)t.e * g.M : 0) + t.lo;
        const auto rsrc = [&](const void* p, int es) {
            return __builtin_amdgcn_make_buffer_rsrc((char*)const_cast<void*>(p) + row0 * g.J * es, 0,
                                                     p ? (uint32_t)t.rows * (uint32_t)g.J * es : 0u, 0x00027000);
        };
        const auto yb = rsrc(g.y, ES), zb = rsrc(g.epi.z, 2), rb = rsrc(g.epi.residual, 2);
        const auto bb = __builtin_amdgcn_make_buffer_rsrc((char*)const_cast<void*>(g.epi.bias) + (int64_t)t.e * g.J * 2, 0,
                                                          g.epi.bias ? (uint32_t)g.J * 2 : 0u, 0x00027000);
        const bool gelu = g.epi.act == MOE_LIN_GELU, lin = g.epi.act == MOE_LIN_NONE;
        const float c1 = gelu ? 1.5957691216057308f : 1.f, c3 = gelu ? 1.5957691216057308f * 0.044715f : 0.f;
#pragma unroll
        for (int f = 0; f < FA; ++f) {
            if (32 * f >= t.rows) break;
            const int i = 16 * (2 * f + wi) + l;
            const uint32_t row = i < t.rows ? (uint32_t)i * (uint32_t)g.J : MM_OOB / 4;
#pragma unroll
            for (int h = 0; h < FB; h += 2) {
                f32x4 v[2] = {acc[f][h], acc[f][h + 1]};
                uint32_t zz[2][2];
                if constexpr (EPI == EPI_LIN) {
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        const int j = jw + 16 * (h + u) + 4 * q;
                        const uint32_t at = j < g.J ? (row + j) * 2 : MM_OOB, bat = j < g.J ? j * 2 : MM_OOB;
                        const u32x2 bw = __builtin_amdgcn_raw_buffer_load_b64(bb, bat, 0, 0);
                        const u32x2 rw = __builtin_amdgcn_raw_buffer_load_b64(rb, at, 0, 0);
#pragma unroll
                        for (int c = 0; c < 4; ++c) v[u][c] += un16<F16>(bw[c >> 1] >> (16 * (c & 1)));
                        zz[u][0] = pack16<F16>(v[u][0], v[u][1]);
                        zz[u][1] = pack16<F16>(v[u][2], v[u][3]);
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            const float z = v[u][c], r = un16<F16>(rw[c >> 1] >> (16 * (c & 1)));
                            v[u][c] = (lin ? z : z * sigmoid_fast(z * (c1 + c3 * (z * z)))) + r;
                        }
                    }
                }
                const int jj = jw + 16 * (h + (q & 1)) + 4 * (q & 2);
                const uint32_t to = jj < g.J ? (row + jj) * 2 : MM_OOB;
                auto put = [&](__amdgpu_buffer_rsrc_t out, uint32_t a0, uint32_t a1, uint32_t b0, uint32_t b1) {
                    __builtin_amdgcn_raw_buffer_store_b128(eight(a0, a1, b0, b1), out, to, 0, 0);
                };
                if (f32) {
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        const int j = jw + 16 * (h + u) + 4 * q;
                        const uint32_t at = j < g.J ? (row + j) * 4 : MM_OOB;
                        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, v[u]), yb, at, 0, 0);
                    }
                } else {
                    put(yb, pack16<F16>(v[0][0], v[0][1]), pack16<F16>(v[0][2], v[0][3]), pack16<F16>(v[1][0], v[1][1]),
                        pack16<F16>(v[1][2], v[1][3]));
                }
                if constexpr (EPI == EPI_LIN) put(zb, zz[0][0], zz[0][1], zz[1][0], zz[1][1]);
                __builtin_amdgcn_sched_barrier(0);   // not all pairs' loads and packed sums at once: they would spill
            }
        }
    }

    // Column pairs (h, h + 1) of 16-bit halves x, y of a lane's row: two column blocks change halves between neighbouring rows of
    // lanes, so that a lane holds eight neighbours.
    static __device__ __forceinline__ u32x4 eight(uint32_t a0, uint32_t a1, uint32_t b0, uint32_t b1) {
        const auto s0 = __builtin_amdgcn_permlane16_swap(a0, b0, false, false);
        const auto s1 = __builtin_amdgcn_permlane16_swap(a1, b1, false, false);
        return (u32x4){s0[0], s1[0], s0[1], s1[1]};
    }
    static __device__ __forceinline__ uint32_t max_rows(uint32_t v) {   // over the four lanes of one output row
        const auto s = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        v = s[0] > s[1] ? s[0] : s[1];
        const auto p = __builtin_amdgcn_permlane32_swap(v, v, false, false);
        return p[0] > p[1] ? p[0] : p[1];
    }
    // EPI_GLU. Two column blocks (32 columns: one block of the 8-bit form) at a time: h = act(gate, up) from the fp32 sums; the
    // kept rows from the sums rounded to 16 bits, as a pass over 16-bit rows would find them.
    static __device__ __forceinline__ void store_glu(const MmArgs& g, const MmTile& t, f32x4 (&acc)[FA][FB], int lane, int wi,
                                                     int wj) {
        constexpr int H = FB / 2;
        static_assert(!GLU || H % 2 == 0, "a block of 32 columns per wave");
        const int l = lane & 15, q = lane >> 4, jw = t.j0 + wj * H * 16, F = g.J;
        const auto rsrc = [&](const void* p, int64_t row_bytes) {
            return __builtin_amdgcn_make_buffer_rsrc((char*)const_cast<void*>(p) + t.lo * row_bytes, 0,
                                                     p ? (uint32_t)t.rows * (uint32_t)row_bytes : 0u, 0x00027000);
        };
        const auto hb = rsrc(g.y, (int64_t)F * 2), gb = rsrc(g.epi.gu, (int64_t)F * 4), cb = rsrc(g.epi.codes, (int64_t)F * 2),
                   sb = rsrc(g.epi.scales, F / 16);
#pragma unroll
        for (int f = 0; f < FA; ++f) {
            if (32 * f >= t.rows) break;
            const int i = 16 * (2 * f + wi) + l;
            const bool in = i < t.rows;
#pragma unroll
            for (int h = 0; h < H; h += 2) {
                const int jj = jw + 16 * (h + (q & 1)) + 4 * (q & 2);   // the eight columns this lane stores
                const bool ok = in && jj < F;
                uint32_t w[2][2][2], o[2][2];   // [gate or up][column block][pair], and h
                uint32_t top[2] = {0, 0};
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const f32x4 a = acc[f][h + u], b = acc[f][H + h + u];
                    float r[4];
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        float x, m, dx, dm;
                        glu_parts(g.epi.act, a[c], b[c], x, m, dx, dm);
                        r[c] = x * m;
                    }
                    o[u][0] = pack16<F16>(r[0], r[1]);
                    o[u][1] = pack16<F16>(r[2], r[3]);
                    w[0][u][0] = pack16<F16>(a[0], a[1]);
                    w[0][u][1] = pack16<F16>(a[2], a[3]);
                    w[1][u][0] = pack16<F16>(b[0], b[1]);
                    w[1][u][1] = pack16<F16>(b[2], b[3]);
                }
                __builtin_amdgcn_raw_buffer_store_b128(eight(o[0][0], o[0][1], o[1][0], o[1][1]), hb,
                                                       ok ? ((uint32_t)i * F + jj) * 2 : MM_OOB, 0, 0);
                if (g.epi.gu) {
#pragma unroll
                    for (int s = 0; s < 2; ++s)
                        __builtin_amdgcn_raw_buffer_store_b128(eight(w[s][0][0], w[s][0][1], w[s][1][0], w[s][1][1]), gb,
                                                               ok ? ((uint32_t)i * 2 * F + s * F + jj) * 2 : MM_OOB, 0, 0);
                }
                if (g.epi.codes) {
#pragma unroll
                    for (int s = 0; s < 2; ++s) {
                        float v[2][4];
#pragma unroll
                        for (int u = 0; u < 2; ++u)
#pragma unroll
                            for (int c = 0; c < 4; ++c) {
                                v[u][c] = un16<F16>(w[s][u][c >> 1] >> (16 * (c & 1)));
                                const uint32_t m = __float_as_uint(v[u][c]) & 0x7fffffffu;
                                top[s] = m > top[s] ? m : top[s];
                            }
                        const uint32_t e = exponent8(max_rows(top[s]));
                        uint32_t k[2] = {0, 0};
                        if (e < 255)
#pragma unroll
                            for (int u = 0; u < 2; ++u)
#pragma unroll
                                for (int c = 0; c < 4; ++c) k[u] |= code8(v[u][c], e) << (8 * c);
                        const auto p = __builtin_amdgcn_permlane16_swap(k[0], k[1], false, false);
                        const uint32_t to = ok ? (uint32_t)i * 2 * F + s * F + jj : MM_OOB;
                        __builtin_amdgcn_raw_buffer_store_b64((u32x2){p[0], p[1]}, cb, to, 0, 0);
                        const uint32_t block = ok ? (uint32_t)i * (F / 16) + (s * F + jw + 16 * h) / 32 : MM_OOB;
                        if (q == 0) __builtin_amdgcn_raw_buffer_store_b8((uint8_t)e, sb, block, 0, 0);
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    }

    static __device__ __forceinline__ void block(const MmArgs& g, char* sm, int* pre) {
        constexpr int L = PA + PB;
        constexpr bool DB = MODE == MM_DW;   // also dbias
        const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wi = wave & 1, wj = wave >> 1;
        const int lw = NL ? wave - NWC : wave;   // among the waves that load
        constexpr bool gath_a = GATHER & 1, gath_b = GATHER & 2;
        static_assert(MODE == MM_DW || !gath_b, "b is weights");
        const int lda2 = g.lda * 2, ldb2 = g.ldb * 2;
        const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)sm;

        const int nj = (g.J + TJ - 1) / TJ;
        int tiles;
        if constexpr (MODE == MM_DW) {
            tiles = g.E * ((g.I + BI - 1) / BI) * nj;
        } else {
            count_tiles<MODE, BI>(g, pre, 0x70000000 / nj);
            tiles = __builtin_amdgcn_readfirstlane(pre[g.E]) * nj;
            if (g.fill && g.offsets) fill_rest<MODE>(g);
        }
        const MmRun run = xcd_run<MODE == MM_DW ? 0 : FA >= 4 ? 2 : 1>(tiles);
        auto tile = [&](int id, MmTile& t) {
            if constexpr (MODE == MM_DW) tile_at_dw<BI, TJ>(g, id, t);
            else tile_at<MODE, BI, TJ>(g, pre, run.tile(id), t);
            if constexpr (MODE != MM_DW) {
                if (id >= run.whole) {   // a piece (the last ones of a tile with few rows are empty)
                    const int n = BI >> run.cut, lo = ((id - run.whole) & ((1 << run.cut) - 1)) * n;
                    t.lo += lo;
                    t.rows = max(0, min(n, t.rows - lo));
                }
            }
        };
        auto r_of = [&](const MmTile& t) -> int { return g.part ? min(g.part, g.R - t.e * g.part) : g.R; };   // forward, dx
        auto steps_of = [&](const MmTile& t) -> int {
            return MODE == MM_DW ? (t.cnt + 63) / 64 : t.rows ? (r_of(t) + 63) / 64 : 0;
        };

        // the stream of loads: its tile, the step in it, and where the operands' next pieces begin
        int lid = -1, ls = 0, lsteps = 0, lrows = 0, lr = 0;
        MmTile lt{};
        const char *pa = nullptr, *pb = nullptr;
        int rowa, cola, rowb, colb;
        A::at(lw, lane, rowa, cola);
        B::at(lw, lane, rowb, colb);
        uint32_t offa[PA], offb[PB];   // each lane's offsets of a step's pieces
        int ia = -1, ib = -1;          // dw, gathered: the step's 64 source rows, one per lane
        auto fetch_rows = [&]() {
            if constexpr (MODE == MM_DW && GATHER) {
                const int p = 64 * ls + lane;
                const bool in = p < lt.cnt;
                if constexpr (gath_a) ia = in ? g.arows[lt.lo + p] : -1;
                if constexpr (gath_b) ib = in ? g.brows[lt.lo + p] : -1;
            }
        };
        auto next_load_tile = [&]() {
            ls = 0;
            do {
                lid = lid < 0 ? run.first : run.next(lid);
                if (lid == MmRun::NONE) {   // no more: empty descriptors
                    lsteps = 0x7fffffff;
                    lrows = lt.cnt = 0;
                    return;
                }
                tile(lid, lt);
                lsteps = steps_of(lt);
            } while (lsteps == 0);
            lrows = 1;
            lr = r_of(lt);
            pa = (const char*)g.a;
            pb = (const char*)g.b;
            const int e = g.part ? 0 : lt.e, first = lt.e * g.part;   // group, and the part's first r
            if constexpr (!AX) pa += (int64_t)first * 2;
            if constexpr (AX) pa += (int64_t)lt.i0 * 2 + (gath_a ? 0 : (int64_t)lt.lo * lda2);
            else if (!gath_a) pa += (int64_t)lt.lo * lda2;
#pragma unroll
            for (int i = 0; i < PA; ++i) {
                const int r = rowa + A::ROWS * i, c = A::col_of(cola, i);
                offa[i] = (uint32_t)(r * lda2 + c * 2);
                if constexpr (AX) {
                    if (lt.i0 + c >= g.I) offa[i] = MM_OOB;
                } else if constexpr (gath_a) {
                    const int src = r < lt.rows ? g.arows[lt.lo + r] : -1;
                    offa[i] = (uint32_t)src < (uint32_t)g.a_n ? (uint32_t)src * (uint32_t)lda2 + c * 2 : MM_OOB;
                }
            }
#pragma unroll
            for (int i = 0; i < PB; ++i) {
                const int c = B::col_of(colb, i), r = rowb + B::ROWS * i;
                offb[i] = (uint32_t)(r * ldb2 + c * 2);
                if (BX && lt.j0 + c >= g.J) offb[i] = MM_OOB;
                if constexpr (GLU) {
                    constexpr int W = 16 * FB, H = W / 2;   // a wave's columns, and its gate ones
                    const int j = lt.j0 + r / W * H + r % H;
                    offb[i] = j < g.J ? (uint32_t)((r % W < H ? j : g.J + j) * ldb2 + c * 2) : MM_OOB;
                }
            }
            if constexpr (GLU) pb += (int64_t)lt.e * 2 * g.J * ldb2;
            else if constexpr (MODE == MM_FWD) pb += ((int64_t)e * g.J + lt.j0) * ldb2 + first * 2;
            if constexpr (MODE == MM_DX) pb += ((int64_t)e * g.R + first) * ldb2 + (int64_t)lt.j0 * 2;
            if constexpr (MODE == MM_DW) pb += (gath_b ? 0 : (int64_t)lt.lo * ldb2) + (int64_t)lt.j0 * 2;
            fetch_rows();
        };
        // bytes of the descriptors for load step ls: up to the end of the last valid row
        auto bytes_a = [&]() -> uint32_t {
            if (!lrows) return 0;
            if constexpr (!AX) return (uint32_t)((gath_a ? g.a_n : lt.rows) - 1) * (uint32_t)lda2 + (uint32_t)(lr - 64 * ls) * 2;
            const int rows = gath_a ? g.a_n : min(64, lt.cnt - 64 * ls);
            return (uint32_t)(rows - 1) * (uint32_t)lda2 + (uint32_t)(g.I - lt.i0) * 2;
        };
        auto bytes_b = [&]() -> uint32_t {
            if (!lrows) return 0;
            if constexpr (!BX) {
                const int rows = GLU ? 2 * g.J : min(BJ, g.J - lt.j0);
                return (uint32_t)(rows - 1) * (uint32_t)ldb2 + (uint32_t)(lr - 64 * ls) * 2;
            }
            const int rows = MODE == MM_DX ? min(64, lr - 64 * ls) : gath_b ? g.b_n : min(64, lt.cnt - 64 * ls);
            return (uint32_t)(rows - 1) * (uint32_t)ldb2 + (uint32_t)(g.J - lt.j0) * 2;
        };
        // dw, gathered: the pieces' rows are other ones in every step
        auto row_off = [&](int ids, int row, int n, int ld2, int c, bool in) -> uint32_t {
            const int src = __shfl(ids, row);
            return in && (uint32_t)src < (uint32_t)n ? (uint32_t)src * (uint32_t)ld2 + c * 2 : MM_OOB;
        };
        auto step_offsets = [&]() {
            if constexpr (MODE == MM_DW && gath_a) {
#pragma unroll
                for (int i = 0; i < PA; ++i) {
                    const int c = A::col_of(cola, i);
                    offa[i] = row_off(ia, rowa + A::ROWS * i, g.a_n, lda2, c, lt.i0 + c < g.I);
                }
            }
            if constexpr (gath_b) {
#pragma unroll
                for (int i = 0; i < PB; ++i) {
                    const int c = B::col_of(colb, i);
                    offb[i] = row_off(ib, rowb + B::ROWS * i, g.b_n, ldb2, c, lt.j0 + c < g.J);
                }
            }
            // a step that ends past R: its pieces there (one with r contiguous has a single column per lane)
            if (!AX && 64 * ls + 64 > lr && lrows) {
                if (64 * ls + cola >= lr)
#pragma unroll
                    for (int i = 0; i < PA; ++i) offa[i] = MM_OOB;
                if (!BX && 64 * ls + colb >= lr)
#pragma unroll
                    for (int i = 0; i < PB; ++i) offb[i] = MM_OOB;
            }
        };
        // pieces i0 .. of either operand, for load step ls into stage buffer `buf`
        constexpr int NA = PA < 4 ? PA : 4, NB = PB < 4 ? PB : 4;
        auto load_a = [&](uint32_t buf, srd_t d, int i) {
            dma16<NA, NW * 1024>(d, offa + i, lds0 + buf + (uint32_t)((i * NW + lw) * 1024));
        };
        auto load_b = [&](uint32_t buf, srd_t d, int i) {
            dma16<NB, NW * 1024>(d, offb + i, lds0 + buf + (uint32_t)(A::BYTES + (i * NW + lw) * 1024));
        };
        auto srd_a = [&]() { return srd_of(pa, bytes_a()); };
        auto srd_b = [&]() { return srd_of(pb, bytes_b()); };
        auto step_loads = [&]() {
            ++ls;
            if (!(AX && gath_a)) pa += AX ? 64 * (int64_t)lda2 : 128;
            if (!gath_b) pb += BX ? 64 * (int64_t)ldb2 : 128;
            fetch_rows();
        };

        uint32_t fra[AX ? FA : 1], frb[BX ? FB : 1];
#pragma unroll
        for (int f = 0; f < (AX ? FA : 1); ++f) fra[f] = A::frag(2 * f + wi, lane);
#pragma unroll
        for (int h = 0; h < (BX ? FB : 1); ++h) frb[h] = A::BYTES + B::frag(wj * FB + h, lane);
        f32x4 acc[FA][FB];
        float sums[DB ? FA : 1];
        s16x8 ra[2][FA], rb[2][FB];   // fragments of the half step that is multiplied and of the next one
        auto mul = [&](int set, int f) {
#pragma unroll
            for (int h = 0; h < FB; ++h) {
                acc[f][h] = mma<F16>(rb[set][h], ra[set][f], acc[f][h]);
            }
        };
        // dbias: this lane's share (8 of 32 r) of its rows' sums over r, in fp32, of dy as it lies in the fragments: in 16 bits. A
        // linear layer's dz is rounded to them for the products; its rows' errors are independent and even, so that of T rows they
        // add sqrt(T) half steps / sqrt(3) of a row's to a sum, below its own rounding unless the rows cancel to less than that.
        auto add_rows = [&](int set) {
#pragma unroll
            for (int f = 0; f < FA; ++f) {
                const u32x4 w = __builtin_bit_cast(u32x4, ra[set][f]);
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    sums[f] = F16 ? dot2_f16(w[c], 0x3C003C00u, sums[f]) : dot2_bf16(w[c], 0x3F803F80u, sums[f]);
            }
        };

        if (run.first == MmRun::NONE) return;
        // dw of ragged groups: with a group of a few steps a tile's loads run only a tile ahead, too little for a group that is
        // not in a cache yet while the stores fill HBM's queues. So the operands' lines are read through once, 64 lines an
        // instruction over the whole grid, into LDS that is free before the first stores (32 experts x 139 slots,
        // [5760, 2880], operands not in a cache: 410 -> 341 us; 64 x 128, [2048, 2048]: 210 -> 160; in a cache 148 -> 158).
        if constexpr (LINES) {
            if (g.touch) {
                auto touch = [&](const void* p, int rows, int cols, int ld2) {
                    const uint32_t lines = (uint32_t)(cols + 63) / 64, n = (uint32_t)rows * lines;
                    const srd_t d = srd_of((const char*)p, (uint32_t)(rows - 1) * (uint32_t)ld2 + (uint32_t)cols * 2);
                    for (uint32_t b = (blockIdx.x * NW + wave) * 64; b < n; b += gridDim.x * NW * 64) {
                        const uint32_t i = b + lane, r = i / lines;
                        dma4(d, i < n ? r * (uint32_t)ld2 + (i - r * lines) * 128 : MM_OOB, lds0 + ST * STAGE + wave * OUT_BYTES);
                    }
                };
                touch(g.a, gath_a ? g.a_n : g.M, g.I, lda2);
                touch(g.b, gath_b ? g.b_n : g.M, g.J, ldb2);
            }
        }
        uint32_t rbuf = 0, wbuf = 0;   // stage buffers of the step that is multiplied, and of the load step
        auto next_buf = [](uint32_t b) -> uint32_t { return b == (ST - 1) * STAGE ? 0 : b + STAGE; };
        const bool loads = !NL || wave >= NWC;
        if (loads) {
#pragma unroll
            for (int s = 0; s < ST; ++s) {
                if (ls >= lsteps) next_load_tile();
                step_offsets();
                const srd_t da = srd_a(), db = srd_b();
#pragma unroll
                for (int i = 0; i < PA; i += NA) load_a(wbuf, da, i);
#pragma unroll
                for (int i = 0; i < PB; i += NB) load_b(wbuf, db, i);
                step_loads();
                wbuf = next_buf(wbuf);
            }
            wait_vm<(ST - 1) * L>();
        }
        barrier_raw();
        if constexpr (NL > 0) {
            if (loads) {
                for (int id = run.first; id != MmRun::NONE; id = run.next(id)) {
                    MmTile t;
                    tile(id, t);
                    for (int s = steps_of(t); s > 0; --s) {
                        if (ls >= lsteps) next_load_tile();
                        step_offsets();
                        const srd_t da = srd_a(), db = srd_b();
                        wait_vm<(ST - 2) * L>();
                        barrier_raw();
#pragma unroll
                        for (int i = 0; i < PB; i += NB) load_b(wbuf, db, i);
#pragma unroll
                        for (int i = 0; i < PA; i += NA) load_a(wbuf, da, i);
                        step_loads();
                        wbuf = next_buf(wbuf);
                    }
                }
                wait_vm<0>();
                return;
            }
        }
#pragma unroll
        for (int f = 0; f < FA; ++f) ra[0][f] = A::read(sm, fra, f, 2, 0);
#pragma unroll
        for (int h = 0; h < FB; ++h) rb[0][h] = B::read(sm, frb, h, 1, 0);

        for (int id = run.first; id != MmRun::NONE; id = run.next(id)) {
            MmTile t;
            tile(id, t);
            const int steps = steps_of(t), nf = (t.rows + 31) / 32;
            const bool bias = DB && g.dbias && t.j0 == 0;
            float zero;   // opaque: zeros kept in accumulation registers for the next tile would take them from the sums
            asm volatile("v_mov_b32 %0, 0" : "=v"(zero));
#pragma unroll
            for (int f = 0; f < FA; ++f)
#pragma unroll
                for (int h = 0; h < FB; ++h) acc[f][h] = (f32x4){zero, zero, zero, zero};
#pragma unroll
            for (int f = 0; f < (DB ? FA : 1); ++f) sums[f] = 0.f;
#pragma nounroll
            for (int s = 0; s < steps; ++s) {
                // first half of r: products of set 0, the second half's fragments on their way
#pragma unroll
                for (int f = 0; f < FA; ++f) {
#pragma unroll
                    for (int h = f * FB / FA; h < (f + 1) * FB / FA; ++h) rb[1][h] = B::read(sm + rbuf, frb, h, 1, 1);
                    if (f < nf) {
                        ra[1][f] = A::read(sm + rbuf, fra, f, 2, 1);
                        mul(0, f);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
                if constexpr (DB) {
                    if (bias) add_rows(0);
                }
                srd_t da = {}, db = {};
                if constexpr (!NL) {
                    if (ls >= lsteps) next_load_tile();
                    step_offsets();
                    da = srd_a(), db = srd_b();
                }
                // every read of this stage is done, so once all waves are here it is free for the load stream; and the next
                // stage has landed for all waves
                wait_lds();
                if constexpr (!NL) wait_vm<(ST - 2) * L>();
                barrier_raw();
                rbuf = next_buf(rbuf);
#pragma unroll
                for (int f = 0; f < FA; ++f) {
#pragma unroll
                    for (int h = f * FB / FA; h < (f + 1) * FB / FA; ++h) rb[0][h] = B::read(sm + rbuf, frb, h, 1, 0);
                    ra[0][f] = A::read(sm + rbuf, fra, f, 2, 0);
                    // the pieces, four at a time, over the row blocks
                    constexpr int CALLS = PA / NA + PB / NB;
#pragma unroll
                    for (int c = NL ? CALLS : f * CALLS / FA; c < (f + 1) * CALLS / FA; ++c) {
                        if (c < PB / NB) load_b(wbuf, db, c * NB);
                        else load_a(wbuf, da, (c - PB / NB) * NA);
                    }
                    if (f < nf) mul(1, f);
                    __builtin_amdgcn_sched_barrier(0);
                }
                if constexpr (DB) {
                    if (bias) add_rows(1);
                }
                if constexpr (!NL) {
                    step_loads();
                    wbuf = next_buf(wbuf);
                }
            }
            if constexpr (GLU) store_glu(g, t, acc, lane, wi, wj);
            else if (LINES && g.ydt != MOE_DTYPE_F32) store_lines(g, t, acc, sm + ST * STAGE + wave * OUT_BYTES, lane, wi, wj);
            else store(g, t, acc, lane, wi, wj);
            if constexpr (DB) {
                if (bias && wj == 0) {
#pragma unroll
                    for (int f = 0; f < FA; ++f) {
                        float v = sums[f] + __shfl_xor(sums[f], 16);
                        v += __shfl_xor(v, 32);
                        const int i = 16 * (2 * f + wi) + lane;
                        const int64_t at = (int64_t)t.e * g.I + t.i0 + i;
                        if (lane < 16 && i < t.rows) {
                            if (g.part) ((float*)g.dbias)[at] = v;
                            else ((uint16_t*)g.dbias)[at] = (uint16_t)pack16<F16>(v, 0.f);
                        }
                    }
                }
            }
        }
        wait_vm<0>();   // no load may still write this workgroup's LDS when it ends
    }
};

template <int MODE, bool F16, int FA, int FB, int NWJ, int ST, int OCC, int GATHER, int EPI, int NL>
__global__ void __launch_bounds__(128 * NWJ + 64 * NL, OCC * (2 * NWJ + NL) / 4) k_mm(const MmArgs g) {
    // LDS of a CU's OCC workgroups: 160 KiB
    constexpr int LDS = 160 * 1024 / OCC, STAGES = ST * 64 * (32 * FA + 16 * NWJ * FB) * 2, PRE = 4 * MM_MAX_E + 64;
    constexpr bool LDS_OUT = OCC == 2 && STAGES + PRE + 2 * NWJ * 16 * (32 * FB + 16) <= LDS;
    using K = MmKernel<MODE, F16, FA, FB, NWJ, ST, GATHER, EPI, LDS_OUT, NL>;
    __shared__ __attribute__((aligned(1024))) char sm[STAGES + (K::LINES ? K::NW * K::OUT_BYTES : 0)];
    __shared__ int pre[MODE == MM_DW ? 1 : MM_MAX_E + 1];
    K::block(g, sm, pre);
}

// Launches one mode's kernels (moe_mm_fwd.hip, moe_mm_dx.hip, moe_mm_dw.hip).
int launch_mm_fwd(const MmArgs& a, hipStream_t st);
int launch_mm_dx(const MmArgs& a, hipStream_t st);
int launch_mm_dw(const MmArgs& a, hipStream_t st);
int launch_mm_rows(const MmArgs& a, hipStream_t st);   // forward, few rows (moe_mm_rows.hip)

// Tiles of the product kernel: 128 x 256 with 8 waves that multiply and 4 that load; 128 x 128 with 4 and 4, one workgroup on a
// CU, 4 stages; 128 x 128 with 4 waves that do both, two workgroups on a CU (dw, and dx of few rows); 64 x 64, two on a CU.
// MM_ROWS: dot products (moe_mm_rows.hip).
enum MmShape { MM_128x256 = 0, MM_128_DEEP = 1, MM_128 = 2, MM_64 = 3, MM_ROWS = 4 };
// Shape and number of parts for a product without offsets: out [rows, J], sums of length R (moe_mm_parts.hip).
struct MmPlan {
    int shape, parts;
};
MmPlan mm_plan(int mode, int64_t rows, int64_t J, int64_t R, bool split);
// Forward with up to 4 rows: dot products, whole (w [4096, 4096], T 1: 8.6 us, 64 x 64 in 4 parts 12.6; T 4: 10.0 and 12.6;
// T 8: 14.4 and 12.8).
constexpr int MM_FEW = 4;

// A product without offsets in its plan's parts, and the parts' sum with the epilogue (part by part in order: the result does not
// depend on which part ends first). ws: parts x rows x J floats, and for dbias parts x I behind them.
int launch_mm_parts(int mode, const MmArgs& a, int parts, float* ws, hipStream_t st);

// Workgroups for tiles of BI rows when the groups' sizes are known on the device only: every group can add a part tile.
inline int64_t mm_row_tiles(const MmArgs& a, int BI) {
    if (!a.offsets) return ((int64_t)a.M + BI - 1) / BI * a.E;
    return a.M / BI + (a.E + 1 < a.M ? a.E + 1 : a.M);
}
inline int64_t round8(int64_t n) { return (n + 7) / 8 * 8; }

template <int MODE, bool F16, int FA, int FB, int NWJ, int ST, int OCC, int NL = 0>
int launch_mm_cfg(const MmArgs& a, hipStream_t st) {
    const bool glu = MODE == MM_FWD && a.kind == EPI_GLU;
    const int bj = 16 * NWJ * FB / (glu ? 2 : 1);
    const int64_t nj = (a.J + bj - 1) / bj;
    const int64_t ni = MODE == MM_DW ? (int64_t)a.E * ((a.I + 32 * FA - 1) / (32 * FA)) : mm_row_tiles(a, 32 * FA);
    if (ni * nj == 0) return MOE_OK;
    if (ni * nj > 0x70000000) return MOE_ERR_ARG;
    constexpr int CUT = MODE == MM_DW ? 1 : FA >= 4 ? 4 : 2;   // pieces that a tile can be cut into
    const int64_t most = 256 * OCC, grid = round8(CUT * ni * nj) < most ? round8(CUT * ni * nj) : most;   // 256 CUs
    auto run = [&](auto epi, auto lists) {
        k_mm<MODE, F16, FA, FB, NWJ, ST, OCC, decltype(lists)::value, decltype(epi)::value, NL>
            <<<(unsigned)grid, 128 * NWJ + 64 * NL, 0, st>>>(a);
    };
    auto go = [&](auto epi) {
        if constexpr (MODE == MM_DW) {
            if (a.arows && a.brows) return run(epi, std::integral_constant<int, 3>{});
            if (a.brows) return run(epi, std::integral_constant<int, 2>{});
        }
        if (a.arows) return run(epi, std::integral_constant<int, 1>{});
        run(epi, std::integral_constant<int, 0>{});
    };
    if constexpr (MODE == MM_FWD) {
        if (glu) {
            if constexpr (FB % 4 == 0) go(std::integral_constant<int, EPI_GLU>{});
            else return MOE_ERR_ARG;
        } else if (a.kind == EPI_LIN) {
            go(std::integral_constant<int, EPI_LIN>{});
        } else {
            go(std::integral_constant<int, EPI_PLAIN>{});
        }
    } else {
        go(std::integral_constant<int, EPI_PLAIN>{});
    }
    return hipGetLastError() == hipSuccess ? MOE_OK : MOE_ERR_LAUNCH;
}

}  // namespace moe
