// Gradients in x of products with MXFP4 weights: dx[p][k] = sum_n dy[p][n] w[e][n][k], dy in 16 bits, w codes with an exponent per
// 32 of k. The sums go over n, along which the exponents change, so the block-scaled instruction does not apply: the codes become
// 16-bit numbers on their way into LDS: in bf16 exactly, in fp16 rounded, past its largest number to infinity (blocks whose exponent
// byte is 141 or more can hold such values, below 104 such that fp16 has no bits for).
#include "moe_mx4.h"

namespace moe {

// Two of the codes of a word times the power of two s, as 16-bit numbers.
template <bool F16, int B>
__device__ __forceinline__ uint32_t decode2(uint32_t w, float s) {
    if constexpr (F16) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, B));
    else return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, B));
}
template <bool F16>
__device__ __forceinline__ u32x4 decode8(uint32_t w, float s) {
    return (u32x4){decode2<F16, 0>(w, s), decode2<F16, 1>(w, s), decode2<F16, 2>(w, s), decode2<F16, 3>(w, s)};
}

// The 16-bit products' tile of 32 FA x 256 outputs (moe_mm.h: fragments, order of the tiles and stores), 8 waves that multiply and 4
// that load. Loads go straight into LDS, dy's rows into a ring of three steps, and of the weights their codes and exponents, 8.5
// KiB a step, into another; the loading waves then decode a step's codes to the 32 KiB that the products read, of which there are
// two. All of it is a step or more ahead, so that a step has one barrier, as the 16-bit products' have. (Codes on their way in
// registers instead: the compiler waits for a load as soon as its count is not certain, 4096^3 190 us.)
// What bounds it: LDS, which takes in dy and the codes, gives the codes to be decoded, takes them in again as numbers and gives the
// fragments: 4096^3 148 us, without decoding 124 (the weights as 16-bit numbers in memory: 124, and 12 to write them), without any
// loads 123. A step takes 0.75 us with 11 rows of the tile and 1.1 with 128. Tiles of 256 x 128 halve the decoding of full ones, but
// few rows then take twice the steps (64 experts x 16, [2048, 2048]: 59 and 115 us).
template <bool F16, int FA>
struct Mx4Dx {
    static constexpr int FB = 4, NWJ = 4, NWC = 2 * NWJ, NL = 4;
    using Tile = MmKernel<MM_DX, F16, FA, FB, NWJ, 3, 0, EPI_PLAIN, false, NL>;
    static constexpr int BI = Tile::BI, BJ = Tile::BJ;
    static_assert(BJ == 256, "a row's exponents of one step");
    static_assert(FA == 4 || FA == 5, "load_a");
    using A = Operand<false, BI, NL>;
    using B = Operand<true, BJ, NL>;
    static constexpr int PA = A::PIECES, PC = 64 * 128 / 1024 / NL, L = PA + PC + 1;   // loads of a wave and step
    // LDS: dy's ring, the decoded weights, and the ring of their codes with the exponents behind them
    static constexpr int RING = 3, DEC = RING * A::BYTES, CODES = 64 * 128, RAW = DEC + 2 * B::BYTES, RAW_STEP = CODES + 1024;
    static constexpr int BYTES = RAW + RING * RAW_STEP;

    // the offset behind `at` in a ring of n slots of `step` bytes
    template <int N>
    static __device__ __forceinline__ uint32_t after(uint32_t at, uint32_t step) { return at == (N - 1) * step ? 0 : at + step; }

    static __device__ __forceinline__ void block(const MmArgs& g, char* sm, int* pre) {
        const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wi = wave & 1, wj = wave >> 1;
        const int lda2 = g.lda * 2, nj = (g.J + BJ - 1) / BJ;
        count_tiles<MM_DX, BI>(g, pre, 0x70000000 / nj);
        const int tiles = __builtin_amdgcn_readfirstlane(pre[g.E]) * nj;
        if (g.fill && g.offsets) fill_rest<MM_DX>(g);
        const MmRun run = xcd_run<2>(tiles);
        auto tile = [&](int id, MmTile& t) {
            tile_at<MM_DX, BI, BJ>(g, pre, run.tile(id), t);
            if (id >= run.whole) {   // a piece (the last ones of a tile with few rows are empty)
                const int n = BI >> run.cut, lo = ((id - run.whole) & ((1 << run.cut) - 1)) * n;
                t.lo += lo;
                t.rows = max(0, min(n, t.rows - lo));
            }
        };
        auto r_of = [&](const MmTile& t) -> int { return g.part ? min(g.part, g.R - t.e * g.part) : g.R; };
        auto steps_of = [&](const MmTile& t) -> int { return t.rows ? (r_of(t) + 63) / 64 : 0; };
        const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)sm;
        if (run.first == MmRun::NONE) return;

        if (wave >= NWC) {
            const int lw = wave - NWC;
            // a stream of loads: its tile and the step in it; past the last tile empty descriptors. dy's and the weights' are at
            // different steps.
            struct Stream {
                int id = -1, s = 0, steps = 0, r = 0;
                bool live = false;
                MmTile t{};
            };
            auto next_tile = [&](Stream& l) {
                l.s = 0;
                do {
                    l.id = l.id < 0 ? run.first : run.next(l.id);
                    if (l.id == MmRun::NONE) {
                        l.steps = 0x7fffffff;
                        l.live = false;
                        return;
                    }
                    tile(l.id, l.t);
                    l.steps = steps_of(l.t);
                } while (l.steps == 0);
                l.live = true;
                l.r = r_of(l.t);
            };
            Stream la, lb;
            int row, col;
            A::at(lw, lane, row, col);
            uint32_t offa[PA], offb[PC];
            const int KB = g.J / 2, ksteps = (g.J + 255) / 256;
            uint32_t wa = 0, wraw = 0, rraw = 0, wdec = 0;   // slots of the next loads, and of the codes and numbers of the next step
            // where the streams are; a step adds to the pointers and takes from the counts
            const char *pa = nullptr, *pc = nullptr, *ps = nullptr;
            int lefta = 0, leftb = 0;      // of r, from the stream's step on
            uint32_t basea = 0, cols = 0;   // bytes of dy's rows but the last, of a row of codes in this tile
            auto load_a = [&]() {
                if (la.s >= la.steps) {
                    next_tile(la);
                    const int first = la.t.e * g.part;
                    pa = (const char*)g.a + (int64_t)la.t.lo * lda2 + (int64_t)first * 2;
                    lefta = la.live ? la.r : 0;
                    basea = la.live ? (uint32_t)(la.t.rows - 1) * (uint32_t)lda2 : 0u;
#pragma unroll
                    for (int i = 0; i < PA; ++i) offa[i] = (uint32_t)((row + A::ROWS * i) * lda2 + col * 2);
                }
                if (lefta < 64 && col >= lefta)   // the last step ends inside a row
#pragma unroll
                    for (int i = 0; i < PA; ++i) offa[i] = MM_OOB;
                const srd_t da = srd_of(pa, basea + (uint32_t)lefta * 2);
                dma16<4, NL * 1024>(da, offa, lds0 + wa + (uint32_t)(lw * 1024));
                if constexpr (PA == 5) dma16<1, 0>(da, offa + 4, lds0 + wa + (uint32_t)((4 * NL + lw) * 1024));
                ++la.s;
                pa += 128;
                lefta = max(lefta - 64, 0);
                wa = after<RING>(wa, A::BYTES);
            };
            auto load_codes = [&]() {
                if (lb.s >= lb.steps) {
                    next_tile(lb);
                    const int first = lb.t.e * g.part, e = g.part ? 0 : lb.t.e;
                    pc = (const char*)g.b + ((int64_t)e * g.R + first) * KB + lb.t.j0 / 2;
                    ps = (const char*)g.sb + (((int64_t)e * ksteps + lb.t.j0 / 256) * g.R + first) * 8;
                    leftb = lb.live ? lb.r : 0;
                    cols = min(128, KB - lb.t.j0 / 2);
#pragma unroll
                    for (int i = 0; i < PC; ++i)   // 8 rows a piece, 16 bytes a lane
                        offb[i] = lb.t.j0 + 32 * (lane & 7) < g.J ? (uint32_t)((i * NL + lw) * 8 + (lane >> 3)) * (uint32_t)KB + (lane & 7) * 16
                                                                  : MM_OOB;
                }
                const int n = min(64, leftb);
                dma16<PC, NL * 1024>(srd_of(pc, n ? (uint32_t)(n - 1) * (uint32_t)KB + cols : 0u), offb,
                                     lds0 + RAW + wraw + (uint32_t)(lw * 1024));
                const uint32_t off = lane * 16;
                dma16<1, 0>(srd_of(ps, (uint32_t)n * 8), &off, lds0 + RAW + wraw + CODES);   // by every wave: each loads as much
                ++lb.s;
                pc += (int64_t)64 * KB;
                ps += 512;
                leftb = max(leftb - 64, 0);
                wraw = after<RING>(wraw, RAW_STEP);
            };
            // A lane decodes rows 32 i + r of a step, columns 32 b ... (16-byte writes take 13 cycles a wave at best, 8-byte ones 6.)
            const int r = 8 * lw + ((lane & 3) | (lane >> 5) << 2), b = (lane >> 2 & 1) << 1 | (lane >> 3 & 1) | (lane >> 4 & 1) << 2;
            const uint32_t from = r * 128 + b * 16, fexp = CODES + r * 8 + mx4_byte(b);
            uint32_t to[2];   // the block's two granules (row r + 32 has the same)
#pragma unroll
            for (int h = 0; h < 2; ++h) to[h] = r * 2 * BJ + (((2 * b + h) ^ gran_swz<BJ>(r)) & (BJ / 16 - 1)) * 32;
            auto decode = [&]() {
                u32x4 c[2];
                uint32_t e[2];
                const char* raw = sm + RAW + rraw;
                char* dec = sm + DEC + wdec;
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    c[i] = *(const u32x4*)(raw + from + i * 32 * 128);
                    e[i] = *(const uint8_t*)(raw + fexp + i * 32 * 8);
                }
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float s = __uint_as_float(e[i] << 23);
#pragma unroll
                    for (int p = 0; p < 4; ++p) *(u32x4*)(dec + to[p >> 1] + i * 64 * BJ + (p & 1) * 16) = decode8<F16>(c[i][p], s);
                }
                if (__ballot(e[0] == 255 || e[1] == 255)) {   // blocks of NaN, whose codes are 0
                    for (int i = 0; i < 2; ++i)
                        if (e[i] == 255)
                            for (int p = 0; p < 4; ++p)
                                *(u32x4*)(dec + to[p >> 1] + i * 64 * BJ + (p & 1) * 16) =
                                    (u32x4){0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu};
                }
                rraw = after<RING>(rraw, RAW_STEP);
                wdec = after<2>(wdec, B::BYTES);
            };
            // Behind the barrier of step s the products read step s + 1. Step s + 2 is decoded (its codes have landed, and step s has
            // been read), dy of step s + 3 is loaded into the slot of step s, and the codes of step s + 4 into that of step s + 1.
            // Before the next barrier, what was loaded behind the last one has to be here. (A ring of four for the codes: no faster.)
            load_codes(), load_codes(), load_codes();
            load_a(), load_a(), load_a();
            wait_vm<0>();
            barrier_raw();
            decode();
            wait_lds();
            barrier_raw();   // step 0 is ready
            load_codes();
            decode();
            wait_lds();
            for (int id = run.first; id != MmRun::NONE; id = run.next(id)) {
                MmTile t;
                tile(id, t);
                for (int s = steps_of(t); s > 0; --s) {
                    barrier_raw();
                    load_a();
                    load_codes();
                    decode();
                    wait_lds();
                    wait_vm<L>();
                }
            }
            wait_vm<0>();   // no load may still write this workgroup's LDS when it ends
            return;
        }

        const uint32_t fra[1] = {A::frag(wi, lane)};
        uint32_t frb[FB];
#pragma unroll
        for (int h = 0; h < FB; ++h) frb[h] = B::frag(wj * FB + h, lane);
        f32x4 acc[FA][FB];
        s16x8 ra[2][FA], rb[2][FB];   // fragments of the half step that is multiplied and of the next one
        auto mul = [&](int set, int f) {
#pragma unroll
            for (int h = 0; h < FB; ++h) acc[f][h] = mma<F16>(rb[set][h], ra[set][f], acc[f][h]);
        };
        uint32_t abuf = 0, bbuf = DEC;
        barrier_raw();
        barrier_raw();
#pragma unroll
        for (int f = 0; f < FA; ++f) ra[0][f] = A::read(sm, fra, f, 2, 0);
#pragma unroll
        for (int h = 0; h < FB; ++h) rb[0][h] = B::read(sm + bbuf, frb, h, 1, 0);
        for (int id = run.first; id != MmRun::NONE; id = run.next(id)) {
            MmTile t;
            tile(id, t);
            const int steps = steps_of(t), nf = (t.rows + 31) / 32;
            float zero;   // opaque: zeros kept in accumulation registers for the next tile would take them from the sums
            asm volatile("v_mov_b32 %0, 0" : "=v"(zero));
#pragma unroll
            for (int f = 0; f < FA; ++f)
#pragma unroll
                for (int h = 0; h < FB; ++h) acc[f][h] = (f32x4){zero, zero, zero, zero};
#pragma nounroll
            for (int s = 0; s < steps; ++s) {
#pragma unroll
                for (int f = 0; f < FA; ++f) {
                    if (f < FB) rb[1][f] = B::read(sm + bbuf, frb, f, 1, 1);
                    if (f < nf) {
                        ra[1][f] = A::read(sm + abuf, fra, f, 2, 1);
                        mul(0, f);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
                wait_lds();   // every read of this stage is done
                barrier_raw();
                abuf = after<RING>(abuf, A::BYTES);
                bbuf = DEC + after<2>(bbuf - DEC, B::BYTES);
#pragma unroll
                for (int f = 0; f < FA; ++f) {
                    if (f < FB) rb[0][f] = B::read(sm + bbuf, frb, f, 1, 0);
                    ra[0][f] = A::read(sm + abuf, fra, f, 2, 0);
                    if (f < nf) mul(1, f);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            Tile::store(g, t, acc, lane, wi, wj);
        }
    }
};

template <bool F16, int FA>
__global__ void __launch_bounds__(64 * (Mx4Dx<F16, FA>::NWC + Mx4Dx<F16, FA>::NL), (Mx4Dx<F16, FA>::NWC + Mx4Dx<F16, FA>::NL) / 4)
k_mm_mx4_dx(const MmArgs g) {
    using K = Mx4Dx<F16, FA>;
    __shared__ __attribute__((aligned(1024))) char sm[K::BYTES];
    __shared__ int pre[MM_MAX_E + 1];
    static_assert(sizeof(sm) + sizeof(pre) <= 160 * 1024, "");
    K::block(g, sm, pre);
}

template <int FA>
static int launch_dx(const MmArgs& a, hipStream_t st) {
    constexpr int BI = Mx4Dx<true, FA>::BI, BJ = Mx4Dx<true, FA>::BJ, CUT = 4;   // pieces that a tile can be cut into
    const int64_t ni = mm_row_tiles(a, BI), nj = (a.J + BJ - 1) / BJ;
    if (ni * nj == 0) return MOE_OK;
    if (ni * nj > 0x70000000) return MOE_ERR_ARG;
    const int64_t grid = round8(CUT * ni * nj) < 256 ? round8(CUT * ni * nj) : 256;   // 256 CUs
    constexpr int threads = 64 * (Mx4Dx<true, FA>::NWC + Mx4Dx<true, FA>::NL);
    if (a.f16) k_mm_mx4_dx<true, FA><<<(unsigned)grid, threads, 0, st>>>(a);
    else k_mm_mx4_dx<false, FA><<<(unsigned)grid, threads, 0, st>>>(a);
    return hipGetLastError() == hipSuccess ? MOE_OK : MOE_ERR_LAUNCH;
}
// Tiles of 160 rows for groups of about 112 and more (of those that can have rows): a step of a full one takes 10% longer, of a short
// one 8%, but there are fewer, and groups that differ a little do not end in a short one each (us in tiles of 128 and 160 rows,
// random routing: 32 experts x 128, [5760, 2880], 237 and 192, x 139 254 and 190, x 256 342 and 308, x 62 152 and 160; 8 x 256,
// [4096, 4096], 119 and 78, x 2048 555 and 503; 64 x 16, [2048, 2048], 59 and 63).
int launch_mm_mx4_dx(const MmArgs& a, hipStream_t st) {
    const int live = a.E < a.M ? a.E : a.M;
    return a.offsets && a.M / live >= 112 ? launch_dx<5>(a, st) : launch_dx<4>(a, st);
}

// Parts of a dense product, by the estimate of mm_plan: rounds of tiles over the CUs, a step at its measured time, a tile's start and
// stores as three more, and the join as a launch and one pass over the parts.
int mx4_dx_parts(int64_t rows, int64_t N, int64_t K) {
    const int64_t tiles = ((rows + 127) / 128) * ((K + 255) / 256), steps = (N + 63) / 64;
    int best = 1;
    float least = 3e38f;
    for (int parts = 1; parts <= 64 && parts <= steps && (parts == 1 || tiles * parts <= 256); parts *= 2) {
        float us = (float)((tiles * parts + 255) / 256) * (float)((steps + parts - 1) / parts + 3);
        if (parts > 1) us += 3.5f + (float)parts * rows * K * 8.f / 4.5e6f;
        if (us < least) {
            least = us;
            best = parts;
        }
    }
    return best;
}

}  // namespace moe
