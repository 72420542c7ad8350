// Products of MXFP4 operands in tiles: y[p][n] = sum_k x[p][k] w[e][n][k], both operands codes with an exponent per 32 of k.
#include "moe_mx4.h"

namespace moe {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

// 32 x 32 outputs, 64 of k: lane l holds 32 codes of row l & 31 (k from 32 (l >> 5) on) and in byte KS of s their exponent.
// The codes fill half of the operand's registers.
template <int KS>
__device__ __forceinline__ f32x16 mma32(s16x8 a, uint32_t sa, s16x8 b, uint32_t sb, f32x16 c) {
    typedef int i32x4 __attribute__((ext_vector_type(4)));
    const auto wide = [](s16x8 v) {
        const i32x4 w = __builtin_bit_cast(i32x4, v);
        return __builtin_shufflevector(w, w, 0, 1, 2, 3, -1, -1, -1, -1);
    };
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wide(a), wide(b), c, 4, 4, KS, (int)sa, KS, (int)sb);
}
// Two pieces of a lane and of the one 16 further on: afterwards the first lane (of 0 .. 15, 32 .. 47) holds its own first piece in a
// and the other's in b, the second one (16 .. 31, 48 .. 63) the first's second piece in a and its own in b. Its own inverse.
__device__ __forceinline__ void swap16(u32x4& a, u32x4& b) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const auto s = __builtin_amdgcn_permlane16_swap(a[i], b[i], false, false);
        a[i] = s[0];
        b[i] = s[1];
    }
}

// The same with the lane 4 further on: the first one is of 0 .. 3 or 8 .. 11 of 16.
__device__ __forceinline__ void swap4(u32x4& a, u32x4& b) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int x = a[i], y = b[i];
        a[i] = __builtin_amdgcn_update_dpp(x, y, 0x114, 0xf, 0xa, false);   // from 4 lanes before, where bit 2 is set
        b[i] = __builtin_amdgcn_update_dpp(y, x, 0x104, 0xf, 0x5, false);   // from 4 lanes after, where it is not
    }
}

// The epilogue: none, bias and residual, or those with an activation. A kernel of its own for each: a branch on the activation
// inside one made the compiler hold both sides' values and spill.
enum MxEpi { MX_PLAIN = 0, MX_LIN = 1, MX_ACT = 2 };

// Tiles of 32 FA NWI x 32 FB NWJ outputs, NWI x NWJ waves that multiply FA x FB blocks of 32 x 32 each (wave (wi, wj): row blocks
// NWI f + wi, columns 32 FB wj ..) and NL waves that only load, k in steps of 256 through ST stages of LDS. The streams of loads
// and products, the tiles' order and the pieces of the last round are those of the 16-bit products (moe_mm.h): sizes along k are
// counted in 16-bit words, four codes each, so that a step is 64 words.
// A stage is the operands' codes, 128 bytes a row, its 16-byte pieces XORed so that a fragment's rows spread over the banks, and
// their exponents, 8 bytes a row. These lie in memory by steps (moe_mx4.h), so that a tile's are 1 KiB pieces, one to a loading
// wave; their bytes are ordered so that a lane's four of a step are one word, which the instruction picks from. GATHER: x's rows, and
// their exponents in words, through the index list.
// The matrix instruction takes w's rows as its first operand, and row m of it is w's row column(m) of a block's 32, so that a lane's
// 16 sums of one row of x are neighbours. Exchanges with the lane of the row 16 further on and with that of the row 4 further on then
// make every store instruction write whole lines, and loads of the residual read them. (Without the second exchange, half lines, and with
// it, each pair measured together: 4096 x 8 rows of 128 experts, [1536, 2048], 97 and 92 us; 32 experts, [5760, 2880], 4444 rows 118 and
// 112.)
// What bounds it: in large tiles a step's fragment reads take LDS as long as the matrix cores take for its products, loads into LDS 40%
// more on top, and beside them the clock falls with the power: [4096, 16384] by [16384, 4096] 155 us, 3.5 PFLOP/s of the 6.3 that the
// instruction reaches by itself, 4096^3 41-46 us (3.0-3.3, by the card; bf16 110), 4096 x 8 rows of 128 experts, [1536, 2048], 88-93 (8
// steps a tile: stores and the first loads are a fifth). A wave to 64 x 128 outputs, which reads a quarter less, has nothing to cover
// its own latency: 4096^3 47 us. In 64 x 64 tiles, L2: 237 rows, [4096, 4096], 10.4 us for 75 MB of loads; 8 stages of one workgroup instead of 4
// of two: 12.3.
template <bool F16, int FA, int FB, int NWI, int NWJ, int ST, int GATHER, int EPI, int NL>
struct MxKernel {
    static constexpr bool LIN = EPI != MX_PLAIN;
    static constexpr int NWC = NWI * NWJ;
    static constexpr int BI = 32 * FA * NWI, BJ = 32 * FB * NWJ;
    static constexpr int PA = BI / 8 / NL, PB = BJ / 8 / NL;                                  // 1 KiB pieces of a loading wave
    static constexpr int SCA = (BI * 8 + 1023) / 1024, SCB = (BJ * 8 + 1023) / 1024;   // pieces of exponents
    static_assert(SCA + SCB <= NL, "one to a wave");
    static constexpr int CODES = (BI + BJ) * 128, STAGE = CODES + (SCA + SCB) * 1024;
    static constexpr int SG = BI * 8 / 256;   // GATHER: pieces of x's exponents, 64 words each
    static constexpr int L = PA + PB + 1 + GATHER;

    // XOR of the 16-byte pieces of a row. Half a wave's reads take two cycles if none of the 16 places that 16 bytes can have in the
    // banks occurs more than twice among them: two rows share a line of all banks, so 32 rows have each piece in four places of
    // 8 with a XOR by the row, in all by its half (column()'s rows too): 588 of a step's 1180 cycles went to conflicts.
    static __device__ __forceinline__ int swz(int r) { return r >> 1 & 7; }
    static __device__ __forceinline__ int column(int m) { return (m >> 2 & 1) * 16 + (m >> 3) * 4 + (m & 3); }

    static __device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_of(const void* p, int64_t row0, int rows, int J, int es) {
        return __builtin_amdgcn_make_buffer_rsrc((char*)const_cast<void*>(p) + row0 * J * es, 0,
                                                 p ? (uint32_t)rows * (uint32_t)J * es : 0u, 0x00027000);
    }
    // Everything goes through buffer descriptors: rows and columns past the tile's valid ones get an offset past the end, absent
    // operands an empty descriptor. Residual rows are loaded as lines, like the stores, all before the first is needed.
    static __device__ __forceinline__ void store(const MmArgs& g, const MmTile& t, f32x16 (&acc)[FA][FB], int lane, int wi, int wj) {
        const bool f32 = g.ydt == MOE_DTYPE_F32;
        const int ES = f32 ? 4 : 2, l = lane & 15, q = lane >> 4;
        const int jw = t.j0 + wj * 32 * FB;   // the wave's columns; a lane's of block h: 32 h + 16 (lane >> 5) ..
        const int64_t row0 = (g.part ? (int64_t)t.e * g.M : 0) + t.lo;
        const auto yb = rows_of(g.y, row0, t.rows, g.J, ES), zb = rows_of(g.epi.z, row0, t.rows, g.J, 2),
                   rb = rows_of(g.epi.residual, row0, t.rows, g.J, 2);
        // 16-bit pieces of 8 columns after both exchanges: the x-th one of rows 16 s .. of row block f (one exchange where a wave has
        // half a line of each row)
        const auto at = [&](int f, int x, int s) -> uint32_t {
            const int i = 32 * (NWI * f + wi) + 16 * s + (FB == 1 ? l : (l & 11) + 4 * x);
            const int c = jw + (FB == 1 ? 0 : 32 * (l >> 2 & 1)) + 8 * q;
            return i < t.rows && c < g.J ? ((uint32_t)i * (uint32_t)g.J + c) * 2 : MM_OOB;
        };
        const auto lines = [&](u32x4 (&v)[FB][2]) {   // between [column block][half of its 16] of a row and [x][s]
            if constexpr (FB == 2) swap4(v[0][0], v[1][0]), swap4(v[0][1], v[1][1]);
        };
        const auto rows = [&](u32x4 (&v)[FB][2]) {
#pragma unroll
            for (int h = 0; h < FB; ++h) swap16(v[h][0], v[h][1]);
        };
        u32x4 res[LIN ? FA : 1][FB][2];
        if constexpr (LIN) {
#pragma unroll
            for (int f = 0; f < FA; ++f)
#pragma unroll
                for (int x = 0; x < FB; ++x)
#pragma unroll
                    for (int s = 0; s < 2; ++s) res[f][x][s] = __builtin_amdgcn_raw_buffer_load_b128(rb, at(f, x, s), 0, 0);
        }
        const bool gelu = g.epi.act == MOE_LIN_GELU;
        const float c1 = gelu ? 1.5957691216057308f : 1.f, c3 = gelu ? 1.5957691216057308f * 0.044715f : 0.f;
#pragma unroll
        for (int f = 0; f < FA; ++f) {
            if (32 * (NWI * f + wi) >= t.rows) break;
            const auto store16 = [&](u32x4 (&v)[FB][2], __amdgpu_buffer_rsrc_t to) {
                rows(v);
                lines(v);
#pragma unroll
                for (int s = 0; s < 2; ++s)
#pragma unroll
                    for (int x = 0; x < FB; ++x) __builtin_amdgcn_raw_buffer_store_b128(v[x][s], to, at(f, x, s), 0, 2);
            };
            if constexpr (LIN) {
                const auto bb = rows_of(g.epi.bias, t.e, 1, g.J, 2);
                u32x4 zz[FB][2];
                lines(res[f]);
                rows(res[f]);
#pragma unroll
                for (int h = 0; h < FB; ++h) {
                    u32x4 bias[2];   // loaded for each row block: kept in fp32 they would spill others
                    const int c0 = jw + 32 * h + 16 * (lane >> 5);
#pragma unroll
                    for (int u = 0; u < 2; ++u)
                        bias[u] = __builtin_amdgcn_raw_buffer_load_b128(bb, c0 + 8 * u < g.J ? (c0 + 8 * u) * 2 : MM_OOB, 0, 0);
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
#pragma unroll
                        for (int c = 0; c < 4; ++c) {   // two neighbours
                            const int i = u * 8 + 2 * c;
                            float v[2];
#pragma unroll
                            for (int p = 0; p < 2; ++p) v[p] = acc[f][h][i + p] + un16<F16>(bias[u][c] >> (16 * p));
                            zz[h][u][c] = pack16<F16>(v[0], v[1]);
#pragma unroll
                            for (int p = 0; p < 2; ++p) {
                                // (the square bounded: SiLU's c3 is 0, and 0 times an infinity NaN)
                                if constexpr (EPI == MX_ACT) v[p] *= sigmoid_fast(v[p] * (c1 + c3 * fminf(v[p] * v[p], 1e30f)));
                                acc[f][h][i + p] = v[p] + un16<F16>(res[f][h][u][c] >> (16 * p));
                            }
                        }
                        __builtin_amdgcn_sched_barrier(0);   // not all pieces at once: they would spill
                    }
                }
                if (g.epi.z) store16(zz, zb);
            }
            if (f32) {   // pieces of 4 columns, a line to a block
#pragma unroll
                for (int h = 0; h < FB; ++h) {
                    u32x4 o[4];
#pragma unroll
                    for (int u = 0; u < 4; ++u)
#pragma unroll
                        for (int c = 0; c < 4; ++c) o[u][c] = __float_as_uint(acc[f][h][u * 4 + c]);
                    swap16(o[0], o[1]), swap16(o[2], o[3]);
                    swap4(o[0], o[2]), swap4(o[1], o[3]);
#pragma unroll
                    for (int s = 0; s < 2; ++s)
#pragma unroll
                        for (int x = 0; x < 2; ++x) {
                            const int i = 32 * (NWI * f + wi) + 16 * s + (l & 11) + 4 * x;
                            const int c = jw + 32 * h + 16 * (q >> 1) + 8 * (l >> 2 & 1) + 4 * (q & 1);
                            __builtin_amdgcn_raw_buffer_store_b128(
                                o[2 * x + s], yb, i < t.rows && c < g.J ? ((uint32_t)i * (uint32_t)g.J + c) * 4 : MM_OOB, 0, 0);
                        }
                }
            } else {
                u32x4 o[FB][2];
#pragma unroll
                for (int h = 0; h < FB; ++h)
#pragma unroll
                    for (int u = 0; u < 2; ++u)
#pragma unroll
                        for (int c = 0; c < 4; ++c) o[h][u][c] = pack16<F16>(acc[f][h][u * 8 + 2 * c], acc[f][h][u * 8 + 2 * c + 1]);
                store16(o, yb);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    }

    static __device__ __forceinline__ void block(const MmArgs& g, char* sm, int* pre) {
        const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wi = wave % NWI, wj = wave / NWI;
        const int ld2 = g.R * 2;   // bytes of a row of codes
        const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)sm;
        const int nj = (g.J + BJ - 1) / BJ, ksteps = (g.R + 63) / 64;
        count_tiles<MM_FWD, BI>(g, pre, 0x70000000 / nj);
        const int tiles = __builtin_amdgcn_readfirstlane(pre[g.E]) * nj;
        if (g.fill && g.offsets) fill_rest<MM_FWD>(g);
        const MmRun run = xcd_run<BI >= 128 ? 2 : 1>(tiles);
        auto tile = [&](int id, MmTile& t) {
            tile_at<MM_FWD, BI, BJ>(g, pre, run.tile(id), t);
            if (id >= run.whole) {   // a piece (the last ones of a tile with few rows are empty)
                const int n = BI >> run.cut, lo = ((id - run.whole) & ((1 << run.cut) - 1)) * n;
                t.lo += lo;
                t.rows = max(0, min(n, t.rows - lo));
            }
        };
        auto r_of = [&](const MmTile& t) -> int { return g.part ? min(g.part, g.R - t.e * g.part) : g.R; };
        auto steps_of = [&](const MmTile& t) -> int { return t.rows ? (r_of(t) + 63) / 64 : 0; };
        auto next_buf = [](uint32_t b) -> uint32_t { return b == (ST - 1) * STAGE ? 0 : b + STAGE; };
        if (run.first == MmRun::NONE) return;

        if (wave >= NWC) {   // loads: ST stages ahead, past the last tile from empty descriptors
            const int lw = wave - NWC, row = 8 * lw + (lane >> 3), piece = lane & 7;
            int lid = -1, ls = 0, lsteps = 0, lrows = 0, lr = 0;
            MmTile lt{};
            const char *pa = nullptr, *pb = nullptr;
            uint32_t offa[PA], offb[PB], offs = 0;   // offs: GATHER, of x's exponents
            auto next_tile = [&]() {
                ls = 0;
                do {
                    lid = lid < 0 ? run.first : run.next(lid);
                    if (lid == MmRun::NONE) {
                        lsteps = 0x7fffffff;
                        lrows = 0;
                        return;
                    }
                    tile(lid, lt);
                    lsteps = steps_of(lt);
                } while (lsteps == 0);
                lrows = lt.rows;
                lr = r_of(lt);
                const int first = lt.e * g.part;   // the part's first word
                pa = (const char*)g.a + (GATHER ? 0 : (int64_t)lt.lo * ld2) + (int64_t)first * 2;
                pb = (const char*)g.b + ((int64_t)(g.part ? 0 : lt.e) * g.J + lt.j0) * ld2 + (int64_t)first * 2;
#pragma unroll
                for (int i = 0; i < PA; ++i) {
                    const int r = row + 8 * NL * i, c = (piece ^ swz(r)) * 16;
                    int src = r;
                    if constexpr (GATHER) src = r < lt.rows ? g.arows[lt.lo + r] : -1;
                    offa[i] = !GATHER || (uint32_t)src < (uint32_t)g.a_n ? (uint32_t)src * (uint32_t)ld2 + c : MM_OOB;
                }
                if constexpr (GATHER) {
                    const int r = lw % SG * 32 + (lane >> 1), src = r < lt.rows ? g.arows[lt.lo + r] : -1;
                    offs = (uint32_t)src < (uint32_t)g.a_n ? (uint32_t)src * 8 + (lane & 1) * 4 : MM_OOB;
                }
#pragma unroll
                for (int i = 0; i < PB; ++i) {
                    const int r = row + 8 * NL * i;
                    offb[i] = (uint32_t)r * (uint32_t)ld2 + (piece ^ swz(r)) * 16;
                }
            };
            auto load = [&](uint32_t buf) {   // step ls
                const int left = (lr - 64 * ls) * 2;   // bytes of a row from here on
                if (left < 128 && lrows) {             // the last step ends inside a row: its pieces past the end
#pragma unroll
                    for (int i = 0; i < PA; ++i)
                        if ((piece ^ swz(row + 8 * NL * i)) * 16 >= left) offa[i] = MM_OOB;
#pragma unroll
                    for (int i = 0; i < PB; ++i)
                        if ((piece ^ swz(row + 8 * NL * i)) * 16 >= left) offb[i] = MM_OOB;
                }
                const uint32_t na = lrows ? (uint32_t)((GATHER ? g.a_n : lrows) - 1) * (uint32_t)ld2 + (uint32_t)left : 0,
                               nb = lrows ? (uint32_t)(min(BJ, g.J - lt.j0) - 1) * (uint32_t)ld2 + (uint32_t)left : 0;
                const srd_t da = srd_of(pa, na), db = srd_of(pb, nb);
                constexpr int NA = PA < 4 ? PA : 4, NB = PB < 4 ? PB : 4;
#pragma unroll
                for (int i = 0; i < PB; i += NB) dma16<NB, NL * 1024>(db, offb + i, lds0 + buf + (uint32_t)(BI * 128 + (i * NL + lw) * 1024));
#pragma unroll
                for (int i = 0; i < PA; i += NA) dma16<NA, NL * 1024>(da, offa + i, lds0 + buf + (uint32_t)((i * NL + lw) * 1024));
                // this wave's piece of a's or b's exponents, GATHER: of each (waves past the last piece load one again)
                const int p = GATHER ? SCA + lw % SCB : lw % (SCA + SCB), step = ls + (g.part ? lt.e * (g.part / 64) : 0), e = g.part ? 0 : lt.e;
                if constexpr (GATHER)
                    dma4(srd_of((const char*)g.sa + (int64_t)step * g.a_n * 8, lrows ? (uint32_t)g.a_n * 8 : 0u), offs,
                         lds0 + buf + CODES + lw % SG * 256);
                const uint8_t* s = g.sa + ((int64_t)step * g.a_n + lt.lo) * 8 + p * 1024;
                int n = (lrows * 8 + 15) / 16 * 16 - p * 1024;
                if (p >= SCA) {
                    s = g.sb + (((int64_t)e * ksteps + step) * g.J + lt.j0) * 8 + (p - SCA) * 1024;
                    n = (g.J - lt.j0) * 8 - (p - SCA) * 1024;
                }
                const uint32_t off = lane * 16;
                dma16<1, 0>(srd_of((const char*)s, lrows && n > 0 ? n : 0), &off, lds0 + buf + CODES + p * 1024);
                ++ls;
                pa += 128;
                pb += 128;
            };
            uint32_t wbuf = 0;
#pragma unroll
            for (int s = 0; s < ST; ++s) {
                if (ls >= lsteps) next_tile();
                load(wbuf);
                wbuf = next_buf(wbuf);
            }
            wait_vm<(ST - 1) * L>();
            barrier_raw();
            for (int id = run.first; id != MmRun::NONE; id = run.next(id)) {
                MmTile t;
                tile(id, t);
                for (int s = steps_of(t); s > 0; --s) {
                    if (ls >= lsteps) next_tile();
                    wait_vm<(ST - 2) * L>();
                    barrier_raw();   // the stage that is multiplied next has landed, the last one is free
                    load(wbuf);
                    wbuf = next_buf(wbuf);
                }
            }
            wait_vm<0>();   // no load may still write this workgroup's LDS when it ends
            return;
        }

        const int r = lane & 31, hb = lane >> 5;
        uint32_t fa[FA], fb[FB], xa[FA], xb[FB];   // LDS offsets: the fragments of k 0 .. 63, and the exponents' words
#pragma unroll
        for (int f = 0; f < FA; ++f) {
            const int i = 32 * (NWI * f + wi) + r;
            fa[f] = i * 128 + (hb ^ swz(i)) * 16;
            xa[f] = CODES + i * 8 + hb * 4;
        }
#pragma unroll
        for (int h = 0; h < FB; ++h) {
            const int j = 32 * (FB * wj + h) + column(r);
            fb[h] = BI * 128 + j * 128 + (hb ^ swz(j)) * 16;
            xb[h] = CODES + SCA * 1024 + j * 8 + hb * 4;
        }
        f32x16 acc[FA][FB];
        s16x8 ra[2][FA], rb[2][FB];        // fragments of the quarter step that is multiplied and of the next one
        uint32_t ea[2][FA], eb[2][FB];   // exponents of the step that is multiplied and of the next one
        auto read = [&](const char* st, int set, int ks) {
#pragma unroll
            for (int h = 0; h < FB; ++h) rb[set][h] = *(const s16x8*)(st + (fb[h] ^ (ks * 32)));
#pragma unroll
            for (int f = 0; f < FA; ++f) ra[set][f] = *(const s16x8*)(st + (fa[f] ^ (ks * 32)));
        };
        auto read_exponents = [&](const char* st, int set) {
#pragma unroll
            for (int h = 0; h < FB; ++h) eb[set][h] = *(const uint32_t*)(st + xb[h]);
#pragma unroll
            for (int f = 0; f < FA; ++f) ea[set][f] = *(const uint32_t*)(st + xa[f]);
        };
        barrier_raw();
        uint32_t rbuf = 0;
        for (int id = run.first; id != MmRun::NONE; id = run.next(id)) {
            MmTile t;
            tile(id, t);
            const int steps = steps_of(t), nf = (t.rows + 32 * NWI - 1) / (32 * NWI);
            float zero;   // opaque: zeros kept in accumulation registers for the next tile would take them from the sums
            asm volatile("v_mov_b32 %0, 0" : "=v"(zero));
#pragma unroll
            for (int f = 0; f < FA; ++f)
#pragma unroll
                for (int h = 0; h < FB; ++h)
#pragma unroll
                    for (int i = 0; i < 16; ++i) acc[f][h][i] = zero;
            read(sm + rbuf, 0, 0);   // again after the last tile's stores, which need the registers
            read_exponents(sm + rbuf, 0);
            auto mul = [&](auto ks) {
                constexpr int K = decltype(ks)::value, set = K & 1;
#pragma unroll
                for (int f = 0; f < FA; ++f)
                    if (f < nf) {
#pragma unroll
                        for (int h = 0; h < FB; ++h) acc[f][h] = mma32<K>(rb[set][h], eb[0][h], ra[set][f], ea[0][f], acc[f][h]);
                    }
            };
#pragma nounroll
            for (int s = 0; s < steps; ++s) {
                read(sm + rbuf, 1, 1);
                mul(std::integral_constant<int, 0>{});
                __builtin_amdgcn_sched_barrier(0);
                read(sm + rbuf, 0, 2);
                mul(std::integral_constant<int, 1>{});
                __builtin_amdgcn_sched_barrier(0);
                read(sm + rbuf, 1, 3);
                mul(std::integral_constant<int, 2>{});
                // every read of this stage is done, so once all waves are here it is free for the loads; and the next stage has
                // landed
                wait_lds();
                barrier_raw();
                rbuf = next_buf(rbuf);
                read(sm + rbuf, 0, 0);
                read_exponents(sm + rbuf, 1);
                mul(std::integral_constant<int, 3>{});
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int h = 0; h < FB; ++h) eb[0][h] = eb[1][h];
#pragma unroll
                for (int f = 0; f < FA; ++f) ea[0][f] = ea[1][f];
            }
            store(g, t, acc, lane, wi, wj);
        }
    }
};

template <bool F16, int FA, int FB, int NWI, int NWJ, int ST, int OCC, int GATHER, int EPI, int NL>
__global__ void __launch_bounds__(64 * (NWI * NWJ + NL), OCC * (NWI * NWJ + NL) / 4) k_mm_mx4(const MmArgs g) {
    using K = MxKernel<F16, FA, FB, NWI, NWJ, ST, GATHER, EPI, NL>;
    __shared__ __attribute__((aligned(1024))) char sm[ST * K::STAGE];
    __shared__ int pre[MM_MAX_E + 1];
    static_assert(sizeof(sm) + sizeof(pre) <= 160 * 1024 / OCC, "");
    K::block(g, sm, pre);
}

template <bool F16, int FA, int FB, int NWI, int NWJ, int ST, int OCC, int NL>
static int launch_cfg(const MmArgs& a, hipStream_t st) {
    constexpr int BI = 32 * FA * NWI, BJ = 32 * FB * NWJ;
    const int64_t ni = mm_row_tiles(a, BI), nj = (a.J + BJ - 1) / BJ;
    if (ni * nj == 0) return MOE_OK;
    if (ni * nj > 0x70000000) return MOE_ERR_ARG;
    constexpr int CUT = BI >= 128 ? 4 : 2;   // pieces that a tile can be cut into
    const int64_t most = 256 * OCC, grid = round8(CUT * ni * nj) < most ? round8(CUT * ni * nj) : most;   // 256 CUs
    auto run = [&](auto lists, auto epi) {
        k_mm_mx4<F16, FA, FB, NWI, NWJ, ST, OCC, decltype(lists)::value, decltype(epi)::value, NL>
            <<<(unsigned)grid, 64 * (NWI * NWJ + NL), 0, st>>>(a);
    };
    auto go = [&](auto lists) {
        if (a.kind != EPI_LIN) run(lists, std::integral_constant<int, MX_PLAIN>{});
        else run(lists, std::integral_constant<int, MX_LIN>{});
    };
    if (a.arows) go(std::integral_constant<int, 1>{});   // moe_mx4_grouped_mm: no activation
    else if (a.epi.act != MOE_LIN_NONE) run(std::integral_constant<int, 0>{}, std::integral_constant<int, MX_ACT>{});
    else go(std::integral_constant<int, 0>{});
    return hipGetLastError() == hipSuccess ? MOE_OK : MOE_ERR_LAUNCH;
}

// A group has about M / 128 + 1/2 row tiles of 128, one at least. Where that makes a tile of 128 x 256 for every CU, it reads the
// weights fastest, however few rows use them (us in 64 x 64, 128 x 128, 128 x 256 tiles: 128 experts x 4 rows, [1536, 2048], 42.8,
// 43.4, 37.1; 64 x 8, [2048, 2048], 29.6, 30.9, 27.4; x 256 rows of 128 experts 156, 87, 78). With fewer, up to 32 rows in
// smaller tiles (8 experts x 32, [4096, 4096]: 16.2, 17.4, 18.4), and more rows in 128 x 128 while those are one round of the CUs
// (4 x 256, [2048, 2048]: 11.1, 9.9, 11.7).
static int grouped(const MmArgs& a) {
    const int64_t live = a.E < a.M ? a.E : a.M, half = live / 2 + a.M / 128, tiles = live > half ? live : half;
    if (tiles * ((a.J + 255) / 256) >= 256) return MM_128x256;
    if (a.M / live <= 32) return MM_64;
    return half * ((a.J + 127) / 128) <= 256 ? MM_128_DEEP : MM_128x256;
}

// The 16-bit products' plan (E: parts), but 64 x 64 only while a CU has one of them at most: codes arrive so fast that a second round
// costs more than larger tiles do (us in 64 x 64 and 128 x 128 tiles: 512 rows, [4096, 4096], 14.4 and 12.7, 256 rows 10.4 and 12.2;
// 128 rows, [14336, 4096], 14.6 and 13.1).
static int dense(const MmArgs& a) {
    const int shape = mm_plan(MM_FWD, a.M, a.J, a.R, a.part != 0).shape;
    return shape == MM_64 && ((int64_t)a.M + 63) / 64 * ((a.J + 63) / 64) * a.E > 256 ? MM_128_DEEP : shape;
}

template <bool F16>
static int launch(const MmArgs& a, hipStream_t st) {
    switch (a.offsets ? grouped(a) : dense(a)) {
        case MM_128x256: return launch_cfg<F16, 2, 2, 2, 4, 3, 1, 4>(a, st);
        case MM_128_DEEP: return launch_cfg<F16, 2, 2, 2, 2, 4, 1, 4>(a, st);
        default: return launch_cfg<F16, 1, 1, 2, 2, 4, 2, 4>(a, st);
    }
}
int launch_mm_mx4(const MmArgs& a, hipStream_t st) { return a.f16 ? launch<true>(a, st) : launch<false>(a, st); }

}  // namespace moe
