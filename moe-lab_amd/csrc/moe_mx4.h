// MXFP4 operands made on the device: E2M1 codes, two to a byte, the low half first, with an E8M0 byte per 32 neighbours.
// A matrix of `rows` rows and K columns is codes [rows, K / 2] and scales [steps, rows, 8], steps = ceil(K / 256): byte
// mx4_byte(b) of (s, row) belongs to the columns 256 s + 32 b ... The products take a step of all rows of a tile at a time, so
// those bytes lie together (in rows of their own, K / 32 bytes each, a tile's step would be a hundred lines for 8 bytes of each),
// the even blocks' before the odd ones': a lane of the matrix instruction holds every second block, so its four bytes are a word.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "moe_mm.h"

namespace moe {

struct Mx4 {
    uint8_t* codes;
    uint8_t* scales;
};
// Bytes of a matrix's scales. Reads of 16 bytes may start at any row, so 8 more lie behind the last one (16: whole pieces).
__host__ __device__ constexpr int mx4_byte(int b) { return (b & 1) * 4 + (b >> 1); }
inline int64_t mx4_steps(int64_t K) { return (K + 255) / 256; }
inline size_t mx4_scale_bytes(int64_t rows, int64_t K) { return (size_t)(mx4_steps(K) * rows * 8 + 16); }

// x: G matrices of `rows` rows each, ld elements between rows (G > 1: contiguous)
int launch_mx4_quantize(const void* x, int64_t ld, int64_t G, int64_t rows, int64_t K, int dtype, Mx4 out, hipStream_t st);
int launch_mx4_dequantize(const uint8_t* codes, const uint8_t* scales, int64_t G, int64_t rows, int64_t K, int dtype, void* out,
                          hipStream_t st);
// Products of few rows per group. x16 not null: a.a's rows are 16-bit numbers of the result's type there (ldx elements between
// them), quantised by every workgroup for itself; else a.a, a.sa (not gathered: row arows[p]).
int launch_mx4_rows(const MmArgs& a, const void* x16, int64_t ldx, hipStream_t st);
// Dense products that the few-rows kernel takes: it reads x once per 16 rows of the weights, the tiles once per 64 or more (16 rows,
// w [4096, 4096]: 4.9 us, in tiles 8.7; 32 rows 6.4 and 8.7, w [14336, 4096] 17.1 and 13.7).
inline bool mx4_few_rows(int64_t T, int64_t N) { return T <= 16 || (T <= 32 && N <= 8192); }
// Sums of dy's rows by group (gradients of biases beside frozen weights): groups of a.M slots, dy = a.a (a.lda), N = a.J, into y
// of dy's type. parts: pieces of a group that workgroups share, > 1: joined from `sums`, fp32 [parts, E, N].
int mx4_sum_parts(int64_t M, int64_t E, int64_t N);
int launch_mx4_sums(const MmArgs& a, int parts, float* sums, hipStream_t st);
int mx4_dx_parts(int64_t rows, int64_t N, int64_t K);   // parts of a dense product of dx (moe_mm_mx4_dx.hip)
// Rows from which a dense dx multiplies by the weights' values, written out once, and not by the codes, which each tile of 128 rows
// decodes anew (us from codes and values, w [4096, 4096]: 2048 rows 72 and 73, 4096 rows 148 and 128, 8192 rows 250 and 231).
constexpr int64_t MX4_DECODE_ONCE = 4096;
constexpr int MX4_FUSE = 4;       // rows that are quantised inside the product (k_mx4_rows)
constexpr int64_t MX4_FUSE_K = 1 << 16;   // and their elements in all, at most (LDS)

}  // namespace moe
