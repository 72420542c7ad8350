// C entry points of the MXFP4 operators (include/moe_mi355x.h): argument checks, then the launchers.
#include "moe_mx4.h"

namespace {
bool misaligned(const void* p) { return ((uintptr_t)p & 15) != 0; }
bool two_byte(int dtype) { return dtype == MOE_DTYPE_BF16 || dtype == MOE_DTYPE_F16; }
bool bad_k(int64_t K) { return K < 32 || K % 32 || K > (1 << 20); }
bool bad_n(int64_t N) { return N < 8 || N % 8 || N > (1 << 20); }
bool bad_ld(int64_t ld, int64_t K) { return ld < K || ld % 8 || ld > (1 << 21); }
constexpr int64_t MAX_ROWS = 0x7fffff00;   // rows and slots are counted in 32 bits, in steps of up to 64 past the last one
bool bad_rows(int64_t n) { return n < 0 || n > MAX_ROWS; }
size_t up256(size_t n) { return (n + 255) / 256 * 256; }
// x's codes and scales in a workspace
size_t x_bytes(int64_t rows, int64_t K) { return up256((size_t)rows * (K / 2)) + up256(moe::mx4_scale_bytes(rows, K)); }
// whether x's rows are quantised inside the product of few rows
bool fused(int64_t rows, int64_t K) { return rows <= moe::MX4_FUSE && moe::MX4_FUSE * K <= moe::MX4_FUSE_K; }

// grouped: whether a group has one slot on average, of those that can have any
bool few_slots(int64_t M, int64_t E) { return M / (E < M ? E : M) <= 1; }

struct Problem {
    const void *x, *xc, *xs, *wc, *ws;
    int64_t x_rows, ldx;
    int K;
};
int check(const Problem& p, int N, int dtype, int y_dtype) {
    if (!two_byte(dtype) || (y_dtype != dtype && y_dtype != MOE_DTYPE_F32)) return MOE_ERR_DTYPE;
    if (bad_n(N) || bad_k(p.K) || bad_rows(p.x_rows) || (p.x && bad_ld(p.ldx, p.K))) return MOE_ERR_ARG;
    return MOE_OK;
}
int check_pointers(const Problem& p, const void* y) {
    if (!p.wc || !p.ws || !y || (!p.x && !p.xc) || !p.xc != !p.xs) return MOE_ERR_ARG;
    if (misaligned(p.x) || misaligned(p.xc) || misaligned(p.xs) || misaligned(p.wc) || misaligned(p.ws) || misaligned(y))
        return MOE_ERR_ALIGN;
    return MOE_OK;
}
// a.a and a.sa: x's form, made here from 16-bit rows
int operand(const Problem& p, int dtype, char*& ws, moe::MmArgs& a, hipStream_t st) {
    moe::Mx4 q{(uint8_t*)const_cast<void*>(p.xc), (uint8_t*)const_cast<void*>(p.xs)};
    if (p.x) {
        if (!q.codes) {
            q = {(uint8_t*)ws, (uint8_t*)ws + up256((size_t)p.x_rows * (p.K / 2))};
            ws += x_bytes(p.x_rows, p.K);
        }
        const int rc = moe::launch_mx4_quantize(p.x, p.ldx, 1, p.x_rows, p.K, dtype, q, st);
        if (rc) return rc;
    }
    a.a = q.codes;
    a.sa = q.scales;
    return MOE_OK;
}
moe::MmArgs product(const Problem& p, int64_t M, int E, int N, int dtype, void* y, int y_dtype) {
    moe::MmArgs a{};
    a.b = p.wc;
    a.sb = (const uint8_t*)p.ws;
    a.y = y;
    a.M = (int)M;
    a.a_n = (int)p.x_rows;
    a.lda = a.ldb = a.R = p.K / 4;
    a.E = E;
    a.J = N;
    a.f16 = dtype == MOE_DTYPE_F16;
    a.ydt = y_dtype;
    return a;
}
moe::MmArgs gradient(const void* dy, int64_t ld, const void* wc, const void* ws, int64_t M, int E, int N, int K, int dtype, void* dx,
                     int dx_dtype) {
    moe::MmArgs a{};
    a.a = dy;
    a.b = wc;
    a.sb = (const uint8_t*)ws;
    a.y = dx;
    a.M = a.a_n = (int)M;
    a.lda = (int)ld;
    a.ldb = K;
    a.E = E;
    a.J = K;
    a.R = N;
    a.f16 = dtype == MOE_DTYPE_F16;
    a.ydt = dx_dtype;
    return a;
}
size_t linear_parts(int64_t T, int N, int K) {
    if (moe::mx4_few_rows(T, N)) return 0;
    const int parts = moe::mm_plan(moe::MM_FWD, T, N, K / 4, true).parts;
    return parts > 1 ? up256((size_t)parts * T * N * 4) : 0;
}
}  // namespace

extern "C" {

size_t moe_mx4_scale_bytes(int64_t matrices, int64_t rows, int K) {
    if (matrices < 0 || bad_rows(rows) || bad_k(K)) return 0;
    return (size_t)(matrices * moe::mx4_steps(K) * rows * 8 + 16);
}

int moe_mx4_quantize(const void* x, int64_t ldx, int64_t matrices, int64_t rows, int K, int dtype, void* codes, void* scales,
                     void* stream) {
    if (!two_byte(dtype) && dtype != MOE_DTYPE_F32) return MOE_ERR_DTYPE;
    if (matrices < 0 || bad_rows(rows) || bad_k(K) || bad_ld(ldx, K) || (matrices > 1 && ldx != K)) return MOE_ERR_ARG;
    if (matrices * rows == 0) return MOE_OK;
    if (matrices > MAX_ROWS / rows || !x || !codes || !scales) return MOE_ERR_ARG;
    if (misaligned(x) || misaligned(codes) || misaligned(scales)) return MOE_ERR_ALIGN;
    return moe::launch_mx4_quantize(x, ldx, matrices, rows, K, dtype, moe::Mx4{(uint8_t*)codes, (uint8_t*)scales},
                                    (hipStream_t)stream);
}

int moe_mx4_dequantize(const void* codes, const void* scales, int64_t matrices, int64_t rows, int K, void* out, int dtype,
                       void* stream) {
    if (!two_byte(dtype) && dtype != MOE_DTYPE_F32) return MOE_ERR_DTYPE;
    if (matrices < 0 || bad_rows(rows) || bad_k(K)) return MOE_ERR_ARG;
    if (matrices * rows == 0) return MOE_OK;
    if (matrices > MAX_ROWS / rows || !out || !codes || !scales) return MOE_ERR_ARG;
    if (misaligned(out) || misaligned(codes) || misaligned(scales)) return MOE_ERR_ALIGN;
    return moe::launch_mx4_dequantize((const uint8_t*)codes, (const uint8_t*)scales, matrices, rows, K, dtype, out,
                                      (hipStream_t)stream);
}

size_t moe_mx4_linear_workspace_bytes(int64_t T, int N, int K) {
    if (bad_rows(T) || T == 0 || bad_n(N) || bad_k(K)) return 0;
    return (fused(T, K) ? 0 : x_bytes(T, K)) + linear_parts(T, N, K);
}

int moe_mx4_linear(const void* x, int64_t ldx, void* xc, void* xs, const void* wc, const void* ws, const void* bias,
                   const void* residual, int act, int64_t T, int N, int K, int dtype, void* y, int y_dtype, void* z,
                   void* workspace, size_t workspace_bytes, void* stream) {
    const Problem p{x, xc, xs, wc, ws, T, ldx, K};
    int rc = check(p, N, dtype, y_dtype);
    if (rc) return rc;
    if (act < MOE_LIN_NONE || act > MOE_LIN_GELU) return MOE_ERR_ARG;
    if (T == 0) return MOE_OK;
    rc = check_pointers(p, y);
    if (rc) return rc;
    if (misaligned(bias) || misaligned(residual) || misaligned(z) || misaligned(workspace)) return MOE_ERR_ALIGN;
    const size_t need = moe_mx4_linear_workspace_bytes(T, N, K);
    if (workspace_bytes < need || (need && !workspace)) return MOE_ERR_WORKSPACE;
    const hipStream_t st = (hipStream_t)stream;
    moe::MmArgs a = product(p, T, 1, N, dtype, y, y_dtype);
    a.epi = moe::MmEpi{bias, residual, z, act, nullptr, nullptr, nullptr};
    a.kind = bias || residual || z || act != MOE_LIN_NONE ? moe::EPI_LIN : moe::EPI_PLAIN;
    if (x && !xc && fused(T, K)) return moe::launch_mx4_rows(a, x, ldx, st);
    char* w = (char*)workspace;
    rc = operand(p, dtype, w, a, st);
    if (rc) return rc;
    if (moe::mx4_few_rows(T, N)) return moe::launch_mx4_rows(a, nullptr, 0, st);
    const int parts = moe::mm_plan(moe::MM_FWD, T, N, K / 4, true).parts;
    if (parts > 1) return moe::launch_mm_parts(moe::MM_FWD, a, parts, (float*)w, st);
    return moe::launch_mm_fwd(a, st);
}

size_t moe_mx4_linear_dx_workspace_bytes(int64_t T, int N, int K) {
    if (bad_rows(T) || T == 0 || bad_n(N) || bad_k(K)) return 0;
    if (T >= moe::MX4_DECODE_ONCE) return up256((size_t)N * K * 2) + moe_linear_dx_workspace_bytes(T, N, K);
    const int parts = moe::mx4_dx_parts(T, N, K);
    return parts > 1 ? (size_t)parts * T * K * 4 : 0;
}

int moe_mx4_linear_dx(const void* dz, int64_t lddz, const void* wc, const void* ws, int64_t T, int N, int K, int dtype, void* dx,
                      void* workspace, size_t workspace_bytes, void* stream) {
    if (!two_byte(dtype)) return MOE_ERR_DTYPE;
    if (bad_rows(T) || bad_n(N) || bad_k(K) || bad_ld(lddz, N)) return MOE_ERR_ARG;
    if (T == 0) return MOE_OK;
    if (!dz || !wc || !ws || !dx) return MOE_ERR_ARG;
    if (misaligned(dz) || misaligned(wc) || misaligned(ws) || misaligned(dx) || misaligned(workspace)) return MOE_ERR_ALIGN;
    const size_t need = moe_mx4_linear_dx_workspace_bytes(T, N, K);
    if (workspace_bytes < need || (need && !workspace)) return MOE_ERR_WORKSPACE;
    if (T >= moe::MX4_DECODE_ONCE) {
        const int rc = moe::launch_mx4_dequantize((const uint8_t*)wc, (const uint8_t*)ws, 1, N, K, dtype, workspace, (hipStream_t)stream);
        if (rc) return rc;
        const size_t used = up256((size_t)N * K * 2);
        return moe_linear_dx(dz, workspace, T, lddz, N, K, dtype, dx, (char*)workspace + used, workspace_bytes - used, stream);
    }
    const moe::MmArgs a = gradient(dz, lddz, wc, ws, T, 1, N, K, dtype, dx, dtype);
    const int parts = moe::mx4_dx_parts(T, N, K);
    if (parts > 1) return moe::launch_mm_parts(moe::MM_DX, a, parts, (float*)workspace, (hipStream_t)stream);
    return moe::launch_mm_dx(a, (hipStream_t)stream);
}

size_t moe_mx4_linear_bwd_workspace_bytes(int64_t T, int N, int K, int act, int dx, int dw, int db) {
    if (bad_rows(T) || bad_n(N) || bad_k(K)) return 0;
    size_t n = 0, m = 0;   // dz and x's values; the gradients' own, one after the other
    if (act != MOE_LIN_NONE) n += up256((size_t)T * N * 2);
    if (dw) n += up256((size_t)T * K * 2);
    if (dx) m = moe_mx4_linear_dx_workspace_bytes(T, N, K);
    const size_t w = dw ? moe_linear_dw_workspace_bytes(T, N, K) : db ? moe_mx4_bias_grad_workspace_bytes(T, 1, N) : 0;
    return n + (w > m ? w : m);
}

int moe_mx4_linear_bwd(const void* dy, int64_t lddy, const void* z, int act, const void* xc, const void* xs, const void* wc,
                       const void* ws, int64_t T, int N, int K, int dtype, void* dx, void* dw, void* db, void* workspace,
                       size_t workspace_bytes, void* stream) {
    if (!two_byte(dtype)) return MOE_ERR_DTYPE;
    if (act < MOE_LIN_NONE || act > MOE_LIN_GELU) return MOE_ERR_ARG;
    if (bad_rows(T) || bad_n(N) || bad_k(K) || bad_ld(lddy, N)) return MOE_ERR_ARG;
    if (T && (!dy || (act != MOE_LIN_NONE && !z) || (dx && (!wc || !ws)) || (dw && (!xc || !xs)))) return MOE_ERR_ARG;
    if (misaligned(dy) || misaligned(z) || misaligned(xc) || misaligned(xs) || misaligned(wc) || misaligned(ws) || misaligned(dx) ||
        misaligned(dw) || misaligned(db) || misaligned(workspace))
        return MOE_ERR_ALIGN;
    const size_t need = moe_mx4_linear_bwd_workspace_bytes(T, N, K, act, dx != nullptr, dw != nullptr, db != nullptr);
    if (workspace_bytes < need || (need && !workspace)) return MOE_ERR_WORKSPACE;
    char* w = (char*)workspace;
    const auto take = [&](size_t n) {
        char* p = w;
        w += up256(n);
        workspace_bytes -= up256(n);
        return p;
    };
    int rc = MOE_OK;
    if (act != MOE_LIN_NONE) {
        void* dz = take((size_t)T * N * 2);
        rc = moe_linear_act_bwd(dy, lddy, z, nullptr, nullptr, act, T, N, dtype, dz, stream);
        dy = dz;
        lddy = N;
    }
    void* x = dw ? take((size_t)T * K * 2) : nullptr;
    if (!rc && dx) rc = moe_mx4_linear_dx(dy, lddy, wc, ws, T, N, K, dtype, dx, w, workspace_bytes, stream);
    if (!rc && dw) {
        rc = moe_mx4_dequantize(xc, xs, 1, T, K, x, dtype, stream);
        if (!rc) rc = moe_linear_dw(dy, x, T, lddy, K, N, K, dtype, dw, db, w, workspace_bytes, stream);
    } else if (!rc && db) {
        rc = moe_mx4_bias_grad(dy, lddy, nullptr, T, 1, N, dtype, db, w, workspace_bytes, stream);
    }
    return rc;
}

int moe_mx4_grouped_mm_dx(const void* dy, int64_t lddy, const void* wc, const void* ws, const int32_t* offsets, int64_t M, int E,
                          int N, int K, int dtype, void* dx, int dx_dtype, int fill, void* stream) {
    if (!two_byte(dtype) || (dx_dtype != dtype && dx_dtype != MOE_DTYPE_F32)) return MOE_ERR_DTYPE;
    if (E < 1 || E > MM_MAX_E || (!offsets && E != 1) || bad_rows(M) || bad_n(N) || bad_k(K) || bad_ld(lddy, N)) return MOE_ERR_ARG;
    if (M == 0) return MOE_OK;
    if (!dy || !wc || !ws || !dx) return MOE_ERR_ARG;
    if (misaligned(dy) || misaligned(wc) || misaligned(ws) || misaligned(dx)) return MOE_ERR_ALIGN;
    moe::MmArgs a = gradient(dy, lddy, wc, ws, M, E, N, K, dtype, dx, dx_dtype);
    a.offsets = offsets;
    a.fill = fill;
    return moe::launch_mm_dx(a, (hipStream_t)stream);
}

size_t moe_mx4_bias_grad_workspace_bytes(int64_t M, int E, int N) {
    if (bad_rows(M) || E < 1 || E > MM_MAX_E || bad_n(N)) return 0;
    const int parts = moe::mx4_sum_parts(M, E, N);
    return parts > 1 ? (size_t)parts * E * N * 4 : 0;
}

int moe_mx4_bias_grad(const void* dy, int64_t lddy, const int32_t* offsets, int64_t M, int E, int N, int dtype, void* db,
                      void* workspace, size_t workspace_bytes, void* stream) {
    if (!two_byte(dtype)) return MOE_ERR_DTYPE;
    if (E < 1 || E > MM_MAX_E || (!offsets && E != 1) || bad_rows(M) || bad_n(N) || bad_ld(lddy, N)) return MOE_ERR_ARG;
    if (!db || (M && !dy)) return MOE_ERR_ARG;
    if (misaligned(dy) || misaligned(db) || misaligned(workspace)) return MOE_ERR_ALIGN;
    const size_t need = moe_mx4_bias_grad_workspace_bytes(M, E, N);
    if (workspace_bytes < need || (need && !workspace)) return MOE_ERR_WORKSPACE;
    moe::MmArgs a{};
    a.a = dy;
    a.y = db;
    a.offsets = offsets;
    a.M = (int)M;
    a.lda = (int)lddy;
    a.E = E;
    a.J = N;
    a.f16 = dtype == MOE_DTYPE_F16;
    return moe::launch_mx4_sums(a, moe::mx4_sum_parts(M, E, N), (float*)workspace, (hipStream_t)stream);
}

size_t moe_mx4_grouped_mm_workspace_bytes(int64_t M, int64_t x_rows, int E, int K, int has_form) {
    if (bad_rows(M) || bad_rows(x_rows) || M == 0 || E < 1 || bad_k(K)) return 0;
    if (few_slots(M, E) && !has_form && fused(1, K)) return 0;
    return has_form ? 0 : x_bytes(x_rows, K);
}

int moe_mx4_grouped_mm(const void* x, int64_t ldx, void* xc, void* xs, int64_t x_rows, const void* wc, const void* ws,
                       const void* bias, const int32_t* offsets, const int32_t* rows, int64_t M, int E, int N, int K, int dtype,
                       void* y, int y_dtype, int fill, void* workspace, size_t workspace_bytes, void* stream) {
    const Problem p{x, xc, xs, wc, ws, x_rows, ldx, K};
    int rc = check(p, N, dtype, y_dtype);
    if (rc) return rc;
    if (E < 1 || E > MM_MAX_E || (!offsets && E != 1) || bad_rows(M)) return MOE_ERR_ARG;
    if (M == 0) return MOE_OK;
    rc = check_pointers(p, y);
    if (rc) return rc;
    if (x_rows < (rows ? 1 : M)) return MOE_ERR_ARG;
    if (rows && x_rows * (K / 2) > 0xB0000000ll) return MOE_ERR_ARG;   // addressed with 32 bits from its start
    if (misaligned(bias) || misaligned(workspace)) return MOE_ERR_ALIGN;
    const size_t need = moe_mx4_grouped_mm_workspace_bytes(M, x_rows, E, K, xc != nullptr);
    if (workspace_bytes < need || (need && !workspace)) return MOE_ERR_WORKSPACE;
    const hipStream_t st = (hipStream_t)stream;
    moe::MmArgs a = product(p, M, E, N, dtype, y, y_dtype);
    a.offsets = offsets;
    a.arows = rows;
    a.fill = fill;
    a.epi.bias = bias;
    a.kind = bias ? moe::EPI_LIN : moe::EPI_PLAIN;
    const bool few = few_slots(M, E);
    if (few && x && !xc && fused(1, K)) return moe::launch_mx4_rows(a, x, ldx, st);
    char* w = (char*)workspace;
    rc = operand(p, dtype, w, a, st);
    if (rc) return rc;
    if (few) return moe::launch_mx4_rows(a, nullptr, 0, st);
    return moe::launch_mm_fwd(a, st);
}

}  // extern "C"
