// C entry points of the 16-bit products (include/moe_mi355x.h): argument checks, then one mode's launcher.
#include "moe_mm.h"
#include "moe_rows.h"

namespace {
bool misaligned(const void* p) { return ((uintptr_t)p & 15) != 0; }
// Columns and row strides: 16-byte pieces, and a tile's rows within a buffer descriptor's reach.
bool bad_dim(int64_t n) { return n < 8 || n % 8 || n > (1 << 20); }
bool bad_ld(int64_t ld, int64_t cols) { return ld < cols || ld % 8 || ld > (1 << 21); }
// Rows reached through a list are addressed with 32 bits from the matrix's start.
bool too_far(int64_t rows, int64_t ld) { return rows * ld * 2 > 0xB0000000ll; }
bool two_byte(int dtype) { return dtype == MOE_DTYPE_BF16 || dtype == MOE_DTYPE_F16; }
// Slots are counted in 32 bits, in steps of up to 64 past the last one and pieces of up to 128.
constexpr int64_t MAX_SLOTS = 0x7fffff00;
bool bad_groups(const int32_t* offsets, int E, int64_t M) {
    return E < 1 || E > MM_MAX_E || (!offsets && E != 1) || M < 0 || M > MAX_SLOTS;
}
bool bad_act8(int64_t M, int64_t C) { return M < 0 || M > 0x7fffffff || C < 32 || C % 32 || C > (1 << 20); }
bool bad_rows(const int32_t* idx, int64_t rows, int64_t M) { return rows > 0x7fffffff || rows < (idx ? 1 : M); }
// Workspace of a product in parts, with `more` floats per part behind the sums.
size_t parts_bytes(int mode, int64_t rows, int64_t J, int64_t R, int64_t more) {
    if (rows < 1 || J < 1 || R < 1) return 0;
    const int parts = moe::mm_plan(mode, rows, J, R, true).parts;
    return parts > 1 ? (size_t)parts * (rows * J + more) * 4 : 0;
}
size_t up256(size_t n) { return (n + 255) / 256 * 256; }

// Parts of the expert layer's buffers, in bytes from their start.
struct MlpLayout {
    size_t offsets, sorted, rows, pos, keep;                 // kept for the backward pass
    size_t counts, active, meta, chunks, h, ys, fwd;     // forward workspace
    size_t dh, dgu, hw, dxs, bwd;                            // backward workspace
    MlpLayout(const moe_mlp_t& m, int64_t n) {
        size_t at = 0;
        auto take = [&](size_t bytes) {
            const size_t o = at;
            at += up256(bytes);
            return o;
        };
        offsets = take((size_t)(m.E + 1) * 4);
        sorted = take((size_t)n * 4);
        rows = take((size_t)n * 4);
        pos = take((size_t)n * 4);
        keep = at;
        at = 0;
        counts = take((size_t)m.E * 4);
        active = take((size_t)m.E * 4);
        meta = take(16);
        chunks = take((size_t)256 * m.E * 4);
        h = take((size_t)n * m.F * 2);
        ys = take((size_t)n * m.d * 4);
        fwd = at;
        at = 0;
        dh = take((size_t)n * m.F * 4);
        dgu = take((size_t)n * 2 * m.F * 2);
        hw = take((size_t)n * m.F * 2);
        dxs = take((size_t)n * m.d * 4);
        bwd = at;
    }
};
int check_mlp(const moe_mlp_t* m, int T, int k) {
    if (!m || T < 0 || k < 1 || m->E < 1 || m->E > MM_MAX_E || (int64_t)T * k > moe::GROUP_MAX_SLOTS) return MOE_ERR_ARG;
    if (!two_byte(m->dtype)) return MOE_ERR_DTYPE;
    if (m->act < 0 || m->act > MOE_ACT_GPTOSS || bad_dim(m->d) || bad_act8(0, m->F) || bad_dim(2 * (int64_t)m->F))
        return MOE_ERR_ARG;
    if (!m->w_gate_up || !m->w_down) return MOE_ERR_ARG;
    if (misaligned(m->w_gate_up) || misaligned(m->w_down)) return MOE_ERR_ALIGN;
    if (too_far(T, m->d) || too_far(2 * (int64_t)m->F, m->d)) return MOE_ERR_ARG;
    return MOE_OK;
}
}  // namespace

extern "C" {

int moe_grouped_mm(const void* x, const void* w, const void* bias, const int32_t* offsets, const int32_t* rows, int64_t M,
                   int64_t x_rows, int64_t ldx, int E, int N, int K, int dtype, void* y, int y_dtype, int fill,
                   void* stream) {
    if (dtype != MOE_DTYPE_BF16 && dtype != MOE_DTYPE_F16) return MOE_ERR_DTYPE;
    if (y_dtype != dtype && y_dtype != MOE_DTYPE_F32) return MOE_ERR_DTYPE;
    if (bad_groups(offsets, E, M) || bad_dim(N) || bad_dim(K) || bad_ld(ldx, K)) return MOE_ERR_ARG;
    if (M == 0) return MOE_OK;
    if (!x || !w || !y || bad_rows(rows, x_rows, M)) return MOE_ERR_ARG;
    if (misaligned(x) || misaligned(w) || misaligned(y) || misaligned(bias)) return MOE_ERR_ALIGN;
    if (rows && too_far(x_rows, ldx)) return MOE_ERR_ARG;
    moe::MmArgs a{};
    a.a = x;
    a.b = w;
    a.offsets = offsets;
    a.arows = rows;
    a.y = y;
    a.M = (int)M;
    a.a_n = (int)x_rows;
    a.lda = (int)ldx;
    a.ldb = K;
    a.E = E;
    a.I = 0;
    a.J = N;
    a.R = K;
    a.f16 = dtype == MOE_DTYPE_F16;
    a.ydt = y_dtype;
    a.fill = fill;
    a.epi.bias = bias;
    a.kind = bias ? moe::EPI_LIN : moe::EPI_PLAIN;
    return moe::launch_mm_fwd(a, (hipStream_t)stream);
}

int moe_grouped_mm_dx(const void* dy, const void* w, const int32_t* offsets, const int32_t* rows, int64_t M,
                      int64_t dy_rows, int64_t lddy, int E, int N, int K, int dtype, void* dx, int dx_dtype, int fill,
                      void* stream) {
    if (dtype != MOE_DTYPE_BF16 && dtype != MOE_DTYPE_F16) return MOE_ERR_DTYPE;
    if (dx_dtype != dtype && dx_dtype != MOE_DTYPE_F32) return MOE_ERR_DTYPE;
    if (bad_groups(offsets, E, M) || bad_dim(N) || bad_dim(K) || bad_ld(lddy, N)) return MOE_ERR_ARG;
    if (M == 0) return MOE_OK;
    if (!dy || !w || !dx || bad_rows(rows, dy_rows, M)) return MOE_ERR_ARG;
    if (misaligned(dy) || misaligned(w) || misaligned(dx)) return MOE_ERR_ALIGN;
    if (rows && too_far(dy_rows, lddy)) return MOE_ERR_ARG;
    moe::MmArgs a{};
    a.a = dy;
    a.b = w;
    a.offsets = offsets;
    a.arows = rows;
    a.y = dx;
    a.M = (int)M;
    a.a_n = (int)dy_rows;
    a.lda = (int)lddy;
    a.ldb = K;
    a.E = E;
    a.J = K;
    a.R = N;
    a.f16 = dtype == MOE_DTYPE_F16;
    a.ydt = dx_dtype;
    a.fill = fill;
    return moe::launch_mm_dx(a, (hipStream_t)stream);
}

int moe_grouped_mm_dw(const void* dy, const void* x, const int32_t* offsets, const int32_t* dy_idx, const int32_t* x_idx,
                      int64_t M, int64_t dy_rows, int64_t lddy, int64_t x_rows, int64_t ldx, int E, int N, int K, int dtype,
                      void* dw, int dw_dtype, void* dbias, void* stream) {
    if (dtype != MOE_DTYPE_BF16 && dtype != MOE_DTYPE_F16) return MOE_ERR_DTYPE;
    if (dw_dtype != dtype && dw_dtype != MOE_DTYPE_F32) return MOE_ERR_DTYPE;
    if (bad_groups(offsets, E, M) || bad_dim(N) || bad_dim(K) || bad_ld(lddy, N) || bad_ld(ldx, K)) return MOE_ERR_ARG;
    if (!dw || (M > 0 && (!dy || !x))) return MOE_ERR_ARG;
    if (M > 0 && (bad_rows(dy_idx, dy_rows, M) || bad_rows(x_idx, x_rows, M))) return MOE_ERR_ARG;
    if (misaligned(dy) || misaligned(x) || misaligned(dw)) return MOE_ERR_ALIGN;
    // with a list for either operand both are addressed from their start
    if ((dy_idx || x_idx) && (too_far(dy_rows, lddy) || too_far(x_rows, ldx))) return MOE_ERR_ARG;
    moe::MmArgs a{};
    a.a = dy;
    a.b = x;
    a.offsets = offsets;
    a.arows = dy_idx;
    a.brows = x_idx;
    a.y = dw;
    a.dbias = dbias;
    a.M = (int)M;
    a.a_n = (int)dy_rows;
    a.b_n = (int)x_rows;
    a.lda = (int)lddy;
    a.ldb = (int)ldx;
    a.E = E;
    a.I = N;
    a.J = K;
    a.f16 = dtype == MOE_DTYPE_F16;
    a.ydt = dw_dtype;
    return moe::launch_mm_dw(a, (hipStream_t)stream);
}

size_t moe_linear_workspace_bytes(int64_t T, int N, int K) { return T <= moe::MM_FEW ? 0 : parts_bytes(moe::MM_FWD, T, N, K, 0); }
size_t moe_linear_dx_workspace_bytes(int64_t T, int N, int K) { return parts_bytes(moe::MM_DX, T, K, N, 0); }
size_t moe_linear_dw_workspace_bytes(int64_t T, int N, int K) { return parts_bytes(moe::MM_DW, N, K, T, N); }

int moe_linear(const void* x, const void* w, const void* bias, const void* residual, int act, int64_t T, int64_t ldx, int N,
               int K, int dtype, void* y, int y_dtype, void* z, void* workspace, size_t workspace_bytes, void* stream) {
    if (!two_byte(dtype) || (y_dtype != dtype && y_dtype != MOE_DTYPE_F32)) return MOE_ERR_DTYPE;
    if (act < MOE_LIN_NONE || act > MOE_LIN_GELU || T < 0 || T > MAX_SLOTS || bad_dim(N) || bad_dim(K) || bad_ld(ldx, K))
        return MOE_ERR_ARG;
    if (T == 0) return MOE_OK;
    if (!x || !w || !y) return MOE_ERR_ARG;
    if (misaligned(x) || misaligned(w) || misaligned(y) || misaligned(bias) || misaligned(residual) || misaligned(z) ||
        misaligned(workspace))
        return MOE_ERR_ALIGN;
    const size_t need = moe_linear_workspace_bytes(T, N, K);
    if (workspace_bytes < need || (need && !workspace)) return MOE_ERR_WORKSPACE;
    moe::MmArgs a{};
    a.a = x;
    a.b = w;
    a.y = y;
    a.M = (int)T;
    a.a_n = (int)T;
    a.lda = (int)ldx;
    a.ldb = K;
    a.E = 1;
    a.J = N;
    a.R = K;
    a.f16 = dtype == MOE_DTYPE_F16;
    a.ydt = y_dtype;
    a.epi = moe::MmEpi{bias, residual, z, act, nullptr, nullptr, nullptr};
    a.kind = bias || residual || z || act != MOE_LIN_NONE ? moe::EPI_LIN : moe::EPI_PLAIN;
    const int parts = T <= moe::MM_FEW ? 1 : moe::mm_plan(moe::MM_FWD, T, N, K, true).parts;
    if (parts > 1) return moe::launch_mm_parts(moe::MM_FWD, a, parts, (float*)workspace, (hipStream_t)stream);
    return moe::launch_mm_fwd(a, (hipStream_t)stream);
}

int moe_linear_dx(const void* dy, const void* w, int64_t T, int64_t lddy, int N, int K, int dtype, void* dx, void* workspace,
                  size_t workspace_bytes, void* stream) {
    if (!two_byte(dtype)) return MOE_ERR_DTYPE;
    if (T < 0 || T > MAX_SLOTS || bad_dim(N) || bad_dim(K) || bad_ld(lddy, N)) return MOE_ERR_ARG;
    if (T == 0) return MOE_OK;
    if (!dy || !w || !dx) return MOE_ERR_ARG;
    if (misaligned(dy) || misaligned(w) || misaligned(dx) || misaligned(workspace)) return MOE_ERR_ALIGN;
    const size_t need = moe_linear_dx_workspace_bytes(T, N, K);
    if (workspace_bytes < need || (need && !workspace)) return MOE_ERR_WORKSPACE;
    moe::MmArgs a{};
    a.a = dy;
    a.b = w;
    a.y = dx;
    a.M = (int)T;
    a.a_n = (int)T;
    a.lda = (int)lddy;
    a.ldb = K;
    a.E = 1;
    a.J = K;
    a.R = N;
    a.f16 = dtype == MOE_DTYPE_F16;
    a.ydt = dtype;
    const int parts = moe::mm_plan(moe::MM_DX, T, K, N, true).parts;
    if (parts > 1) return moe::launch_mm_parts(moe::MM_DX, a, parts, (float*)workspace, (hipStream_t)stream);
    return moe::launch_mm_dx(a, (hipStream_t)stream);
}

int moe_linear_dw(const void* dy, const void* x, int64_t T, int64_t lddy, int64_t ldx, int N, int K, int dtype, void* dw,
                  void* dbias, void* workspace, size_t workspace_bytes, void* stream) {
    if (!two_byte(dtype)) return MOE_ERR_DTYPE;
    if (T < 0 || T > MAX_SLOTS || bad_dim(N) || bad_dim(K) || bad_ld(lddy, N) || bad_ld(ldx, K)) return MOE_ERR_ARG;
    if (!dw || (T > 0 && (!dy || !x))) return MOE_ERR_ARG;
    if (misaligned(dy) || misaligned(x) || misaligned(dw) || misaligned(workspace)) return MOE_ERR_ALIGN;
    const size_t need = moe_linear_dw_workspace_bytes(T, N, K);
    if (workspace_bytes < need || (need && !workspace)) return MOE_ERR_WORKSPACE;
    moe::MmArgs a{};
    a.a = dy;
    a.b = x;
    a.y = dw;
    a.dbias = dbias;
    a.M = (int)T;
    a.a_n = (int)T;
    a.b_n = (int)T;
    a.lda = (int)lddy;
    a.ldb = (int)ldx;
    a.E = 1;
    a.I = N;
    a.J = K;
    a.f16 = dtype == MOE_DTYPE_F16;
    a.ydt = dtype;
    const int parts = moe::mm_plan(moe::MM_DW, N, K, T, true).parts;
    if (parts > 1) return moe::launch_mm_parts(moe::MM_DW, a, parts, (float*)workspace, (hipStream_t)stream);
    return moe::launch_mm_dw(a, (hipStream_t)stream);
}

int moe_linear_act_bwd(const void* dy, int64_t lddy, const void* z, const void* codes, const void* scales, int act, int64_t T,
                       int N, int dtype, void* dz, void* stream) {
    if (!two_byte(dtype)) return MOE_ERR_DTYPE;
    if ((act != MOE_LIN_SILU && act != MOE_LIN_GELU) || T < 0 || T > 0x7fffffff || bad_dim(N) || bad_ld(lddy, N))
        return MOE_ERR_ARG;
    if (codes && bad_act8(T, N)) return MOE_ERR_ARG;
    if (T == 0) return MOE_OK;
    if (!dy || !dz || (!z && (!codes || !scales)) || (z && codes)) return MOE_ERR_ARG;
    if (misaligned(dy) || misaligned(z) || misaligned(codes) || misaligned(dz)) return MOE_ERR_ALIGN;
    return moe::launch_lin_act_bwd(dy, lddy, z, (const uint8_t*)codes, (const uint8_t*)scales, T, N, act, dtype == MOE_DTYPE_F16,
                                   dz, (hipStream_t)stream);
}

int moe_act8_pack(const void* x, int64_t ldx, int64_t M, int C, int dtype, void* codes, void* scales, void* stream) {
    if (!two_byte(dtype)) return MOE_ERR_DTYPE;
    if (bad_act8(M, C) || bad_ld(ldx, C)) return MOE_ERR_ARG;
    if (M == 0) return MOE_OK;
    if (!x || !codes || !scales) return MOE_ERR_ARG;
    if (misaligned(x) || misaligned(codes)) return MOE_ERR_ALIGN;
    return moe::launch_pack8(x, ldx, M, C, dtype == MOE_DTYPE_F16, (uint8_t*)codes, (uint8_t*)scales, (hipStream_t)stream);
}

int moe_act8_unpack(const void* codes, const void* scales, int64_t M, int C, void* out, int dtype, void* stream) {
    if (!two_byte(dtype) && dtype != MOE_DTYPE_F32) return MOE_ERR_DTYPE;
    if (bad_act8(M, C)) return MOE_ERR_ARG;
    if (M == 0) return MOE_OK;
    if (!out || !codes || !scales) return MOE_ERR_ARG;
    if (misaligned(out) || misaligned(codes)) return MOE_ERR_ALIGN;
    return moe::launch_unpack8((const uint8_t*)codes, (const uint8_t*)scales, M, C, dtype, out, (hipStream_t)stream);
}

int moe_glu_fwd(const void* gu, int64_t ldgu, int64_t M, int F, int act, int dtype, void* h, void* codes, void* scales,
                void* stream) {
    if (!two_byte(dtype)) return MOE_ERR_DTYPE;
    if (act < 0 || act > MOE_ACT_GPTOSS || bad_act8(M, F) || bad_ld(ldgu, 2 * (int64_t)F)) return MOE_ERR_ARG;
    if (M == 0) return MOE_OK;
    if (!gu || !h || !codes != !scales) return MOE_ERR_ARG;
    if (misaligned(gu) || misaligned(h) || misaligned(codes)) return MOE_ERR_ALIGN;
    return moe::launch_glu_fwd(gu, ldgu, M, F, act, dtype == MOE_DTYPE_F16, h, (uint8_t*)codes, (uint8_t*)scales,
                               (hipStream_t)stream);
}

int moe_glu_bwd(const void* codes, const void* scales, const void* gu, int64_t ldgu, const void* dh, int dh_dtype,
                const float* wts, int64_t M, int F, int act, int dtype, void* dgu, void* hw, float* dwts, void* stream) {
    if (!two_byte(dtype) || (dh_dtype != dtype && dh_dtype != MOE_DTYPE_F32)) return MOE_ERR_DTYPE;
    if (act < 0 || act > MOE_ACT_GPTOSS || bad_act8(M, F)) return MOE_ERR_ARG;
    if (M == 0) return MOE_OK;
    if (!dh || !dgu || (codes ? !scales || gu : !gu || bad_ld(ldgu, 2 * (int64_t)F))) return MOE_ERR_ARG;
    if (misaligned(codes) || misaligned(gu) || misaligned(dh) || misaligned(dgu) || misaligned(hw)) return MOE_ERR_ALIGN;
    const moe::GluBwd a{(const uint8_t*)codes, (const uint8_t*)scales, (const uint16_t*)gu, ldgu, dh, dh_dtype == MOE_DTYPE_F32,
                        wts, nullptr, nullptr, M, F, act, (uint16_t*)dgu, (uint16_t*)hw, dwts};
    return moe::launch_glu_bwd(a, dtype == MOE_DTYPE_F16, (hipStream_t)stream);
}

size_t moe_mlp_keep_bytes(const moe_mlp_t* m, int T, int k) {
    return m && T >= 0 && k > 0 ? MlpLayout(*m, (int64_t)T * k).keep : 0;
}
size_t moe_mlp_fwd_workspace_bytes(const moe_mlp_t* m, int T, int k) {
    return m && T >= 0 && k > 0 ? MlpLayout(*m, (int64_t)T * k).fwd : 0;
}
size_t moe_mlp_bwd_workspace_bytes(const moe_mlp_t* m, int T, int k) {
    return m && T >= 0 && k > 0 ? MlpLayout(*m, (int64_t)T * k).bwd : 0;
}

int moe_mlp_fwd(const moe_mlp_t* m, const void* x, const int32_t* idx, const float* wts, int T, int k, const void* residual,
                void* y, int y_dtype, void* keep, void* gu, void* codes, void* scales, void* workspace, size_t workspace_bytes,
                void* stream) {
    int rc = check_mlp(m, T, k);
    if (rc) return rc;
    if (y_dtype != m->dtype && y_dtype != MOE_DTYPE_F32) return MOE_ERR_DTYPE;
    if (T == 0) return MOE_OK;
    if (!x || !idx || !wts || !y || !keep || !codes != !scales) return MOE_ERR_ARG;
    if (misaligned(x) || misaligned(residual) || misaligned(y) || misaligned(keep) || misaligned(gu) || misaligned(codes) ||
        misaligned(workspace))
        return MOE_ERR_ALIGN;
    const int64_t n = (int64_t)T * k;
    const MlpLayout L(*m, n);
    if (!workspace || workspace_bytes < L.fwd) return MOE_ERR_WORKSPACE;
    char *kp = (char*)keep, *ws = (char*)workspace;
    const hipStream_t st = (hipStream_t)stream;
    const bool f16 = m->dtype == MOE_DTYPE_F16;
    int32_t *offsets = (int32_t*)(kp + L.offsets), *sorted = (int32_t*)(kp + L.sorted), *rows = (int32_t*)(kp + L.rows),
            *pos = (int32_t*)(kp + L.pos);
    const moe::GroupBufs gb{(int32_t*)(ws + L.counts), offsets, sorted, (int32_t*)(ws + L.active), (int32_t*)(ws + L.meta), nullptr,
                            nullptr};
    rc = moe::launch_group(idx, (int)n, m->E, gb, moe::GroupScratch{(int32_t*)(ws + L.chunks), (size_t)256 * m->E}, st);
    if (rc) return rc;
    rc = moe::launch_slots(idx, sorted, offsets, (int)n, k, m->E, rows, pos, st);
    if (rc) return rc;
    moe::MmArgs a{};
    a.a = x;
    a.b = m->w_gate_up;
    a.offsets = offsets;
    a.arows = rows;
    a.y = ws + L.h;
    a.M = (int)n;
    a.a_n = T;
    a.lda = m->d;
    a.ldb = m->d;
    a.E = m->E;
    a.J = m->F;
    a.R = m->d;
    a.f16 = f16;
    a.ydt = m->dtype;
    a.kind = moe::EPI_GLU;
    a.epi.act = m->act;
    a.epi.gu = gu;
    a.epi.codes = (uint8_t*)codes;
    a.epi.scales = (uint8_t*)scales;
    rc = moe::launch_mm_fwd(a, st);
    if (rc) return rc;
    a.a = ws + L.h;
    a.b = m->w_down;
    a.arows = nullptr;
    a.y = ws + L.ys;
    a.a_n = (int)n;
    a.lda = m->F;
    a.ldb = m->F;
    a.J = m->d;
    a.R = m->F;
    a.kind = moe::EPI_PLAIN;
    a.epi = moe::MmEpi{};
    a.ydt = MOE_DTYPE_F32;   // the slots' rows: rounded before their sum, they took y's error from 2.4e-3 to 2.9e-3
    rc = moe::launch_mm_fwd(a, st);
    if (rc) return rc;
    return moe::launch_slot_sum((const float*)(ws + L.ys), pos, wts, residual, n, T, k, m->d, f16, y, y_dtype, st);
}

int moe_mlp_bwd(const moe_mlp_t* m, const void* x, const float* wts, const void* dy, int T, int k, const void* keep, const void* gu,
                const void* codes, const void* scales, void* dx, float* dwts, void* dw_gate_up, void* dw_down, void* workspace,
                size_t workspace_bytes, void* stream) {
    int rc = check_mlp(m, T, k);
    if (rc) return rc;
    if (!keep || (T > 0 && (!x || !wts || !dy || (codes ? !scales || gu : !gu)))) return MOE_ERR_ARG;
    if (misaligned(x) || misaligned(dy) || misaligned(keep) || misaligned(gu) || misaligned(codes) || misaligned(dx) ||
        misaligned(dw_gate_up) || misaligned(dw_down) || misaligned(workspace))
        return MOE_ERR_ALIGN;
    if (T == 0) return MOE_ERR_ARG;   // nothing was kept: the caller's gradients are zeros
    const int64_t n = (int64_t)T * k;
    const MlpLayout L(*m, n);
    if (!workspace || workspace_bytes < L.bwd) return MOE_ERR_WORKSPACE;
    const char* kp = (const char*)keep;
    char* ws = (char*)workspace;
    const hipStream_t st = (hipStream_t)stream;
    const bool f16 = m->dtype == MOE_DTYPE_F16;
    const int32_t *offsets = (const int32_t*)(kp + L.offsets), *sorted = (const int32_t*)(kp + L.sorted),
                  *rows = (const int32_t*)(kp + L.rows), *pos = (const int32_t*)(kp + L.pos);
    // dh[p] = dy[token] . w_down, unweighted and in fp32: the weights' gradient is its product with h, and a router's
    // gradient is a difference of such sums
    moe::MmArgs a{};
    a.a = dy;
    a.b = m->w_down;
    a.offsets = offsets;
    a.arows = rows;
    a.y = ws + L.dh;
    a.M = (int)n;
    a.a_n = (int)T;
    a.lda = m->d;
    a.ldb = m->F;
    a.E = m->E;
    a.J = m->F;
    a.R = m->d;
    a.f16 = f16;
    a.ydt = MOE_DTYPE_F32;
    rc = moe::launch_mm_dx(a, st);
    if (rc) return rc;
    const moe::GluBwd b{(const uint8_t*)codes, (const uint8_t*)scales, (const uint16_t*)gu, 2 * (int64_t)m->F, ws + L.dh, 1, wts,
                        sorted, offsets + m->E, n, m->F, m->act, (uint16_t*)(ws + L.dgu),
                        dw_down ? (uint16_t*)(ws + L.hw) : nullptr, dwts};
    rc = moe::launch_glu_bwd(b, f16, st);
    if (rc) return rc;
    // the slots' rows of dx in fp32: rounded to 16 bits before their sum, they took dx's error from 2.4e-3 to 2.9e-3
    if (dx) {
        a.a = ws + L.dgu;
        a.b = m->w_gate_up;
        a.arows = nullptr;
        a.y = ws + L.dxs;
        a.a_n = (int)n;
        a.lda = 2 * m->F;
        a.ldb = m->d;
        a.J = m->d;
        a.R = 2 * m->F;
        rc = moe::launch_mm_dx(a, st);
        if (rc) return rc;
        rc = moe::launch_slot_sum((const float*)(ws + L.dxs), pos, nullptr, nullptr, n, T, k, m->d, f16, dx, m->dtype, st);
        if (rc) return rc;
    }
    moe::MmArgs w{};
    w.offsets = offsets;
    w.M = (int)n;
    w.E = m->E;
    w.f16 = f16;
    w.ydt = m->dtype;
    if (dw_gate_up) {
        w.a = ws + L.dgu;
        w.b = x;
        w.brows = rows;
        w.y = dw_gate_up;
        w.a_n = (int)n;
        w.b_n = T;
        w.lda = 2 * m->F;
        w.ldb = m->d;
        w.I = 2 * m->F;
        w.J = m->d;
        rc = moe::launch_mm_dw(w, st);
        if (rc) return rc;
    }
    if (dw_down) {
        w.a = dy;
        w.b = ws + L.hw;
        w.arows = rows;
        w.brows = nullptr;
        w.y = dw_down;
        w.a_n = T;
        w.b_n = (int)n;
        w.lda = m->d;
        w.ldb = m->F;
        w.I = m->d;
        w.J = m->F;
        rc = moe::launch_mm_dw(w, st);
        if (rc) return rc;
    }
    return MOE_OK;
}

}  // extern "C"
