// Routing by scores and groups: the k experts of each token, their weights, and the gradient of the logits.
//   s = sigmoid(l) or softmax(l);  an expert ranks by c = s + bias, without a bias by l itself (s grows with l);
//   a group's value is the largest c in it or the sum of its two largest (without a bias of s); the best groups stay, in them the
//   k largest c, of equals the lowest id; w = scale s, divided by the chosen ones' sum with norm.
// Two experts' scores can differ by less than fp32 keeps, and which one is chosen is the result, so scores and their sums are
// fp64; ranking works on 64-bit integers that order as the numbers do, 32-bit ones without a bias.
// One wave per token, expert 64 j + lane in a lane's slot j. Bound by the latency of its chain, not by bytes or operations: the logits,
// for a softmax its maximum and total, the groups' values, then k rounds of a maximum over the wave and one over its lanes' slots
// (traced: 256 experts in 8 groups, k 8: 6.5 us for one token, 12 for 4096, whose logits are read in 1, in a captured graph 7.0 and
// 11.5; 8191 tokens of 64 experts, k 6, softmax without norm: forward 11 us, backward 8). With more tokens than the CUs hold waves the
// fp64 exponentials add up: they are taken only where they rank or scale.
#include "moe_common.h"
#include "moe_scored.h"

namespace moe {

template <typename LT>
__device__ __forceinline__ float as_f32(LT v);
template <>
__device__ __forceinline__ float as_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ float as_f32<uint16_t>(uint16_t v) { return bf16_to_f32(v); }
template <>
__device__ __forceinline__ float as_f32<_Float16>(_Float16 v) { return (float)v; }

// A logit as the formulas read it: NaN counts as -inf.
__device__ __forceinline__ float clean(float l) { return l == l ? l : -INFINITY; }
__device__ __forceinline__ double sigmoid64(float l) { return 1.0 / (1.0 + exp(-(double)l)); }
// e^(l - m), m the largest; +inf: every such logit has the same share
__device__ __forceinline__ double share64(float l, float m) { return l == m ? (l == -INFINITY ? 0.0 : 1.0) : exp((double)l - (double)m); }

__device__ __forceinline__ uint64_t key_of(double v) {   // orders as v does; -0 as +0
    const uint64_t b = (uint64_t)__double_as_longlong(v + 0.0);
    return b >> 63 ? ~b : b | 1ull << 63;
}
__device__ __forceinline__ uint32_t key_of(float v) {
    const uint32_t b = __float_as_uint(v + 0.f);
    return b >> 31 ? ~b : b | 1u << 31;
}
// Sums and maxima over lanes by DPP moves: a move through LDS (ds_bpermute) takes about ten times as long, and a token is a chain
// of them (256 experts, k 8, one token: 10.0 us with those, 5.1 so; 4096 tokens 17.6 and 9.8: both measured together,
// on an earlier form of the kernel than the figures above).
template <int CTRL, int ROWS = 0xF>
__device__ __forceinline__ double moved64(double v) {   // lanes without a source: 0
    const u32x2 w = __builtin_bit_cast(u32x2, v);
    const u32x2 o = {(uint32_t)__builtin_amdgcn_update_dpp(0, (int)w[0], CTRL, ROWS, 0xF, false),
                     (uint32_t)__builtin_amdgcn_update_dpp(0, (int)w[1], CTRL, ROWS, 0xF, false)};
    return __builtin_bit_cast(double, o);
}
__device__ __forceinline__ double lane64(double v, int lane) {   // of one lane, wave-uniform
    const u32x2 w = __builtin_bit_cast(u32x2, v);
    const u32x2 o = {(uint32_t)__builtin_amdgcn_readlane((int)w[0], lane), (uint32_t)__builtin_amdgcn_readlane((int)w[1], lane)};
    return __builtin_bit_cast(double, o);
}
__device__ __forceinline__ double wave_sum64(double v) {
    v += moved64<0xB1>(v);
    v += moved64<0x4E>(v);
    v += moved64<0x141>(v);
    v += moved64<0x140>(v);
    v += moved64<0x142, 0xA>(v);
    v += moved64<0x143, 0xC>(v);
    return lane64(v, 63);
}

// The value by which an expert ranks, or -inf (behind all others, weight 0) where the logit or its bias says so.
__device__ __forceinline__ double ranked(float l, double s, const float* bias, int e) {
    if (l == -INFINITY) return -INFINITY;
    if (!bias) return (double)l;
    const double c = s + (double)bias[e];
    return c == c ? c : -INFINITY;
}

// The larger two of a lane's pair and another's.
__device__ __forceinline__ void join2(double& top, double& next, double t2, double n2) {
    next = fmax(fmax(next, n2), fmin(top, t2));
    top = fmax(top, t2);
}
// The two largest over aligned groups of `share` lanes (a power of two), in every lane.
__device__ __forceinline__ void largest2(double& top, double& next, int share) {
    if (share > 1) join2(top, next, moved64<0xB1>(top), moved64<0xB1>(next));
    if (share > 2) join2(top, next, moved64<0x4E>(top), moved64<0x4E>(next));
    if (share > 4) join2(top, next, moved64<0x141>(top), moved64<0x141>(next));
    if (share > 8) join2(top, next, moved64<0x140>(top), moved64<0x140>(next));
    if (share > 16) join2(top, next, __shfl_xor(top, 16), __shfl_xor(next, 16));
}

// WIDE: with a bias, 64-bit ranks.
constexpr int SC_WAVES = 4;   // tokens of a workgroup
template <typename LT, int JM, bool WIDE>
__global__ void __launch_bounds__(64 * SC_WAVES) k_topk_scored(const LT* logits, const ScoredArgs a, int32_t* idx, float* wts) {
    __shared__ double val[SC_WAVES][JM * 64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int t = blockIdx.x * SC_WAVES + wave, E = a.E;
    if (t >= a.T) return;
    const LT* row = logits + (int64_t)t * E;
    float l[JM];
#pragma unroll
    for (int j = 0; j < JM; ++j) l[j] = 64 * j + lane < E ? clean(as_f32<LT>(row[64 * j + lane])) : -INFINITY;
    const bool soft = a.score == MOE_SCORE_SOFTMAX, sums = a.groups > 1 && a.group_score == MOE_GROUP_TOP2;
    // scores, where they rank or scale: all of them with a bias or sums of two; for a softmax its total without norm too
    float m = -INFINITY;
    double total = 1.0;
    if (soft) {
#pragma unroll
        for (int j = 0; j < JM; ++j) m = fmaxf(m, l[j]);
        m = wave_max_dpp(m);
        if (WIDE || sums || !a.norm) {
            double p = 0.0;
#pragma unroll
            for (int j = 0; j < JM; ++j) p += share64(l[j], m);
            total = wave_sum64(p);
            total = total > 0.0 ? total : 1.0;
        }
    }
    // keys: the high words, and (WIDE) the low ones; 0: not to be chosen (any more)
    uint32_t hi[JM], lo[WIDE ? JM : 1];
#pragma unroll
    for (int j = 0; j < JM; ++j) {
        const int e = 64 * j + lane;
        double s = 0.0;
        if (WIDE || sums) s = soft ? share64(l[j], m) / total : sigmoid64(l[j]);
        if constexpr (WIDE) {
            const double c = e < E ? ranked(l[j], s, a.bias, e) : -INFINITY;
            const uint64_t k = key_of(c);
            hi[j] = (uint32_t)(k >> 32);
            lo[j] = (uint32_t)k;
            if (a.groups > 1) val[wave][e] = c;
        } else {
            hi[j] = key_of(l[j]);
            if (a.groups > 1) val[wave][e] = sums && l[j] != -INFINITY ? s : (double)l[j];
        }
        if (e >= E) hi[j] = 0;
    }
    if (a.groups > 1) {
        const int size = E / a.groups;
        __builtin_amdgcn_wave_barrier();
        int share = 64;   // lanes of a group
        while (share * a.groups > 64) share >>= 1;
        const int g = lane / share;
        double top = -INFINITY, next = -INFINITY;
        if (g < a.groups)
            for (int i = lane & (share - 1); i < size; i += share) {
                const double v = val[wave][g * size + i];
                next = fmax(next, fmin(top, v));
                top = fmax(top, v);
            }
        largest2(top, next, share);
        double v = sums ? top + next : top;
        v = v == v ? v : -INFINITY;
        int before = 0;
        for (int h = 0; h < a.groups; ++h) {
            const double o = lane64(v, h * share);
            before += o > v || (o == v && h < g);
        }
        const uint64_t stay = __ballot(g < a.groups && before < a.top_groups);   // all of a group's lanes
#pragma unroll
        for (int j = 0; j < JM; ++j) {
            const int e = 64 * j + lane;
            if (e < E && !(stay >> (e / size * share) & 1)) hi[j] = 0;
        }
    }
    const uint64_t none64 = key_of(-(double)INFINITY);
    const uint32_t none = WIDE ? (uint32_t)(none64 >> 32) : key_of(-INFINITY), none_lo = (uint32_t)none64;
    int mine = 0;        // lane r holds round r's expert
    float ml = -INFINITY;
    for (int r = 0; r < a.k; ++r) {
        uint32_t bh = hi[0], bl = WIDE ? lo[0] : 0;
        int bj = 0;
#pragma unroll
        for (int j = 1; j < JM; ++j) {
            const bool more = hi[j] > bh || (WIDE && hi[j] == bh && lo[j] > bl);
            bh = more ? hi[j] : bh;
            if constexpr (WIDE) bl = more ? lo[j] : bl;
            bj = more ? j : bj;
        }
        const uint32_t mh = wave_umax_dpp(bh);
        uint64_t hit = __ballot(bh == mh);
        uint32_t id;
        if constexpr (WIDE) {
            if (hit & (hit - 1)) {
                const uint32_t low = wave_umax_dpp(bh == mh ? bl : 0);   // by all lanes
                hit &= __ballot(bl == low);
            }
        }
        if (hit & (hit - 1)) id = wave_min_dpp(hit >> lane & 1 ? (uint32_t)(64 * bj + lane) : 0xffffffffu);
        else id = 64 * __builtin_amdgcn_readlane(bj, __builtin_ctzll(hit)) + __builtin_ctzll(hit);
        const uint32_t ml_lo = WIDE ? (uint32_t)__builtin_amdgcn_readlane((int)bl, id & 63) : 0;
        const bool out = mh == none && (!WIDE || ml_lo == none_lo);
        float lv = -INFINITY;
#pragma unroll
        for (int j = 0; j < JM; ++j)
            if (j == (int)(id >> 6)) {   // wave-uniform
                lv = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(l[j]), id & 63));
                if ((int)(id & 63) == lane) {
                    hi[j] = 0;
                    if constexpr (WIDE) lo[j] = 0;
                }
            }
        if (lane == r) {
            mine = id;
            ml = out ? -INFINITY : lv;
        }
    }
    double s = 0.0;
    if (ml != -INFINITY) s = !soft ? sigmoid64(ml) : a.norm ? 1.0 : share64(ml, m) / total;
    if (a.norm) {
        if (soft) s = share64(ml, wave_max_dpp(ml));
        const double sum = wave_sum64(s);
        s = sum > 0.0 ? s / sum : 0.0;
    }
    if (lane < a.k) {
        idx[(int64_t)t * a.k + lane] = mine;
        wts[(int64_t)t * a.k + lane] = (float)(s * (double)a.scale);
    }
}

// dlogits from the weights' gradients, at the chosen experts:
//   norm: ds_j = scale / S (dw_j - sum_i dw_i s_i / S), else scale dw_j;
//   sigmoid: dl_e = ds_e s_e (1 - s_e);   softmax: dl_e = p_e (ds_e - sum_j ds_j p_j), which with norm is 0 elsewhere, since
//   the weights are the softmax of the chosen logits alone. Experts that were chosen at -inf have weight 0 and no gradient.
template <typename LT, int JM>
__global__ void __launch_bounds__(64 * SC_WAVES) k_topk_scored_bwd(const LT* logits, const ScoredArgs a, const int32_t* idx,
                                                                   const float* dwts, LT* dlogits) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int t = blockIdx.x * SC_WAVES + wave, E = a.E;
    if (t >= a.T) return;
    const LT* row = logits + (int64_t)t * E;
    const bool soft = a.score == MOE_SCORE_SOFTMAX, dense = soft && !a.norm;
    int id = -1;
    float l = -INFINITY;
    double dw = 0.0;
    if (lane < a.k) {
        id = idx[(int64_t)t * a.k + lane];
        if ((uint32_t)id < (uint32_t)E) {   // (no expert: no gradient)
            l = clean(as_f32<LT>(row[id]));
            if (a.bias && ranked(l, 0.0, a.bias, id) == -INFINITY) l = -INFINITY;
        }
        if (l != -INFINITY) dw = (double)dwts[(int64_t)t * a.k + lane] * (double)a.scale;
    }
    float v[JM], m = -INFINITY;
    double total = 1.0;
    if (dense) {
        double p = 0.0;
#pragma unroll
        for (int j = 0; j < JM; ++j) {
            v[j] = 64 * j + lane < E ? clean(as_f32<LT>(row[64 * j + lane])) : -INFINITY;
            m = fmaxf(m, v[j]);
        }
        m = wave_max_dpp(m);
#pragma unroll
        for (int j = 0; j < JM; ++j) p += share64(v[j], m);
        total = wave_sum64(p);
        total = total > 0.0 ? total : 1.0;
    } else if (soft) {
        m = wave_max_dpp(l);
    }
    double s = 0.0, mean = 0.0;   // this lane's score (with norm: its share), and sum_j dw_j s_j
    if (l != -INFINITY) s = soft ? share64(l, m) : sigmoid64(l);
    double g;
    if (a.norm) {
        const double sum = wave_sum64(s), inv = sum > 0.0 ? 1.0 / sum : 0.0;
        mean = wave_sum64(dw * s) * inv;
        g = soft ? s * inv * (dw - mean) : s * inv * (dw - mean) * (1.0 - s);
    } else if (soft) {
        s /= total;
        mean = wave_sum64(dw * s);
        g = s * dw;
    } else {
        g = dw * s * (1.0 - s);
    }
    double out[JM];   // what a softmax's total does to all of them, and the chosen ones' own part
#pragma unroll
    for (int j = 0; j < JM; ++j) out[j] = dense ? -share64(v[j], m) / total * mean : 0.0;
    for (int r = 0; r < a.k; ++r) {
        const int i = __builtin_amdgcn_readlane(id, r);
        const double o = lane64(g, r);
#pragma unroll
        for (int j = 0; j < JM; ++j) out[j] += i == 64 * j + lane ? o : 0.0;
    }
#pragma unroll
    for (int j = 0; j < JM; ++j) {
        const int e = 64 * j + lane;
        if (e >= E) break;
        if constexpr (sizeof(LT) == 4) dlogits[(int64_t)t * E + e] = (float)out[j];
        else if constexpr (std::is_same<LT, _Float16>::value) dlogits[(int64_t)t * E + e] = (_Float16)(float)out[j];
        else dlogits[(int64_t)t * E + e] = f32_to_bf16((float)out[j]);
    }
}

template <typename LT, typename F>
static int by_size(const ScoredArgs& a, F run) {
    if (a.T == 0) return MOE_OK;
    if (a.E <= 64) run(std::integral_constant<int, 1>{});
    else if (a.E <= 128) run(std::integral_constant<int, 2>{});
    else if (a.E <= 256) run(std::integral_constant<int, 4>{});
    else if (a.E <= 512) run(std::integral_constant<int, 8>{});
    else run(std::integral_constant<int, 16>{});
    return hipGetLastError() == hipSuccess ? MOE_OK : MOE_ERR_LAUNCH;
}
template <typename LT>
static int forward(const void* logits, const ScoredArgs& a, int32_t* idx, float* wts, hipStream_t st) {
    return by_size<LT>(a, [&](auto jm) {
        const unsigned grid = (a.T + SC_WAVES - 1) / SC_WAVES;
        if (a.bias) k_topk_scored<LT, decltype(jm)::value, true><<<grid, 64 * SC_WAVES, 0, st>>>((const LT*)logits, a, idx, wts);
        else k_topk_scored<LT, decltype(jm)::value, false><<<grid, 64 * SC_WAVES, 0, st>>>((const LT*)logits, a, idx, wts);
    });
}
template <typename LT>
static int backward(const void* logits, const ScoredArgs& a, const int32_t* idx, const float* dwts, void* dl, hipStream_t st) {
    return by_size<LT>(a, [&](auto jm) {
        k_topk_scored_bwd<LT, decltype(jm)::value><<<(a.T + SC_WAVES - 1) / SC_WAVES, 64 * SC_WAVES, 0, st>>>((const LT*)logits, a, idx,
                                                                                                   dwts, (LT*)dl);
    });
}

int launch_topk_scored(const void* logits, int dtype, const ScoredArgs& a, int32_t* idx, float* wts, hipStream_t st) {
    if (dtype == MOE_DTYPE_F32) return forward<float>(logits, a, idx, wts, st);
    if (dtype == MOE_DTYPE_F16) return forward<_Float16>(logits, a, idx, wts, st);
    return forward<uint16_t>(logits, a, idx, wts, st);
}
int launch_topk_scored_bwd(const void* logits, int dtype, const ScoredArgs& a, const int32_t* idx, const float* dwts, void* dlogits,
                           hipStream_t st) {
    if (dtype == MOE_DTYPE_F32) return backward<float>(logits, a, idx, dwts, dlogits, st);
    if (dtype == MOE_DTYPE_F16) return backward<_Float16>(logits, a, idx, dwts, dlogits, st);
    return backward<uint16_t>(logits, a, idx, dwts, dlogits, st);
}

}  // namespace moe

namespace {
int check(const moe_scored_t* r, int T) {
    if (!r || T < 0 || T > 0x7fffff00 || r->E < 1 || r->E > 1024 || r->k < 1 || r->k > 32) return MOE_ERR_ARG;
    if (r->score != MOE_SCORE_SOFTMAX && r->score != MOE_SCORE_SIGMOID) return MOE_ERR_ARG;
    if (r->group_score != MOE_GROUP_MAX && r->group_score != MOE_GROUP_TOP2) return MOE_ERR_ARG;
    if (r->groups < 1 || r->groups > 64 || r->E % r->groups || r->top_groups < 1 || r->top_groups > r->groups) return MOE_ERR_ARG;
    const int size = r->E / r->groups;
    if (r->k > r->top_groups * size || (r->groups > 1 && r->group_score == MOE_GROUP_TOP2 && size < 2)) return MOE_ERR_ARG;
    return MOE_OK;
}
moe::ScoredArgs args_of(const moe_scored_t* r, int T) {
    return {T, r->E, r->k, r->score, r->groups, r->top_groups, r->group_score, r->norm != 0, r->scale, r->bias};
}
bool float_type(int dtype) { return dtype == MOE_DTYPE_BF16 || dtype == MOE_DTYPE_F16 || dtype == MOE_DTYPE_F32; }
}  // namespace

extern "C" {

int moe_topk_scored(const moe_scored_t* r, const void* logits, int dtype, int T, int32_t* idx, float* wts, void* stream) {
    const int rc = check(r, T);
    if (rc) return rc;
    if (!float_type(dtype)) return MOE_ERR_DTYPE;
    if (T == 0) return MOE_OK;
    if (!logits || !idx || !wts) return MOE_ERR_ARG;
    return moe::launch_topk_scored(logits, dtype, args_of(r, T), idx, wts, (hipStream_t)stream);
}

int moe_topk_scored_bwd(const moe_scored_t* r, const void* logits, int dtype, int T, const int32_t* idx, const float* dwts,
                        void* dlogits, void* stream) {
    const int rc = check(r, T);
    if (rc) return rc;
    if (!float_type(dtype)) return MOE_ERR_DTYPE;
    if (T == 0) return MOE_OK;
    if (!logits || !idx || !dwts || !dlogits) return MOE_ERR_ARG;
    return moe::launch_topk_scored_bwd(logits, dtype, args_of(r, T), idx, dwts, dlogits, (hipStream_t)stream);
}

int moe_router_scored(const moe_scored_t* r, const void* x, const void* wr, const float* wr_bias, int T, int d, float* logits,
                      int32_t* idx, float* wts, void* stream) {
    int rc = check(r, T);
    if (rc) return rc;
    if (d < 8 || d % 8) return MOE_ERR_ARG;
    if (T == 0) return MOE_OK;
    if (!x || !wr || !logits || !idx || !wts) return MOE_ERR_ARG;
    if (((uintptr_t)x | (uintptr_t)wr) & 15) return MOE_ERR_ALIGN;
    rc = moe::launch_router_logits((const uint16_t*)x, (const uint16_t*)wr, wr_bias, T, d, r->E, logits, (hipStream_t)stream);
    if (rc) return rc;
    return moe::launch_topk_scored(logits, MOE_DTYPE_F32, args_of(r, T), idx, wts, (hipStream_t)stream);
}

}  // extern "C"
