// Launchers of the elementwise passes of the 16-bit expert layer (moe_act8.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "moe_mi355x.h"

namespace moe {

struct GluBwd {
    const uint8_t* codes;    // [M, 2 F], scales [M, 2 F / 32]; or null:
    const uint8_t* scales;
    const uint16_t* gu;      // [M, 2 F] of row stride ldg
    int64_t ldg;
    const void* dh;          // [M, F] 16-bit, or fp32 with dh32
    int dh32;
    const float* wts;        // or null: 1
    const int32_t* idx;      // place of row r in wts and dwts, or null: r
    const int32_t* count;    // rows that are in use, or null: M
    int64_t M;
    int F, act;
    uint16_t* dgu;           // [M, 2 F]
    uint16_t* hw;            // [M, F] or null
    float* dwts;             // or null
};

int launch_glu_fwd(const void* gu, int64_t ldg, int64_t M, int F, int act, bool f16, void* h, uint8_t* codes, uint8_t* scales,
                   hipStream_t st);
int launch_glu_bwd(const GluBwd& a, bool f16, hipStream_t st);
int launch_pack8(const void* x, int64_t ld, int64_t M, int64_t C, bool f16, uint8_t* codes, uint8_t* scales, hipStream_t st);
int launch_unpack8(const uint8_t* codes, const uint8_t* scales, int64_t M, int64_t C, int dtype, void* out, hipStream_t st);
int launch_lin_act_bwd(const void* dy, int64_t ldy, const void* z, const uint8_t* codes, const uint8_t* scales, int64_t M,
                       int64_t N, int act, bool f16, void* dz, hipStream_t st);
int launch_slots(const int32_t* idx, const int32_t* sorted, const int32_t* offsets, int n, int k, int E, int32_t* rows,
                 int32_t* pos, hipStream_t st);
int launch_slot_sum(const float* ys, const int32_t* pos, const float* wts, const void* residual, int64_t M, int64_t T, int k,
                    int d, bool f16, void* y, int ydt, hipStream_t st);

}  // namespace moe
