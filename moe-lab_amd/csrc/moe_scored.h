// Launchers of the routing by scores and groups (moe_scored.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "moe_internal.h"

namespace moe {

struct ScoredArgs {
    int T, E, k;
    int score;                // MOE_SCORE_*
    int groups, top_groups;   // E % groups == 0
    int group_score;          // MOE_GROUP_*
    int norm;
    float scale;
    const float* bias;        // [E] or null
};
int launch_topk_scored(const void* logits, int dtype, const ScoredArgs& a, int32_t* idx, float* wts, hipStream_t st);
int launch_topk_scored_bwd(const void* logits, int dtype, const ScoredArgs& a, const int32_t* idx, const float* dwts, void* dlogits,
                           hipStream_t st);

}  // namespace moe
