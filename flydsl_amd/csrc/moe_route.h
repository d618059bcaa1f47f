// Arguments of the routing with a bias and groups of experts.  Plain data, passed by value.
#pragma once
#include "psg_common.h"

struct RouteParams {
    const void* gating;  // [tokens, experts] fp32 / bf16 / fp16
    const float* bias;   // [experts] or nullptr
    float* weights;      // [tokens, topk]
    int32_t* indices;    // [tokens, topk]
    int tokens, experts, topk;
    int softmax;         // else sigmoid
    int groups, topk_groups;
    int top2;            // a run of experts is worth its two best, else its best
    int renorm;
    float scale;
    int lanes, lanes_group;  // set by the launcher: lanes of a token and of a run of experts
    int vec;                 // set by the launcher: a lane's logits and bias are whole vectors
};
hipError_t psg_launch_moe_route(RouteParams p, int dtype, hipStream_t stream);
