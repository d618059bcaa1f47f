// Arguments of the products with 4-bit weights and group scales.  Plain data, passed by value.
#pragma once
#include "psg_common.h"

struct W4Params {
    void* c;               // [M, N]
    const void* a;         // [M, K]
    const uint8_t* w;      // [N/16][ceil(K/128)][4][16][16 bytes]
    const uint16_t* scales;  // [N/16][K/group][16]
    const uint8_t* zeros;  // [N/16][K/group][8], or nullptr
    const uint16_t* bias;  // [N]
    int M, N, K;
    int out, epi;          // OUT_*, EPI_*
    int passes, per;       // set by the launcher: passes over the columns, 128-element steps of a wavefront in each
    int unit_q, unit_r;    // set by the launcher: a workgroup has unit_q units of 8 columns, the first unit_r of them one more
};
