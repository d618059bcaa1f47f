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
    int ks;                // set by the launcher: K slices of a workgroup (a power of two)
    int groups;            // set by the launcher: column groups of the launch, unit_q units of 8 columns each,
    int unit_q, unit_r;    // the first unit_r of them one more
};
