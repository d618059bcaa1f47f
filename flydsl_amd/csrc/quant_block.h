// Arguments of the quantiser with one scale for every 128 columns of a row.  Plain data, passed by value.
#pragma once
#include "psg_common.h"

struct QuantBlockParams {
    const void* x;           // [rows, dim], or [rows, 2 dim] with gated
    uint8_t* q;              // [rows, dim] e4m3, dense
    float* scale;            // [ceil(dim / 128), rows]
    int64_t x_stride;        // elements from a row of x to the next
    int64_t scale_stride;    // floats from a block's scales to the next block's
    int64_t rows;
    int dim;
    int gated;
};
hipError_t psg_launch_quant_block(QuantBlockParams p, int x_dtype, hipStream_t stream);
