// Arguments of the norm with quantised rows.  Plain data, passed by value.
#pragma once
#include "psg_common.h"

enum { NORM_INT8 = 0, NORM_FP8 = 1, NORM_NONE = 2 };
struct NormParams {
    const void* x;         // [rows, dim]
    const void* residual;  // [rows, dim] in the type of x, or nullptr
    const void* weight;    // [dim] in the type of x, or fp32
    void* h;               // x + residual, in the type of x (with a residual only; may be `residual` or `x`)
    void* normed;          // normalised rows in the type of x, or nullptr
    uint8_t* q;            // [rows, dim], dense
    float* scale;          // [rows]
    int64_t x_stride, r_stride, h_stride, n_stride;  // elements from a row to the next
    int64_t rows;
    int dim;
    int w_f32;             // the weight is fp32 (always with fp32 x)
    int out;               // NORM_*
    float eps;
};
