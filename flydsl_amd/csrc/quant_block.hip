// Rows to e4m3 with one fp32 scale for every 128 columns, what the block-scaled products read (gfx950).
//
//   y = x                        or, gated, y = (g sigmoid(g)) u with g = x[:, :dim], u = x[:, dim:], in fp32
//   s[b, r] = max|y| / 448       over the columns [128 b, 128 b + 128) of row r; 1 where that is 0
//   q = y / s                    rounded once, to nearest even; NaN -> 0, +-Inf -> +-448 in front of the maximum, as k_quant_pertoken has it
//
// A block belongs to 16 lanes, eight columns each: its maximum is four exchanges inside a row of lanes (DPP), no LDS and no barrier.  A wavefront takes 512 columns of one row, which it
// reads as one kilobyte; the other wavefronts hide its wait (four rows a wavefront, all loads ahead, were 2 to 30 % slower from 256 x 4096 to 8192 x 4096).
// The scales lie block by block, so that a tile of a product finds those of its rows together: its lanes fetch a block's scales of 64 rows as 256 bytes in a row.
// Bound: HBM, 8192 x 8192 of bf16 in 39.8 us (5.05 TB/s, a copy's rate; fp32 57.6 us, 5.8 TB/s), gated 68.0 us (4.94 TB/s; 96 where most groups of eight have a g beyond 83 and take the form that every g needs, the instructions');
// of few rows the launch, 256 x 4096 in 3.1 us.
#include "psg_common.h"
#include "quant_rows.h"
#include "quant_block.h"

namespace {

// v of lane ^ 1, 2, and of the mirrored half row and row: the maximum over 16 lanes
__device__ __forceinline__ uint32_t max16(uint32_t v) {
    auto of = [](uint32_t a, uint32_t b) { return a > b ? a : b; };
    v = of(v, (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, 0xB1, 0xF, 0xF, false));
    v = of(v, (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, 0x4E, 0xF, 0xF, false));
    v = of(v, (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, 0x141, 0xF, 0xF, false));
    return of(v, (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, 0x140, 0xF, 0xF, false));
}

// g sigmoid(g) for |g| <= 83 (and NaN): exp(-g) and its reciprocal are normal numbers.  The product of g with log2(e) is taken to twice the bits: its rounding alone would be |g| units of the result.
__device__ __forceinline__ float silu_near(float g) {
    constexpr float L = 1.44269502162933349609375f, L2 = 1.92596298909109e-8f, LN2 = 0.693147180559945f;  // L + L2 = log2(e)
    const float hi = g * L, lo = __builtin_fmaf(g, L2, __builtin_fmaf(g, L, -hi));
    float z = __builtin_amdgcn_exp2f(-hi);
    z = __builtin_fmaf(-lo * LN2, z, z);
    const float d = 1.0f + z;
    float r = __builtin_amdgcn_rcpf(d);
    r = __builtin_fmaf(__builtin_fmaf(-d, r, 1.0f), r, r);
    return g * r;
}

// g sigmoid(g) u for every g, off by a few units in the last place: with z = exp(-|g|), sigmoid is 1 / (1 + z) or z / (1 + z).  Below -83 sigmoid is z itself, from -87 on below the normal range, where the
// exponential instruction has no results and fp32 no precision; but u can be 2^127 and the product an ordinary number.  There z is kept times 2^160 until u has multiplied it, half of that taken off u, half
// off the product: z 2^160 is a normal number down to exp(-198), 2^-286, whose product with every u is nothing; and where u 2^-80 is subnormal the product is.
__device__ __forceinline__ float silu_times(float g, float u) {
    constexpr float L = 1.44269502162933349609375f, L2 = 1.92596298909109e-8f, LN2 = 0.693147180559945f;  // L + L2 = log2(e)
    const float a = fminf(fabsf(g), 300.0f);
    const float hi = a * L, lo = __builtin_fmaf(a, L2, __builtin_fmaf(a, L, -hi));
    const bool far = hi > 120.0f && g < 0.0f;
    float z = __builtin_amdgcn_exp2f((far ? 160.0f : 0.0f) - hi);
    z = __builtin_fmaf(-lo * LN2, z, z);
    const float d = 1.0f + (far ? 0.0f : z), half = far ? 0x1p-80f : 1.0f;
    float r = __builtin_amdgcn_rcpf(d);
    r = __builtin_fmaf(__builtin_fmaf(-d, r, 1.0f), r, r);
    return g * ((g < 0.0f ? z : 1.0f) * r) * (u * half) * half;
}

// WHOLE: rows are whole vectors of eight
template <int XT, bool GATED, bool WHOLE>
__global__ void __launch_bounds__(256) k_quant_block(QuantBlockParams p, int chunks) {
    const int lane = (int)(threadIdx.x & 63), wave = wave_id();
    const int tile = (int)(blockIdx.x / (unsigned)chunks), chunk = (int)blockIdx.x - tile * chunks;
    const int k = chunk * 512 + lane * 8, left = p.dim - k;
    const bool in = left > 0;
    const int64_t row = (int64_t)tile * 4 + wave;
    if (row >= p.rows) return;  // (uniform: a wavefront has one row)
    // lanes past the row read its front: no load stands behind a branch
    const int64_t at = row * p.x_stride + (in ? k : 0);
    Raw8<XT> a = load_row<XT, WHOLE>(p.x, at, in ? left : p.dim, p.dim), b;
    if constexpr (GATED) b = load_row<XT, WHOLE>(p.x, at + p.dim, in ? left : p.dim, p.dim);
    if (!WHOLE && left < 8 && left > 0 && p.dim >= 8) {
        line_up<XT>(a, left);
        if constexpr (GATED) line_up<XT>(b, left);
    }
    float v[8];
    a.values(v);
    if constexpr (GATED) {
        float w[8];
        b.values(w);
        float top = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; e++) top = fmaxf(top, fabsf(v[e]));
        if (top <= 83.0f) {
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] = silu_near(v[e]) * w[e];
        } else {
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] = silu_times(v[e], w[e]);
        }
    }
    if (!in) {
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = 0.0f;
    }
    // magnitudes as bits, which order like them: NaN above Inf above every finite value
    uint32_t mb = 0;
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const uint32_t m = __builtin_bit_cast(uint32_t, v[e]) & 0x7FFFFFFFu;
        mb = m > mb ? m : mb;
    }
    mb = max16(mb);
    const bool special = mb >= 0x7F800000u;  // the block holds an Inf or NaN
    if (special) {
        mb = 0;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            v[e] = clean(v[e], 448.0f);
            const uint32_t m = __builtin_bit_cast(uint32_t, v[e]) & 0x7FFFFFFFu;
            mb = m > mb ? m : mb;
        }
        mb = max16(mb);  // (all 16 lanes of the block are here)
    }
    float s = __builtin_bit_cast(float, mb) / 448.0f;
    if (s == 0.0f) s = 1.0f;
    if (s >= 0x1p-80f && s <= 0x1p100f) {
        const float rs = 1.0f / s;
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = quotient(v[e], s, rs);
    } else {
        // (a scale of a few bits may be below max|y| / 448 by more than a code)
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = fminf(fmaxf(v[e] / s, -448.0f), 448.0f);
    }
    const v2i o = quant_pack8<1>(v);
    if (in) {
        uint8_t* q = p.q + row * p.dim + k;
        if (WHOLE || left >= 8) {
            *reinterpret_cast<v2i_any*>(q) = o;
        } else {
            int w = o[0];
            if (left & 4) *reinterpret_cast<int_any*>(q) = w, q += 4, w = o[1];
            if (left & 2) *reinterpret_cast<half_any*>(q) = (uint16_t)w, q += 2, w >>= 16;
            if (left & 1) *q = (uint8_t)w;
        }
        if ((lane & 15) == 0) p.scale[(int64_t)(chunk * 4 + (lane >> 4)) * p.scale_stride + row] = s;
    }
}

template <int XT, bool GATED, bool WHOLE>
hipError_t launch(QuantBlockParams p, hipStream_t stream) {
    const int chunks = (p.dim + 511) / 512;
    const int64_t most = ((1ll << 23) / chunks > 0 ? (1ll << 23) / chunks : 1) * 4, all = p.rows;  // rows a launch (256 threads each: a grid holds less than 2^32)
    for (int64_t done = 0; done < all; done += most) {
        p.rows = all - done < most ? all - done : most;
        const dim3 grid((unsigned)((p.rows + 3) / 4 * chunks));
        hipLaunchKernelGGL((k_quant_block<XT, GATED, WHOLE>), grid, dim3(256), 0, stream, p, chunks);
        if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
        p.x = static_cast<const uint8_t*>(p.x) + most * p.x_stride * (XT == X_F32 ? 4 : 2);
        p.q += most * p.dim;
        p.scale += most;
    }
    return hipSuccess;
}

template <int XT>
hipError_t launch_x(const QuantBlockParams& p, hipStream_t stream) {
    if (p.dim % 8) return p.gated ? launch<XT, true, false>(p, stream) : launch<XT, false, false>(p, stream);
    return p.gated ? launch<XT, true, true>(p, stream) : launch<XT, false, true>(p, stream);
}

}  // namespace

// x_dtype: 0 fp32, 1 bf16, 2 fp16
hipError_t psg_launch_quant_block(QuantBlockParams p, int x_dtype, hipStream_t stream) {
    switch (x_dtype) {
        case X_F32: return launch_x<X_F32>(p, stream);
        case X_BF16: return launch_x<X_BF16>(p, stream);
        case X_F16: return launch_x<X_F16>(p, stream);
    }
    return hipErrorInvalidValue;
}
