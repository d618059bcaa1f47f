// What the kernels that quantise rows share: eight elements of a row as loaded, the cleaning of special values, the exact quotient by the row's scale and
// the packing of eight 8-bit outputs.
#pragma once
#include "psg_common.h"

namespace {

enum { X_F32 = 0, X_BF16 = 1, X_F16 = 2 };

// NaN -> 0, +-Inf -> +-dtypeMax, finite values untouched
__device__ __forceinline__ float clean(float t, float dmax) {
    if (t != t) return 0.0f;
    if (__builtin_isinf(t)) return t > 0.0f ? dmax : -dmax;
    return t;
}

// x / s, rounded to nearest even, for a scale s inside [2^-80, 2^100]: y is the correctly rounded 1 / s, so two correction
// steps make the quotient the correctly rounded one (P. Markstein, "Computation of elementary functions on the IBM RISC
// System/6000 processor", 1990: a faithful q, the exact remainder r = x - q s and one more fma).  Inside the bounds a
// remainder can only underflow where |q| < 2^-20, and there every output is a zero; the sign is copied from x because a
// remainder of +0 would turn -0 into +0.  Six instructions for an element against eleven of the IEEE division sequence.
__device__ __forceinline__ float quotient(float x, float s, float y) {
    float q = x * y;
    q = __builtin_fmaf(__builtin_fmaf(-q, s, x), y, q);
    q = __builtin_fmaf(__builtin_fmaf(-q, s, x), y, q);
    return __builtin_copysignf(q, x);
}

template <int OUT_FP8>
__device__ __forceinline__ v2i quant_pack8(const float* q) {
    v2i o;
    if constexpr (OUT_FP8) {
        // v_cvt_pk_fp8_f32: two fp32 -> two OCP e4m3 bytes, round to nearest even (|q| <= 448 here, so its
        // saturation never comes into play)
        unsigned w0 = 0, w1 = 0;
        w0 = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], w0, false);
        w0 = __builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], w0, true);
        w1 = __builtin_amdgcn_cvt_pk_fp8_f32(q[4], q[5], w1, false);
        w1 = __builtin_amdgcn_cvt_pk_fp8_f32(q[6], q[7], w1, true);
        o[0] = (int)w0;
        o[1] = (int)w1;
    } else {
        uint32_t b[8];
#pragma unroll
        for (int e = 0; e < 8; e++) b[e] = (uint32_t)(int32_t)q[e] & 0xFFu;  // float -> int truncates toward zero
        o[0] = (int)(b[0] | (b[1] << 8) | (b[2] << 16) | (b[3] << 24));
        o[1] = (int)(b[4] | (b[5] << 8) | (b[6] << 16) | (b[7] << 24));
    }
    return o;
}

// Eight consecutive elements as they are loaded, and what the two passes need of them
typedef unsigned short v2us __attribute__((ext_vector_type(2)));
template <int XT>
struct Raw8 {
    v4i w[XT == X_F32 ? 2 : 1];
    __device__ __forceinline__ void load(const void* base, size_t elem) {
        const v4i* p = reinterpret_cast<const v4i*>(static_cast<const uint8_t*>(base) + elem * (XT == X_F32 ? 4 : 2));
        w[0] = p[0];
        if constexpr (XT == X_F32) w[1] = p[1];
    }
    // running maximum of |x| on the bit patterns, which order like the magnitudes (NaN above Inf above every finite value):
    // fp32 as 32 bits, the 16-bit types as two packed halves
    __device__ __forceinline__ uint32_t max_bits(uint32_t m) const {
#pragma unroll
        for (int j = 0; j < (XT == X_F32 ? 2 : 1); j++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                if constexpr (XT == X_F32) {
                    const uint32_t u = (uint32_t)w[j][i] & 0x7FFFFFFFu;
                    m = u > m ? u : m;
                } else {
                    const v2us a = __builtin_bit_cast(v2us, (uint32_t)w[j][i] & 0x7FFF7FFFu), b = __builtin_bit_cast(v2us, m);
                    m = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(a, b));
                }
            }
        return m;
    }
    __device__ __forceinline__ void values(float* v) const {
        if constexpr (XT == X_F32) {
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] = __int_as_float(w[e >> 2][e & 3]);
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const uint32_t u = (uint32_t)w[0][i];
                if constexpr (XT == X_BF16) {
                    v[2 * i] = __builtin_bit_cast(float, u << 16);
                    v[2 * i + 1] = __builtin_bit_cast(float, u & 0xFFFF0000u);
                } else {
                    v[2 * i] = (float)__builtin_bit_cast(_Float16, (uint16_t)(u & 0xFFFF));
                    v[2 * i + 1] = (float)__builtin_bit_cast(_Float16, (uint16_t)(u >> 16));
                }
            }
        }
    }
};

}  // namespace
