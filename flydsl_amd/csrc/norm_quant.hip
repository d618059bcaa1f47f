// Residual addition, root-mean-square norm and per-row quantisation in one pass (gfx950): what stands in front of every quantised product of a
// decoder layer.
//
//   h = round(x + r)                       the residual stream, in the type of x (h = x without a residual)
//   y = (h w) / sqrt(mean(h^2) + eps)      fp32
//   s = max|y| / dmax, q = y / s           the rule of k_quant_pertoken: s = 1 for a row of zeros, NaN -> 0, +-Inf -> +-dmax, int8 towards zero, fp8 to nearest even
//
// The norm is of the rounded h, so that it is the norm of what the layers behind read as residual; q is made of y, not of its 16-bit rounding.
// One pass: the maximum does not need the norm, max|y| = max|h w| / rms with the same rounding (a product with a positive factor is monotone), so the sum of squares and
// the maximum leave a row together, with one barrier, and the row stays in registers as h w in between.  The rms cancels in q = h w dmax / max|h w|, which is taken
// like this, to fp32 with one rounding: q is the definition's but where that rounding meets a border, and the row's maximum is dmax exactly.
// A row whose squares are beyond fp32 or below it (h from about 2^58 on; below 2^-50 with an eps below 2^-60) is read a second and a third time, scaled by powers of two.
// Bound: HBM, every operand read once and every output written once, behind 2.9 us that a launch takes whatever it moves.  us, bf16 to fp8 with a residual, launches on end over three sets of
// operands: 8192 rows of 8192 82.7 (470 MB, 5.7 TB/s), 256 of 4096 4.4, 67 of 8192 4.7, one of 4096 3.9.  Rows that begin off 16 bytes cost nothing (8192 of 2048, 2048 to 2056 elements apart,
// 26.3 to 28.5), off four bytes some, and so does an end that is no whole vector: 8192 of 2048 25.0, 2056 29.3, 2046 28.4, 2050 30.8, 2047 31.0, 2049 35.3.
#include "psg_common.h"
#include "quant_rows.h"
#include "norm_quant.h"

namespace {

// (a row's end in pieces of 4, 2 and 1)
template <int XT, bool WHOLE>
__device__ __forceinline__ void store_row(void* base, int64_t i, int n, const Raw8<XT>& r) {
    constexpr int B = XT == X_F32 ? 4 : 2;
    uint8_t* at = static_cast<uint8_t*>(base) + i * B;
    if (WHOLE || n >= 8) {
        v4i_any* p = reinterpret_cast<v4i_any*>(at);
        p[0] = r.w[0];
        if constexpr (XT == X_F32) p[1] = r.w[1];
    } else if constexpr (XT == X_F32) {
        v4i w = r.w[0];
        if (n & 4) *reinterpret_cast<v4i_any*>(at) = w, at += 16, w = r.w[1];
        if (n & 2) *reinterpret_cast<v2i_any*>(at) = (v2i){w[0], w[1]}, at += 8, w[0] = w[2];
        if (n & 1) *reinterpret_cast<int*>(at) = w[0];
    } else {
        v2i w = {r.w[0][0], r.w[0][1]};
        if (n & 4) *reinterpret_cast<v2i_any*>(at) = w, at += 8, w = (v2i){r.w[0][2], r.w[0][3]};
        if (n & 2) *reinterpret_cast<int_any*>(at) = w[0], at += 4, w[0] = w[1];
        if (n & 1) *reinterpret_cast<uint16_t*>(at) = (uint16_t)w[0];
    }
}

// eight values rounded to the type of x
template <int XT>
__device__ __forceinline__ Raw8<XT> round8(const float* v) {
    Raw8<XT> r;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if constexpr (XT == X_F32) {
            r.w[i >> 1][2 * (i & 1)] = __float_as_int(v[2 * i]);
            r.w[i >> 1][2 * (i & 1) + 1] = __float_as_int(v[2 * i + 1]);
        } else {
            r.w[0][i] = pack2_out16<XT == X_BF16 ? OUT_BF16 : OUT_FP16>(v[2 * i], v[2 * i + 1]);
        }
    }
    return r;
}

// v d / m rounded once, for m inside the bounds of quotient() and |v| <= m: its correction steps on the whole product.  SHORT: the product is exact (8 + 8 bits of a bf16
// value and weight and 7 of d).
template <bool SHORT>
__device__ __forceinline__ float times_over(float v, float d, float m, float rm) {
    const float hi = v * d;
    if constexpr (SHORT) return quotient(hi, m, rm);
    const float lo = __builtin_fmaf(v, d, -hi);
    float q = hi * rm;
    q = __builtin_fmaf(__builtin_fmaf(-q, m, hi) + lo, rm, q);
    q = __builtin_fmaf(__builtin_fmaf(-q, m, hi) + lo, rm, q);
    return __builtin_copysignf(q, v);
}

// A row belongs to a workgroup of up to MOST threads.  (Rows of up to 256 vectors as four to a workgroup, one to a wavefront, without
// the barrier, took / take like this, 8192 of them, us: 280 6.9 / 7.3, 512 9.2 / 8.1, 1024 14.2 / 12.3, 2048 25.5 / 25.0, but with ends 2041 28.7 / 30.9, 2047 29.9 / 31.1, 2049 40.0 / 35.3.)  The first KEEP 8-element vectors of every thread stay in registers; a
// longer row writes its h, or has it in x, and reads the rest of it once more, every thread what it has written itself.
// WHOLE: rows are whole vectors.  WT: type of the weight.
template <int XT, int WT, int MOST, int KEEP, bool WHOLE>
__global__ void __launch_bounds__(MOST) k_rmsnorm_quant(NormParams p) {
    __shared__ float red_s[MOST / 64];
    __shared__ uint32_t red_m[MOST / 64];
    const int NT = (int)blockDim.x, tid = (int)threadIdx.x, wave = wave_id();
    const int64_t row = blockIdx.x;
    const int nvec = (p.dim + 7) >> 3;
    const int64_t xb = row * p.x_stride, rb = row * p.r_stride, hb = row * p.h_stride, nb = row * p.n_stride, qb = row * (int64_t)p.dim;
    auto left = [&](int vi) { return p.dim - vi * 8; };
    auto weights = [&](int vi) __attribute__((always_inline)) { return load_row<WT, WHOLE>(p.weight, (int64_t)vi * 8, left(vi), p.dim); };

    float sum = 0.f, hw[KEEP][8];
    uint32_t mb = 0;
    // adds a vector's squares and its maximum, as h w with its sign dropped, on the bit patterns: NaN above Inf above every finite value
    auto take = [&](const float* h, const float* w, float* out) __attribute__((always_inline)) {
#pragma unroll
        for (int e = 0; e < 8; e++) {
            sum = __builtin_fmaf(h[e], h[e], sum);
            out[e] = h[e] * w[e];
            const uint32_t u = __builtin_bit_cast(uint32_t, out[e]) & 0x7FFFFFFFu;
            mb = u > mb ? u : mb;
        }
    };
    // (a vector that begins less than eight elements in front of the row's end, of a row that has eight)
    auto is_end = [&](int vi) { return !WHOLE && left(vi) < 8 && p.dim >= 8; };
    auto add = [&](const Raw8<XT>& x, const Raw8<XT>& r, int vi, bool live, float* h) __attribute__((always_inline)) {
        x.values(h);
        if (p.residual) {
            float v[8];
            r.values(v);
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] = h[e] + v[e];
            const Raw8<XT> k = round8<XT>(v);
            k.values(h);
            if (live) store_row<XT, WHOLE>(p.h, hb + (int64_t)vi * 8, left(vi), k);
        }
    };

    {
        // threads past the row read its first vector again: no load stands behind a branch of its own
        Raw8<XT> x[KEEP], r[KEEP];
        Raw8<WT> w[KEEP];
        auto at = [&](int it) { return tid + it * NT < nvec ? tid + it * NT : 0; };
#pragma unroll
        for (int it = 0; it < KEEP; it++) r[it] = x[it] = load_row<XT, WHOLE>(p.x, xb + (int64_t)at(it) * 8, left(at(it)), p.dim);
        if (p.residual) {
#pragma unroll
            for (int it = 0; it < KEEP; it++) r[it] = load_row<XT, WHOLE>(p.residual, rb + (int64_t)at(it) * 8, left(at(it)), p.dim);
        }
#pragma unroll
        for (int it = 0; it < KEEP; it++) w[it] = weights(at(it));
#pragma unroll
        for (int it = 0; it < KEEP; it++) {
            const bool live = tid + it * NT < nvec;
            if (live && is_end(tid + it * NT)) {
                line_up<XT>(x[it], left(tid + it * NT));
                line_up<XT>(r[it], left(tid + it * NT));
                line_up<WT>(w[it], left(tid + it * NT));
            }
            float h[8], wv[8];
            add(x[it], r[it], tid + it * NT, live, h);
            w[it].values(wv);
            if (!live) {
#pragma unroll
                for (int e = 0; e < 8; e++) h[e] = wv[e] = 0.f;
            }
            take(h, wv, hw[it]);
        }
    }
    for (int vi = tid + KEEP * NT; vi < nvec; vi += NT) {
        Raw8<XT> x = load_row<XT, WHOLE>(p.x, xb + (int64_t)vi * 8, left(vi), p.dim);
        Raw8<XT> r = p.residual ? load_row<XT, WHOLE>(p.residual, rb + (int64_t)vi * 8, left(vi), p.dim) : x;
        Raw8<WT> wr = weights(vi);
        if (is_end(vi)) {
            line_up<XT>(x, left(vi));
            line_up<XT>(r, left(vi));
            line_up<WT>(wr, left(vi));
        }
        float w[8], h[8], y[8];
        wr.values(w);
        add(x, r, vi, true, h);
        take(h, w, y);
    }

    auto over_row = [&](float& s, uint32_t& m) __attribute__((always_inline)) {
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) {
            s += __shfl_xor(s, off, 64);
            const uint32_t o = (uint32_t)__shfl_xor((int)m, off, 64);
            m = o > m ? o : m;
        }
        if ((tid & 63) == 0) red_s[wave] = s, red_m[wave] = m;
        __syncthreads();
        s = red_s[0], m = red_m[0];
        for (int i = 1; i < NT / 64; i++) {
            s += red_s[i];
            m = red_m[i] > m ? red_m[i] : m;
        }
    };
    over_row(sum, mb);
    const float mean = sum / (float)p.dim + p.eps;
    float rinv = 1.0f / __builtin_sqrtf(mean);
    int up = 0;  // h is taken times 2^up, rinv is of that

    // h w of a vector that is not in registers
    auto again = [&](int vi, float* v, bool product) __attribute__((always_inline)) {
        Raw8<XT> h = p.residual ? load_row<XT, WHOLE>(p.h, hb + (int64_t)vi * 8, left(vi), p.dim) : load_row<XT, WHOLE>(p.x, xb + (int64_t)vi * 8, left(vi), p.dim);
        Raw8<WT> wr = weights(vi);
        if (is_end(vi)) {
            line_up<XT>(h, left(vi));
            line_up<WT>(wr, left(vi));
        }
        float w[8];
        h.values(v);
        wr.values(w);
        if (up) {
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] = __builtin_ldexpf(v[e], up);
        }
        if (!product) return;
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] *= w[e];
    };

    // Rows whose squares, whose sum of them or whose products with the weight leave fp32's range, though y does not, are taken once more: the sum of (h 2^-80)^2 or (h 2^100)^2, all of
    // whose terms that matter are normal numbers, then h 2^up with a root mean square from 1/2 to 1, so that its products leave the range only where y does.  What the first sum
    // is short of, squares below 2^-149, is less than 2^-125 and is nothing beside an eps from 2^-60 on.  (Infinities and NaN of h stay: their sum is none either way.)
    const bool far_sum = mean == __builtin_inff() || (sum < 0x1p-100f && p.eps < 0x1p-60f);
    // (What asks for it costs every launch 0.05 to 0.12 us: 67 rows of 8192 4.58 / 4.67, 8192 level.)
    if (__builtin_expect(far_sum || mb == 0x7F800000u || (mb < 0x17800000u && sum > 0.f && mean < 0.25f), 0)) {  // (the bits of infinity and of 2^-80)
        float sq = sum, unused_s = 0.f;
        uint32_t m = 0;
        if (sum == __builtin_inff()) up = -80;
        else if (sum < 0x1p-100f) up = 100;
        const int first = up;
        if (first) {
            sq = 0.f;
            for (int vi = tid; vi < nvec; vi += NT) {
                float h[8];
                again(vi, h, false);
#pragma unroll
                for (int e = 0; e < 8; e++) sq = __builtin_fmaf(h[e], h[e], sq);
            }
            __syncthreads();  // everybody has read what over_row left
            over_row(sq, m);
        }
        const double ms = __builtin_ldexp((double)sq, -2 * first) / p.dim + (double)p.eps;
        up = 0;
        if (ms > 0.0 && sq < __builtin_inff()) {
            const double rms = __builtin_sqrt(ms);
            up = -__builtin_amdgcn_frexp_exp(rms);
            rinv = (float)(1.0 / __builtin_ldexp(rms, up));
            mb = 0;
            auto largest = [&](const float* v) __attribute__((always_inline)) {
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const uint32_t u = __builtin_bit_cast(uint32_t, v[e]) & 0x7FFFFFFFu;
                    mb = u > mb ? u : mb;
                }
            };
#pragma unroll
            for (int it = 0; it < KEEP; it++)
                if (tid + it * NT < nvec) {
                    again(tid + it * NT, hw[it], true);
                    largest(hw[it]);
                }
            for (int vi = tid + KEEP * NT; vi < nvec; vi += NT) {
                float v[8];
                again(vi, v, true);
                largest(v);
            }
            __syncthreads();
            over_row(unused_s, mb);
        }
    }

    const float dmax = p.out == NORM_FP8 ? 448.0f : 127.0f;
    float s = 1.0f;
    const float mhw = __builtin_bit_cast(float, mb);
    const float rm = 1.0f / mhw;
    bool exact = true;  // no value needs cleaning, and the maximum lies where quotient() is exact; uniform over the row
    if (p.out != NORM_NONE) {
        float amax = mhw * rinv;
        const bool special = !(amax < __builtin_inff());  // an Inf or NaN among the row's values, or a norm that is none
        if (special) {
            float m = 0.f, unused = 0.f;
#pragma unroll
            for (int it = 0; it < KEEP; it++)
#pragma unroll
                for (int e = 0; e < 8; e++) m = fmaxf(m, fabsf(clean(hw[it][e] * rinv, dmax)));
            for (int vi = tid + KEEP * NT; vi < nvec; vi += NT) {
                float v[8];
                again(vi, v, true);
#pragma unroll
                for (int e = 0; e < 8; e++) m = fmaxf(m, fabsf(clean(v[e] * rinv, dmax)));
            }
            uint32_t bits = __builtin_bit_cast(uint32_t, m);
            __syncthreads();  // everybody has read what over_row left
            over_row(unused, bits);
            amax = __builtin_bit_cast(float, bits);
        }
        s = amax / dmax;
        exact = !special && s >= 0x1p-80f && s <= 0x1p100f && mhw >= 0x1p-80f && mhw <= 0x1p100f;
        if (s == 0.0f) s = 1.0f;  // (a row of zeros, or of values whose scale is rounded to zero, and their codes with it)
        if (tid == 0) p.scale[row] = s;
    }
    auto finish = [&](int vi, const float* v) __attribute__((always_inline)) {
        const int n = left(vi);
        float y[8];
#pragma unroll
        for (int e = 0; e < 8; e++) y[e] = v[e] * rinv;
        if (p.normed) store_row<XT, WHOLE>(p.normed, nb + (int64_t)vi * 8, n, round8<XT>(y));
        if (p.out == NORM_NONE) return;
        if (exact) {
#pragma unroll
            for (int e = 0; e < 8; e++) y[e] = times_over<XT == X_BF16 && WT == X_BF16>(v[e], dmax, mhw, rm);
        } else {
            // (a scale near the smallest number has a few bits only and may be too small by a third: held within +-dmax, where int8 would wrap and fp8 has no number)
#pragma unroll
            for (int e = 0; e < 8; e++) y[e] = fminf(fmaxf(clean(y[e], dmax) / s, -dmax), dmax);
        }
        const v2i o = p.out == NORM_FP8 ? quant_pack8<1>(y) : quant_pack8<0>(y);
        uint8_t* dst = p.q + qb + (int64_t)vi * 8;
        if (WHOLE || n >= 8) {
            *reinterpret_cast<v2i_any*>(dst) = o;
        } else {
            uint32_t b = (uint32_t)o[0];
            if (n & 4) *reinterpret_cast<int_any*>(dst) = (int)b, dst += 4, b = (uint32_t)o[1];
            if (n & 2) *reinterpret_cast<half_any*>(dst) = (uint16_t)b, dst += 2, b >>= 16;
            if (n & 1) *dst = (uint8_t)b;
        }
    };
#pragma unroll
    for (int it = 0; it < KEEP; it++) {
        const int vi = tid + it * NT;
        if (vi < nvec) finish(vi, hw[it]);
    }
    for (int vi = tid + KEEP * NT; vi < nvec; vi += NT) {
        float v[8];
        again(vi, v, true);
        finish(vi, v);
    }
}

// `threads` a row, in launches of 2^31 threads at most: a grid holds no more than 2^32
template <int XT, int WT, int MOST, int KEEP, bool WHOLE>
hipError_t launch_rows(NormParams p, int threads, hipStream_t stream) {
    constexpr int64_t B = XT == X_F32 ? 4 : 2;
    const int64_t most = (1ll << 31) / MOST;
    for (int64_t left = p.rows;; left -= most) {
        p.rows = left < most ? left : most;
        hipLaunchKernelGGL((k_rmsnorm_quant<XT, WT, MOST, KEEP, WHOLE>), dim3((unsigned)p.rows), dim3(threads), 0, stream, p);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess || left <= most) return e;
        p.x = static_cast<const uint8_t*>(p.x) + most * p.x_stride * B;
        if (p.residual) {
            p.residual = static_cast<const uint8_t*>(p.residual) + most * p.r_stride * B;
            p.h = static_cast<uint8_t*>(p.h) + most * p.h_stride * B;
        }
        if (p.normed) p.normed = static_cast<uint8_t*>(p.normed) + most * p.n_stride * B;
        if (p.out != NORM_NONE) p.q += most * p.dim, p.scale += most;
    }
}

template <int XT, int WT, bool WHOLE>
hipError_t launch(const NormParams& p, hipStream_t stream) {
    const int nvec = (p.dim + 7) / 8;
    const int64_t cus = psg_cu_count();
#define PSG_NORM(MOST_, KEEP_) return launch_rows<XT, WT, MOST_, KEEP_, WHOLE>(p, (nvec + KEEP_ * 64 - 1) / (KEEP_ * 64) * 64, stream);
    // Vectors of a thread; as many wavefronts as the row then fills (all sixteen of 1024 threads where nine have work: 8192 rows of 9042 169 us / 111).  us, bf16 to fp8 with a residual.
    // One vector or two, few or short rows, which want their loads at once: 4 rows of 1204 3.3 / 3.9, 777 of 2051 5.9 / 6.4, 300 of 3401 5.1 / 5.3 (of 3584, without an end, level); of many rows a CU
    // holds more with two, 8192 of 2048 27.4 / 25.2, of 2880 40.7 / 33.4, of 5120 70 / 54.6.
    if (nvec <= 64 || (nvec <= (WHOLE ? 320 : 512) && p.rows * nvec <= 1024 * cus)) PSG_NORM(512, 1)
    // Two or four: 4 of 1204 3.9 / 4.5, 300 of 3401 5.3 / 6.4, 8192 of 2048 25.2 / 25.3, of 5120 54.6 / 54.2; but with the code for a row's end 8192 of 5124 66 / 59, 300 6.1 / 6.6.
    if (nvec <= 512 || (nvec <= 1024 && (WHOLE || p.rows <= 4 * cus))) PSG_NORM(512, 2)
    // The same on up to 768 threads: 4 of 9042 4.7 / 5.5, 1100 of 12288 20.9 / 22.8, 8192 122 / 125; but with ends 8192 of 9715 147 / 136, and 13 to 15 wavefronts leave room for no second workgroup
    // beside them, 8192 of 14336 157 / 143.
    if (nvec > 1024 && nvec <= 1536 && (WHOLE || p.rows <= 4 * cus)) PSG_NORM(1024, 2)
    if (nvec <= 2048) PSG_NORM(512, 4)
    return launch_rows<XT, WT, 1024, 4, WHOLE>(p, nvec > 4096 ? 1024 : (nvec + 255) / 256 * 64, stream);  // (beyond 32768 elements threads come back for the rest)
#undef PSG_NORM
}

}  // namespace

// x_dtype: 0 fp32, 1 bf16, 2 fp16.  Requires rows, dim >= 1 and addresses that are multiples of their elements.
hipError_t psg_launch_rmsnorm_quant(const NormParams& p, int x_dtype, hipStream_t stream) {
    // (what WHOLE spares is the code for the end of a row: 8192 rows of 2048 25.0 / 27.3 us, in fp32 44.0 / 49.4, of 8192 82.8 / 88.4)
    const bool whole = p.dim % 8 == 0;
#define PSG_NORM_T(XT_, WT_) return whole ? launch<XT_, WT_, true>(p, stream) : launch<XT_, WT_, false>(p, stream);
    switch (x_dtype) {
        case X_F32: PSG_NORM_T(X_F32, X_F32)
        case X_BF16: if (p.w_f32) PSG_NORM_T(X_BF16, X_F32) else PSG_NORM_T(X_BF16, X_BF16)
        case X_F16: if (p.w_f32) PSG_NORM_T(X_F16, X_F32) else PSG_NORM_T(X_F16, X_F16)
    }
#undef PSG_NORM_T
    return hipErrorInvalidValue;
}
