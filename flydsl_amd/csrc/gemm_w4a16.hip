// A few rows of 16-bit activations times 4-bit weights with a 16-bit scale, and a zero point or none, per group of 32, 64 or 128 elements along K (gfx950).
//
//   C[m, n] = sum over the groups g of  s[n, g] (P[m, n, g] - z[n, g] X[m, g]),   P = sum over k in g of A[m, k] (16 + q[n, k]),   X = sum over k in g of A[m, k]
//
// with z = 16 + zero point (24 without zero points: codes 0..15 stand for -8..7).  A code q is made an operand of the matrix cores by two instructions for two of them: shifted to
// the upper bits of a mantissa, masked and joined with the exponent of 16 it is the 16-bit number 16 + q exactly, in bf16 as in fp16.  The 16 and the zero point come off the group's sum
// in fp32, and X of a lane's own row is what the same MFMA gives for a weight of ones.  (P is at most 31/16 of the sum with the 16 alone: the difference loses four or five of 24
// bits, far below the 16-bit output's rounding.)
//
// Bound: the weights' way from memory.  The columns are dealt out in units of 8, evenly, one workgroup a CU; its eight wavefronts are eight slices of K.  A wavefront's part of A, 16
// rows of up to 1024 elements, stays in registers (128 of them) while the workgroup's columns go by in windows of 16, and so do the X of its groups: what moves is W alone, asked for
// eight steps ahead, windows on end, without a barrier.  The slices' sums meet in LDS in a fixed order: one launch, no workspace.  Longer rows take several passes over the
// columns, each with its part of A.
//
// Layout: W in blocks of 16 rows x 128 elements, 1 KB: lane l = 16 g + r of a wavefront reads 16 bytes, row r, dword j of them elements 32 j + 8 g .. + 7, what
// it multiplies in MFMA j; the even ones are the nibbles of the lower half of the dword, the odd ones those of the upper half, so that two of them are a mask away from a
// packed pair.  Rows end on whole blocks (elements past K are not looked at: A reads as zero there and X with it).  Scales [N/16][K/group][16], zero points the same as
// nibbles, lower one first: a lane's four columns are 8 and 2 bytes.
#include "gemm_w4a16.h"

namespace {

// Constants in registers of the two files: an instruction that masks and joins takes one from each, and the compiler would otherwise make two of it, a literal each
template <int MASK, int BASE>
struct Join {
    int mask = MASK, base = BASE;
    __device__ __forceinline__ Join() { asm("" : "+s"(mask), "+v"(base)); }
    __device__ __forceinline__ int operator()(int x) const { return (x & mask) | base; }
};
__device__ __forceinline__ int shift(int x, int left) { return left >= 0 ? x << left : (int)((unsigned)x >> -left); }

template <bool BF16>
__device__ __forceinline__ v4f mfma16(v4i w, v4i a, v4f c) {
    if constexpr (BF16) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, w), __builtin_bit_cast(v8bf, a), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, w), __builtin_bit_cast(v8h, a), c, 0, 0, 0);
}

constexpr int W4_WAVES = 8;

// MB: 16-row blocks of A.  GS: elements of a group.  ZP: zero points.  SPW: 128-element steps of a wavefront's part of A.  R: windows that are asked for ahead.
template <bool BF16, int MB, int GS, bool ZP, int SPW, int R>
__global__ void __launch_bounds__(W4_WAVES * 64, 2) k_w4a16(W4Params p) {
    constexpr int GPS = 128 / GS, MPG = GS / 32;  // groups of a step, MFMAs of a group
    extern __shared__ v4f part[];                 // [wavefront][window][16-row block][lane]
    const int tid = threadIdx.x, wave = wave_id(), lane = tid & 63, li = lane & 15, lg = lane >> 4;
    auto unit_begin = [&](int g) { return g * p.unit_q + (g < p.unit_r ? g : p.unit_r); };
    // an XCD owns one range of columns: workgroups go round the XCDs
    const int wg = (gridDim.x & 7) == 0 ? (int)((blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3)) : (int)blockIdx.x;
    const int n_begin = unit_begin(wg) * 8, n_end = unit_begin(wg + 1) * 8, windows = (n_end - n_begin + 15) >> 4;
    const int m0 = (int)blockIdx.y * MB * 16, M = p.M - m0, K = p.K, steps = (K + 127) >> 7, groups = K / GS;

    const __amdgpu_buffer_rsrc_t rw = make_rsrc(p.w, (uint64_t)p.N * (uint64_t)steps * 64ull), rs = make_rsrc(p.scales, (uint64_t)p.N * (uint64_t)groups * 2ull),
                                 rz = make_rsrc(ZP ? p.zeros : p.w, (uint64_t)p.N * (uint64_t)groups / 2ull),
                                 ra = make_rsrc(static_cast<const uint16_t*>(p.a) + (uint64_t)m0 * (uint64_t)K, (uint64_t)M * (uint64_t)K * 2ull);
    // a lane reads row n of W, and the scales of the four columns from c on that it holds of C; a window is 16 rows on
    const int n_lane = n_begin + li, c_lane = n_begin + lg * 4;
    const uint32_t w_lane = (uint32_t)(n_lane >> 4) * (uint32_t)steps * 1024u + (uint32_t)(lg * 256 + (n_lane & 15) * 16);
    const uint32_t s_lane = (uint32_t)(c_lane >> 4) * (uint32_t)groups * 32u + (uint32_t)(c_lane & 15) * 2u;
    uint32_t a_lane[MB];
#pragma unroll
    for (int mb = 0; mb < MB; mb++) a_lane[mb] = mb * 16 + li < M ? (uint32_t)(mb * 16 + li) * (uint32_t)K * 2u + (uint32_t)lg * 16u : OOB;
    const Join<BF16 ? 0x00780078 : 0x03C003C0, BF16 ? 0x41804180 : 0x4C004C00> code;  // a code in the bits of the mantissa that count 1 to 8 beside 16
    const Join<0x00780000, 0x41800000> zero;                                           // the same in fp32

    for (int pass = 0; pass < p.passes; pass++) {
        const int s0 = (pass * W4_WAVES + wave) * p.per, s1 = s0 + p.per < steps ? s0 + p.per : steps;
        v4i w[R][SPW];
        v2i sc[R][SPW][GPS];
        int z[R][SPW][ZP ? GPS : 1];
        auto load = [&](int win, int t, auto I) __attribute__((always_inline)) {
            constexpr int i = decltype(I)::value;
            const bool in = win < windows && s0 + t < s1;  // uniform
            const bool row = in && n_lane + win * 16 < n_end, col = in && c_lane + win * 16 < n_end;
            w[i][t] = buf_load16_nt(rw, row ? w_lane : OOB, in ? ((uint32_t)win * (uint32_t)steps + (uint32_t)(s0 + t)) * 1024u : 0u);
#pragma unroll
            for (int g = 0; g < GPS; g++) {
                const int at = (s0 + t) * GPS + g;
                const bool has = in && at < groups;
                const uint32_t so = has ? (uint32_t)win * (uint32_t)groups + (uint32_t)at : 0u;
                sc[i][t][g] = buf_load8(rs, col && has ? s_lane : OOB, so * 32u);
                if constexpr (ZP) z[i][t][g] = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(rz, (int)(col && has ? s_lane >> 2 : OOB), (int)(so * 8u), 0);
            }
        };
        v4i a[SPW][4][MB];
#pragma unroll
        for (int t = 0; t < SPW; t++)
#pragma unroll
            for (int j = 0; j < 4; j++)
#pragma unroll
                for (int mb = 0; mb < MB; mb++) {
                    const int k = (s0 + t) * 128 + j * 32;
                    const bool in = s0 + t < s1 && k < K;  // (K is a multiple of 32)
                    a[t][j][mb] = buf_load16(ra, in ? a_lane[mb] : OOB, in ? (uint32_t)k * 2u : 0u);
                }
        static_for<R>([&](auto I) {
#pragma unroll
            for (int t = 0; t < SPW; t++) load(decltype(I)::value, t, I);
        });
        __builtin_amdgcn_sched_barrier(0);

        // X of every group, times -24 without zero points
        float x[SPW][GPS][MB];
        const int one = BF16 ? (ZP ? 0x3F803F80 : (int)0xC1C0C1C0) : (ZP ? 0x3C003C00 : (int)0xCE00CE00);
        const v4i ones = {one, one, one, one};
#pragma unroll
        for (int t = 0; t < SPW; t++)
#pragma unroll
            for (int g = 0; g < GPS; g++)
#pragma unroll
                for (int mb = 0; mb < MB; mb++) {
                    v4f y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int j = g * MPG; j < (g + 1) * MPG; j++) y = mfma16<BF16>(ones, a[t][j][mb], y);
                    x[t][g][mb] = y[0];
                }

        auto window = [&](int win, auto I) __attribute__((always_inline)) {
            constexpr int i = decltype(I)::value;
            v4f acc[MB];
#pragma unroll
            for (int mb = 0; mb < MB; mb++) acc[mb] = (v4f){0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int t = 0; t < SPW; t++) {
#pragma unroll
                for (int g = 0; g < GPS; g++) {
                    v4f pr[MB];
#pragma unroll
                    for (int mb = 0; mb < MB; mb++) pr[mb] = (v4f){0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int j = g * MPG; j < (g + 1) * MPG; j++) {
                        v4i b;
#pragma unroll
                        for (int q = 0; q < 4; q++) b[q] = code(shift(w[i][t][j], (BF16 ? 3 : 6) - 4 * q));
#pragma unroll
                        for (int mb = 0; mb < MB; mb++) pr[mb] = mfma16<BF16>(b, a[t][j][mb], pr[mb]);
                    }
#pragma unroll
                    for (int v = 0; v < 4; v++) {
                        const float s = from_out16<BF16 ? OUT_BF16 : OUT_FP16>((uint16_t)((uint32_t)sc[i][t][g][v >> 1] >> (16 * (v & 1))));
                        const float zc = ZP ? __builtin_bit_cast(float, zero(z[i][t][g] << (19 - 4 * v))) : 0.f;
#pragma unroll
                        for (int mb = 0; mb < MB; mb++) acc[mb][v] = __builtin_fmaf(s, ZP ? __builtin_fmaf(-zc, x[t][g][mb], pr[mb][v]) : pr[mb][v] + x[t][g][mb], acc[mb][v]);
                    }
                }
                load(win + R, t, I);
                __builtin_amdgcn_sched_barrier(0);
            }
#pragma unroll
            for (int mb = 0; mb < MB; mb++) {
                v4f* at = part + ((wave * windows + win) * MB + mb) * 64 + lane;
                *at = pass ? *at + acc[mb] : acc[mb];
            }
        };
        int w0 = 0;
        for (; w0 + R <= windows; w0 += R) static_for<R>([&](auto I) { window(w0 + decltype(I)::value, I); });
        static_for<R - 1>([&](auto I) {
            if (w0 + decltype(I)::value < windows) window(w0 + decltype(I)::value, I);
        });
    }

    __syncthreads();
    // the slices' sums, in their order
    for (int t = tid; t < windows * MB * 64; t += W4_WAVES * 64) {
        const int frag = t >> 6, m = (frag % MB) * 16 + li, n = n_begin + (frag / MB) * 16 + lg * 4;
        if (n >= n_end || m >= M) continue;
        v4f sum = part[t];
#pragma unroll
        for (int j = 1; j < W4_WAVES; j++) sum += part[j * windows * MB * 64 + t];
        store_c4(p, (size_t)(m0 + m) * (size_t)p.N + (size_t)n, n, sum);
    }
}

template <bool BF16, int MB, int GS, bool ZP, int SPW, int R>
hipError_t go(W4Params p, hipStream_t stream) {
    const int steps = (p.K + 127) / 128;
    p.passes = (steps + W4_WAVES * SPW - 1) / (W4_WAVES * SPW);
    p.per = (steps + W4_WAVES * p.passes - 1) / (W4_WAVES * p.passes);
    // units of 8 columns: at most `most` a workgroup (its sums take 1 KB of LDS a wavefront, window and 16-row block, 64 KB in all), a whole number of workgroups a CU
    const long units = p.N / 8, cus = psg_cu_count(), most = 16 / MB, rounds = (units + most * cus - 1) / (most * cus), wgs = units < cus * rounds ? units : cus * rounds;
    p.unit_q = (int)(units / wgs), p.unit_r = (int)(units % wgs);
    const long windows = (units + wgs - 1) / wgs + 1 >> 1;
    hipLaunchKernelGGL((k_w4a16<BF16, MB, GS, ZP, SPW, R>), dim3((unsigned)wgs, (unsigned)((p.M + MB * 16 - 1) / (MB * 16))), dim3(W4_WAVES * 64), (size_t)windows * MB * W4_WAVES * 1024, stream, p);
    return hipGetLastError();
}

template <bool BF16, int GS, bool ZP>
hipError_t launch(const W4Params& p, hipStream_t stream) {
    // steps of K that a wavefront has: the least part of A that holds them, or the largest
    const int per = ((p.K + 127) / 128 + W4_WAVES - 1) / W4_WAVES;
    constexpr int AHEAD = GS == 32 ? 4 : 8;  // steps asked for ahead
    if (p.M <= 16) {
        if (per <= 2) return go<BF16, 1, GS, ZP, 2, AHEAD / 2>(p, stream);
        if (per <= 4 || GS == 32) return go<BF16, 1, GS, ZP, 4, AHEAD / 4>(p, stream);
        return go<BF16, 1, GS, ZP, GS == 32 ? 4 : 8, 1>(p, stream);
    }
    if (per <= 2 || GS == 32) return go<BF16, 2, GS, ZP, 2, AHEAD / 2>(p, stream);
    return go<BF16, 2, GS, ZP, GS == 32 ? 2 : 4, GS == 32 ? AHEAD / 2 : AHEAD / 4>(p, stream);
}

template <bool BF16, int GS>
hipError_t launch_zp(const W4Params& p, hipStream_t stream) {
    return p.zeros ? launch<BF16, GS, true>(p, stream) : launch<BF16, GS, false>(p, stream);
}

}  // namespace

// p.out: type of A, the scales, the bias and C; group: 32, 64 or 128
hipError_t psg_launch_w4a16(const W4Params& p, int group, hipStream_t stream) {
    const bool bf16 = p.out == OUT_BF16;
    switch (group) {
        case 32: return bf16 ? launch_zp<true, 32>(p, stream) : launch_zp<false, 32>(p, stream);
        case 64: return bf16 ? launch_zp<true, 64>(p, stream) : launch_zp<false, 64>(p, stream);
        case 128: return bf16 ? launch_zp<true, 128>(p, stream) : launch_zp<false, 128>(p, stream);
    }
    return hipErrorInvalidValue;
}
