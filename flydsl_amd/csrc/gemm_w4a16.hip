// A few rows of 16-bit activations times 4-bit weights with a 16-bit scale, and a zero point or none, per group of 32, 64 or 128 elements along K (gfx950).
//
//   C[m, n] = sum over the groups g of  s[n, g] (P[m, n, g] - z[n, g] X[m, g]),   P = sum over k in g of A[m, k] (16 + q[n, k]),   X = sum over k in g of A[m, k]
//
// with z = 16 + zero point (24 without zero points: codes 0..15 stand for -8..7).  A code q is made an operand of the matrix cores by two instructions for two of them: shifted to
// the upper bits of a mantissa, masked and joined with the exponent of 16 it is the 16-bit number 16 + q exactly, in bf16 as in fp16.  The 16 and the zero point come off the group's sum
// in fp32, and X of a lane's own row is what the same MFMA gives for a weight of ones.  (P is at most 31/16 of the sum with the 16 alone: the difference loses four or five of 24
// bits, far below the 16-bit output's rounding.)
//
// Bound: the weights' way from memory, like the streaming kernel of the wider types (gemm_a8w8_stream.hip), and dealt out like there: columns in units of 8, evenly over the workgroups,
// a wavefront with up to four units in one or two 16-column windows; the wavefronts of a workgroup are K slices x column groups, their sums meet in LDS in a fixed order, one launch,
// no workspace.
//
// Layout: W in blocks of 16 rows x 128 elements, 1 KB: lane l = 16 g + r of a wavefront reads 16 bytes, row r, dword j of them elements 32 j + 8 g .. + 7, what
// it multiplies in MFMA j; the even ones are the nibbles of the lower half of the dword, the odd ones those of the upper half, so that two of them are a mask away from a
// packed pair.  Rows end on whole blocks (elements past K are not looked at: A reads as zero there and X with it).  Scales [N/16][K/group][16], zero points the same as
// nibbles, lower one first: a lane's four columns are 8 and 2 bytes.
#include "gemm_w4a16.h"

namespace {

// eight codes -> eight operands 16 + q
template <bool BF16>
__device__ __forceinline__ v4i widen(int w) {
    constexpr int UP = BF16 ? 3 : 6;  // from the lowest nibble to the bits of the mantissa that count 1..8 beside 16
    constexpr int MASK = BF16 ? 0x00780078 : 0x03C003C0, BASE = BF16 ? 0x41804180 : 0x4C004C00;
    v4i r;
#pragma unroll
    for (int t = 0; t < 4; t++) {
        const int s = UP - 4 * t;
        r[t] = ((s >= 0 ? w << s : (int)((unsigned)w >> -s)) & MASK) | BASE;
    }
    return r;
}

template <bool BF16>
__device__ __forceinline__ v4f mfma16(v4i w, v4i a, v4f c) {
    if constexpr (BF16) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, w), __builtin_bit_cast(v8bf, a), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, w), __builtin_bit_cast(v8h, a), c, 0, 0, 0);
}

// MB: 16-row blocks of A.  NWIN: 16-column windows of a wavefront.  GS: elements of a group.  ZP: zero points.  CH: 128-element steps that are asked for together.
template <bool BF16, int MB, int NWIN, int GS, bool ZP, int NWAVES, int CH>
__global__ void __launch_bounds__(NWAVES * 64) k_w4a16(W4Params p) {
    constexpr int GPS = 128 / GS, MPG = GS / 32;  // groups of a step, MFMAs of a group
    __shared__ v4f part[NWAVES][NWIN * MB * 64];
    const int tid = threadIdx.x, wave = wave_id(), lane = tid & 63, li = lane & 15, lg = lane >> 4;
    const int ksh = __builtin_ctz(p.ks), gpw = NWAVES >> ksh;  // column groups of a workgroup
    auto unit_begin = [&](int g) { return g * p.unit_q + (g < p.unit_r ? g : p.unit_r); };
    // an XCD owns one range of columns: workgroups go round the XCDs
    const int bid = (gridDim.x & 7) == 0 ? (int)((blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3)) : (int)blockIdx.x;
    const int grp = bid * gpw + (wave >> ksh), m0 = (int)blockIdx.y * MB * 16, M = p.M - m0;
    const int K = p.K, steps = (K + 127) >> 7, groups = K / GS;
    const int per = (steps + p.ks - 1) >> ksh, s0 = (wave & (p.ks - 1)) * per, s1 = s0 + per < steps ? s0 + per : steps;
    const int n_begin = grp < p.groups ? unit_begin(grp) * 8 : 0, n_end = grp < p.groups ? unit_begin(grp + 1) * 8 : 0;

    v4f acc[NWIN][MB];
#pragma unroll
    for (int w = 0; w < NWIN; w++)
#pragma unroll
        for (int mb = 0; mb < MB; mb++) acc[w][mb] = (v4f){0.f, 0.f, 0.f, 0.f};

    if (s0 < s1 && n_begin < n_end) {
        const __amdgpu_buffer_rsrc_t rw = make_rsrc(p.w, (uint64_t)p.N * (uint64_t)steps * 64ull), rs = make_rsrc(p.scales, (uint64_t)p.N * (uint64_t)groups * 2ull),
                                     rz = make_rsrc(ZP ? p.zeros : p.w, (uint64_t)p.N * (uint64_t)groups / 2ull),
                                     ra = make_rsrc(static_cast<const uint16_t*>(p.a) + (uint64_t)m0 * (uint64_t)K, (uint64_t)M * (uint64_t)K * 2ull);
        uint32_t w_off[NWIN], s_off[NWIN];
#pragma unroll
        for (int w = 0; w < NWIN; w++) {
            // a lane reads row n of W, and scales of the four columns that it holds of C
            const int n = n_begin + w * 16 + li, c = n_begin + w * 16 + lg * 4;
            w_off[w] = n < n_end ? (uint32_t)(n >> 4) * (uint32_t)steps * 1024u + (uint32_t)(lg * 256 + (n & 15) * 16) : OOB;
            s_off[w] = c < n_end ? (uint32_t)(c >> 4) * (uint32_t)groups * 32u + (uint32_t)(c & 15) * 2u : OOB;
        }
        uint32_t a_off[MB];
#pragma unroll
        for (int mb = 0; mb < MB; mb++) a_off[mb] = mb * 16 + li < M ? (uint32_t)(mb * 16 + li) * (uint32_t)K * 2u + (uint32_t)lg * 16u : OOB;
        const int one = BF16 ? 0x3F803F80 : 0x3C003C00;
        const v4i ones = {one, one, one, one};

        for (int c0 = s0; c0 < s1; c0 += CH) {
            v4i a[CH][4][MB], w[CH][NWIN];
            v2i sc[CH][GPS][NWIN];
            uint32_t z[CH][GPS][NWIN];
#pragma unroll
            for (int t = 0; t < CH; t++)
#pragma unroll
                for (int j = 0; j < 4; j++)
#pragma unroll
                    for (int mb = 0; mb < MB; mb++) {
                        const int k = (c0 + t) * 128 + j * 32;
                        const bool in = c0 + t < s1 && k < K;  // (K is a multiple of 32)
                        a[t][j][mb] = buf_load16(ra, in ? a_off[mb] : OOB, in ? (uint32_t)k * 2u : 0u);
                    }
#pragma unroll
            for (int t = 0; t < CH; t++)
#pragma unroll
                for (int win = 0; win < NWIN; win++) {
                    const bool in = c0 + t < s1;
                    w[t][win] = buf_load16_nt(rw, in ? w_off[win] : OOB, in ? (uint32_t)(c0 + t) * 1024u : 0u);
#pragma unroll
                    for (int g = 0; g < GPS; g++) {
                        const int at = (c0 + t) * GPS + g;
                        const bool has = in && at < groups;
                        sc[t][g][win] = buf_load8(rs, has ? s_off[win] : OOB, has ? (uint32_t)at * 32u : 0u);
                        // (all zero points are less than 2^27 bytes: a quarter of OOB lies behind them too)
                        if constexpr (ZP) z[t][g][win] = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(rz, (int)(has ? s_off[win] >> 2 : OOB), has ? at * 8 : 0, 0);
                    }
                }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int t = 0; t < CH; t++)
#pragma unroll
                for (int g = 0; g < GPS; g++) {
                    v4f x[MB], pr[NWIN][MB];
#pragma unroll
                    for (int mb = 0; mb < MB; mb++) {
                        x[mb] = (v4f){0.f, 0.f, 0.f, 0.f};
#pragma unroll
                        for (int win = 0; win < NWIN; win++) pr[win][mb] = x[mb];
                    }
#pragma unroll
                    for (int j = g * MPG; j < (g + 1) * MPG; j++) {
#pragma unroll
                        for (int mb = 0; mb < MB; mb++) x[mb] = mfma16<BF16>(ones, a[t][j][mb], x[mb]);
#pragma unroll
                        for (int win = 0; win < NWIN; win++) {
                            const v4i b = widen<BF16>(w[t][win][j]);
#pragma unroll
                            for (int mb = 0; mb < MB; mb++) pr[win][mb] = mfma16<BF16>(b, a[t][j][mb], pr[win][mb]);
                        }
                    }
#pragma unroll
                    for (int win = 0; win < NWIN; win++)
#pragma unroll
                        for (int v = 0; v < 4; v++) {
                            const float s = from_out16<BF16 ? OUT_BF16 : OUT_FP16>((uint16_t)((uint32_t)sc[t][g][win][v >> 1] >> (16 * (v & 1))));
                            const float zc = ZP ? 16.0f + (float)((z[t][g][win] >> (4 * v)) & 15u) : 24.0f;
#pragma unroll
                            for (int mb = 0; mb < MB; mb++) acc[win][mb][v] = __builtin_fmaf(s, __builtin_fmaf(-zc, x[mb][v], pr[win][mb][v]), acc[win][mb][v]);
                        }
                }
        }
    }

    // the K slices' sums, in their order
#pragma unroll
    for (int w = 0; w < NWIN; w++)
#pragma unroll
        for (int mb = 0; mb < MB; mb++) part[wave][(w * MB + mb) * 64 + lane] = acc[w][mb];
    __syncthreads();
    for (int t = tid; t < gpw * NWIN * MB * 64; t += NWAVES * 64) {
        const int g = (t >> 6) / (NWIN * MB), frag = (t >> 6) % (NWIN * MB), gq = bid * gpw + g;
        const int m = (frag % MB) * 16 + li, n = (gq < p.groups ? unit_begin(gq) * 8 : 0) + (frag / MB) * 16 + lg * 4, ne = gq < p.groups ? unit_begin(gq + 1) * 8 : 0;
        if (n >= ne || m >= M) continue;
        v4f sum = part[g << ksh][frag * 64 + lane];
        for (int j = 1; j < p.ks; j++) sum += part[(g << ksh) + j][frag * 64 + lane];
        store_c4(p, (size_t)(m0 + m) * (size_t)p.N + (size_t)n, n, sum);
    }
}

template <bool BF16, int GS, bool ZP>
hipError_t launch(W4Params p, hipStream_t stream) {
    constexpr int NWAVES = 8, CH = 4;
    const int steps = (p.K + 127) / 128, mb = p.M > 16 ? 2 : 1, rows = (p.M + 31) / 32;
    int ks = NWAVES;
    while (ks > 1 && ks > steps) ks >>= 1;
    const int gpw = NWAVES / ks;
    const long units = p.N / 8, cus = psg_cu_count();
    const long rounds = (units + 4 * cus * gpw - 1) / (4 * cus * gpw);
    long tg = cus * gpw * rounds;
    if (tg > units) tg = units;
    p.ks = ks, p.groups = (int)tg, p.unit_q = (int)(units / tg), p.unit_r = (int)(units % tg);
    const bool two = (units + tg - 1) / tg > 2;
    const dim3 grid((unsigned)((tg + gpw - 1) / gpw), (unsigned)rows);
    if (mb == 1 && two) hipLaunchKernelGGL((k_w4a16<BF16, 1, 2, GS, ZP, NWAVES, CH>), grid, dim3(NWAVES * 64), 0, stream, p);
    else if (mb == 1) hipLaunchKernelGGL((k_w4a16<BF16, 1, 1, GS, ZP, NWAVES, CH>), grid, dim3(NWAVES * 64), 0, stream, p);
    else if (two) hipLaunchKernelGGL((k_w4a16<BF16, 2, 2, GS, ZP, NWAVES, 2>), grid, dim3(NWAVES * 64), 0, stream, p);
    else hipLaunchKernelGGL((k_w4a16<BF16, 2, 1, GS, ZP, NWAVES, 2>), grid, dim3(NWAVES * 64), 0, stream, p);
    return hipGetLastError();
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
