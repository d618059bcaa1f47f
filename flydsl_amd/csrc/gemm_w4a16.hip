// A few rows of 16-bit activations times 4-bit weights with a 16-bit scale, and a zero point or none, per group of 32, 64 or 128 elements along K (gfx950).
//
//   C[m, n] = sum over the groups g of  s[n, g] (P[m, n, g] - z[n, g] X[m, g]),   P = sum over k in g of A[m, k] (16 + q[n, k]),   X = sum over k in g of A[m, k]
//
// with z = 16 + zero point (24 without zero points: codes 0..15 stand for -8..7).  A code q is made an operand of the matrix cores by two instructions for two of them: shifted to
// the upper bits of a mantissa, masked and joined with the exponent of 16 it is the 16-bit number 16 + q exactly, in bf16 as in fp16.  The 16 and the zero point come off the group's sum
// in fp32, and X of a lane's own row is what the same MFMA gives for a weight of ones.  (Both parts are at most 31 times the group's sum of |A|, of which an fp32 addition loses 2^-24; the terms
// A (q - z) are at most 8 times it, 15 with zero points: the 16 costs up to two bits, far below the 16-bit output's rounding but where terms of both signs cancel.)
//
// Bound: the weights' way from memory, and at a few MB of them the 3 us that a launch takes whatever it reads.  The columns are dealt out in units of 8, evenly, over one workgroup a CU;
// its eight wavefronts are eight slices of K.  A wavefront's part of A (SPW steps of 128 elements of the 16 rows) stays in registers while the workgroup's columns go by in windows of 16,
// the sums X of its groups too: what moves is W alone, the next window asked for as this one's registers become free, without a barrier.  The slices' sums meet in LDS in a fixed order:
// one launch, no workspace.  Rows too long for the registers take several passes over the columns; the next pass's part of A comes into LDS meanwhile, and W does not wait
// at their ends.
//   * A comes row by row, by DMA, only the rows there are: as fragments, 16 rows times 64 bytes an instruction and those of absent rows too, they took the address units longer than
//     the weights (16x6144x4096 8.1 us against 6.2, 1x2048x2048 5.0 / 3.4).
//   * A lane of every 16 reads the scales (and zero points) of one group for its four columns; the others take them from it by DPP.  One load a window instead of one a group (5x1040x2080,
//     groups of 32, 6.0 / 4.8).
//   * Reading A once and not once for every four units of columns: 16x28672x8192 58 -> 25, 5.0 TB/s.
//   Deeper prefetch (two windows), sixteen wavefronts and A read from LDS for every window were level or slower.
//
// Layout: W in blocks of 16 rows x 128 elements, 1 KB: lane l = 16 g + r of a wavefront reads 16 bytes, row r, dword j of them elements 32 j + 8 g .. + 7, what
// it multiplies in MFMA j; the even ones are the nibbles of the lower half of the dword, the odd ones those of the upper half, so that two of them are a mask away from a
// packed pair.  Rows end on whole blocks (elements past K are not looked at: A reads as zero there and X with it).  Scales [N/16][K/group][16], zero points the same as
// nibbles, lower one first: a lane's four columns are 8 and 2 bytes.
#include "gemm_w4a16.h"
#include "lds_dma.h"

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

// lane n of every 16
template <int N>
__device__ __forceinline__ int of_lane(int x) { return __builtin_amdgcn_update_dpp(0, x, 0x150 + N, 0xF, 0xF, true); }

// Row `row` of A times the four columns of W from n on, by all lanes of a wavefront: fp32 products with (q - z) s, which is exact (4 bits and a sign times 11), lanes eight elements of K each in turn.
template <bool BF16, int GS, bool ZP>
__device__ __forceinline__ v4f plain_sums(const W4Params& p, uint64_t row, int n, int steps, int groups, int lane) {
    constexpr int OUT = BF16 ? OUT_BF16 : OUT_FP16;
    const uint16_t* const a = static_cast<const uint16_t*>(p.a) + row * (uint64_t)p.K;
    v4f d = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
    for (int c = lane; c < p.K / 8; c += 64) {
        const v4i a8 = *reinterpret_cast<const v4i*>(a + (size_t)c * 8);
        const uint64_t g = (uint64_t)(n >> 4) * (uint64_t)groups + (uint64_t)(c * 8 / GS);
        // block, lane group and dword of these eight elements
        const uint8_t* const w = p.w + ((uint64_t)(n >> 4) * (uint64_t)steps + (uint64_t)(c >> 4)) * 1024u + (uint32_t)((c & 3) * 256 + ((c >> 2) & 3) * 4);
#pragma unroll
        for (int v = 0; v < 4; v++) {
            const int r = (n & 15) + v;
            const uint32_t q8 = *reinterpret_cast<const uint32_t*>(w + r * 16);
            const float s = from_out16<OUT>(p.scales[g * 16 + r]);
            const int z = ZP ? p.zeros[g * 8 + (r >> 1)] >> (4 * (r & 1)) & 15 : 8;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const int q = (int)(q8 >> (e & 1 ? 14 + 2 * e : 2 * e)) & 15;
                d[v] = __builtin_fmaf(from_out16<OUT>((uint16_t)((uint32_t)a8[e >> 1] >> (16 * (e & 1)))), (float)(q - z) * s, d[v]);
            }
        }
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1)
#pragma unroll
        for (int v = 0; v < 4; v++) d[v] += __shfl_xor(d[v], off, 64);
    return d;
}

constexpr int W4_WAVES = 8, W4_LDS = 160 * 1024;

// MB: 16-row blocks of A.  GS: elements of a group.  ZP: zero points.  SPW: 128-element steps of a wavefront's part of A.  SH: those that come through LDS at a time.  MANY: several
// passes.  ROWS: rows that the patch has room for, 16 MB, or less where M is not more.
template <bool BF16, int MB, int GS, bool ZP, int SPW, int SH, bool MANY, int ROWS>
__global__ void __launch_bounds__(W4_WAVES * 64, 2) k_w4a16(W4Params p) {
    constexpr int NW = W4_WAVES;
    constexpr int GPS = 128 / GS, MPG = GS / 32;              // groups of a step, MFMAs of a group
    constexpr int CPR = SH * 16, PATCH = ROWS * CPR * 16;  // 16-byte pieces of a staged row, bytes of a wavefront's patch
    static_assert(SPW * GPS <= 16, "a load of scales holds 16 groups");
    static_assert(ROWS > 16 * (MB - 1) && ROWS <= 16 * MB && PATCH % 1024 == 0, "rows of the patch, whole instructions of DMA");
    static_assert(!MANY || SH == SPW, "the next pass's part of A lies in the patch");
    __shared__ __attribute__((aligned(1024))) uint8_t lds[MANY ? W4_LDS : NW * PATCH];
    const int tid = threadIdx.x, wave = wave_id(), lane = tid & 63, li = lane & 15, lg = lane >> 4;
    auto unit_begin = [&](int g) { return g * p.unit_q + (g < p.unit_r ? g : p.unit_r); };
    // an XCD owns one range of columns: workgroups go round the XCDs
    const int wg = (gridDim.x & 7) == 0 ? (int)((blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3)) : (int)blockIdx.x;
    const int n_begin = unit_begin(wg) * 8, n_end = unit_begin(wg + 1) * 8, windows = (n_end - n_begin + 15) >> 4;
    const int m0 = (int)blockIdx.y * MB * 16, M = p.M - m0 < MB * 16 ? p.M - m0 : MB * 16, K = p.K, steps = (K + 127) >> 7, groups = K / GS;

    const __amdgpu_buffer_rsrc_t rw = make_rsrc(p.w, (uint64_t)p.N * (uint64_t)steps * 64ull), rs = make_rsrc(p.scales, (uint64_t)p.N * (uint64_t)groups * 2ull),
                                 rz = make_rsrc(ZP ? p.zeros : p.w, (uint64_t)p.N * (uint64_t)groups / 2ull),
                                 ra = make_rsrc_uniform(static_cast<const uint16_t*>(p.a) + (uint64_t)m0 * (uint64_t)K, (uint64_t)M * (uint64_t)K * 2ull);
    // a lane reads row n of W; of the scales it reads group li's for the four columns from c on that it holds of C; a window is 16 rows on
    const int n_lane = n_begin + li, c_lane = n_begin + lg * 4;
    const uint32_t w_lane = (uint32_t)(n_lane >> 4) * (uint32_t)steps * 1024u + (uint32_t)(lg * 256 + (n_lane & 15) * 16);
    const uint32_t s_lane = (uint32_t)(c_lane >> 4) * (uint32_t)groups * 32u + (uint32_t)(c_lane & 15) * 2u + (uint32_t)li * 32u;
    const Join<BF16 ? 0x00780078 : 0x03C003C0, BF16 ? 0x41804180 : 0x4C004C00> code;  // a code in the bits of the mantissa that count 1 to 8 beside 16
    const Join<0x00780000, 0x41800000> zero;                                           // the same in fp32
    uint8_t* const patch = lds + wave * PATCH;
    // [window][16-row block][lane], wavefronts `apart`: in the patch, free again once A is in registers, or beside it
    const int apart = MANY ? windows * MB * 64 : PATCH / 16;
    v4f* const all = reinterpret_cast<v4f*>(MANY ? lds + NW * PATCH : lds);
    auto first = [&](int pass) { return (pass * NW + wave) * p.per; };
    auto last = [&](int pass) { const int e = first(pass) + p.per; return e < steps ? e : steps; };

    v4i w[SPW];
    v2i sc;
    int z = 0;
    int l_pass = 0, l_win = 0;  // what is asked for next: windows on end, pass after pass
    auto load_w = [&](int t) __attribute__((always_inline)) {
        const int s = first(l_pass) + t;
        const bool in = (MANY ? l_pass < p.passes : l_win < windows) && s < last(l_pass);  // uniform
        w[t] = buf_load16_nt(rw, in && n_lane + l_win * 16 < n_end ? w_lane : OOB, in ? ((uint32_t)l_win * (uint32_t)steps + (uint32_t)s) * 1024u : 0u);
    };
    auto load_s = [&]() __attribute__((always_inline)) {
        const int at = first(l_pass) * GPS, e = last(l_pass) * GPS < groups ? last(l_pass) * GPS : groups;
        const bool in = MANY ? l_pass < p.passes : l_win < windows, has = in && at + li < e && c_lane + l_win * 16 < n_end;
        const uint32_t so = in ? (uint32_t)l_win * (uint32_t)groups + (uint32_t)at : 0u;
        sc = buf_load8(rs, has ? s_lane : OOB, so * 32u);
        // (all zero points are less than 2^27 bytes: a quarter of OOB lies behind them too)
        if constexpr (ZP) z = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(rz, (int)(has ? s_lane >> 2 : OOB), (int)(so * 8u), 0);
        l_win++;
        if (MANY && l_win == windows) l_win = 0, l_pass++;
    };
    // part of A, SH steps at a time: rows by DMA into the wavefront's patch (16-byte pieces XORed with the row), from there in fragments
    const int pieces = (M * CPR + 63) >> 6;
    auto stage = [&](int pass, int h) __attribute__((always_inline)) {
        const int k0 = (first(pass) + h * SH) * 128, ke = last(pass) * 128 < K ? last(pass) * 128 : K;
        for (int i = 0; i < pieces; i++) {
            const int q = i * 64 + lane, row = q / CPR, k = k0 + ((q % CPR) ^ (row & 15)) * 8;
            dma16(ra, (uint32_t)(uintptr_t)patch + (uint32_t)i * 1024u, row < M && k < ke ? (uint32_t)row * (uint32_t)K * 2u + (uint32_t)k * 2u : OOB, 0u);
        }
    };
    stage(0, 0);
#pragma unroll
    for (int t = 0; t < SPW; t++) load_w(t);
    load_s();
    __builtin_amdgcn_sched_barrier(0);

    for (int pass = 0; pass < (MANY ? p.passes : 1); pass++) {
        v4i a[SPW][4][MB];
        // the part has landed once only what was asked for behind it, a window of W at least, is on its way
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(SPW + (ZP ? 2 : 1)) : "memory");
#pragma unroll
        for (int h = 0; h < SPW / SH; h++) {
            if (h) {
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                stage(pass, h);
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            }
#pragma unroll
            for (int t = 0; t < SH; t++)
#pragma unroll
                for (int j = 0; j < 4; j++)
#pragma unroll
                    for (int mb = 0; mb < MB; mb++) {
                        const int r = mb * 16 + li < M ? mb * 16 + li : M - 1;  // (rows past M: any, they are not written)
                        a[h * SH + t][j][mb] = *reinterpret_cast<const v4i*>(patch + r * (CPR * 16) + (((t * 16 + j * 4 + lg) ^ (r & 15)) << 4));
                    }
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        if (MANY && pass + 1 < p.passes) stage(pass + 1, 0);

        // X of every group, times -24 without zero points
        float x[SPW][GPS][MB];
        const int one = BF16 ? (ZP ? 0x3F803F80 : (int)0xC1C0C1C0) : (ZP ? 0x3C003C00 : (int)0xCE00CE00);
        const v4i ones = {one, one, one, one};
#pragma unroll
        for (int t = 0; t < SPW; t++) {
            v4f y[GPS][MB];
#pragma unroll
            for (int g = 0; g < GPS; g++)
#pragma unroll
                for (int mb = 0; mb < MB; mb++) {
                    y[g][mb] = (v4f){0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int j = g * MPG; j < (g + 1) * MPG; j++) y[g][mb] = mfma16<BF16>(ones, a[t][j][mb], y[g][mb]);
                }
            // (all four rows of a result are the same; whole until they are there, so that no later MFMA's registers overlap one that is on its way)
#pragma unroll
            for (int g = 0; g < GPS; g++)
#pragma unroll
                for (int mb = 0; mb < MB; mb++) asm volatile("" : "+v"(y[g][mb]));
            asm volatile("s_nop 7");
#pragma unroll
            for (int g = 0; g < GPS; g++)
#pragma unroll
                for (int mb = 0; mb < MB; mb++) x[t][g][mb] = y[g][mb][0];
            __builtin_amdgcn_sched_barrier(0);
        }

        for (int win = 0; win < windows; win++) {
            v4f* const at = all + wave * apart + win * MB * 64 + lane;
            v4f acc[MB];
#pragma unroll
            for (int mb = 0; mb < MB; mb++) acc[mb] = MANY && pass ? at[mb * 64] : (v4f){0.f, 0.f, 0.f, 0.f};
            const v2i sc_ = sc;
            const int z_ = z;
            static_for<SPW>([&](auto T) {
                constexpr int t = decltype(T)::value;
                static_for<GPS>([&](auto G) {
                    constexpr int g = decltype(G)::value, q0 = t * GPS + g;
                    v4f pr[MB];
#pragma unroll
                    for (int mb = 0; mb < MB; mb++) pr[mb] = (v4f){0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int j = g * MPG; j < (g + 1) * MPG; j++) {
                        v4i b;
#pragma unroll
                        for (int q = 0; q < 4; q++) b[q] = code(shift(w[t][j], (BF16 ? 3 : 6) - 4 * q));
#pragma unroll
                        for (int mb = 0; mb < MB; mb++) pr[mb] = mfma16<BF16>(b, a[t][j][mb], pr[mb]);
                    }
                    const int s2[2] = {of_lane<q0>(sc_[0]), of_lane<q0>(sc_[1])};
                    const int z4 = ZP ? of_lane<q0>(z_) : 0;
#pragma unroll
                    for (int v = 0; v < 4; v++) {
                        const float s = from_out16<BF16 ? OUT_BF16 : OUT_FP16>((uint16_t)((uint32_t)s2[v >> 1] >> (16 * (v & 1))));
                        const float zc = ZP ? __builtin_bit_cast(float, zero(z4 << (19 - 4 * v))) : 0.f;
#pragma unroll
                        for (int mb = 0; mb < MB; mb++) acc[mb][v] = __builtin_fmaf(s, ZP ? __builtin_fmaf(-zc, x[t][g][mb], pr[mb][v]) : pr[mb][v] + x[t][g][mb], acc[mb][v]);
                    }
                });
                load_w(t);
                __builtin_amdgcn_sched_barrier(0);
            });
            load_s();
#pragma unroll
            for (int mb = 0; mb < MB; mb++) at[mb * 64] = acc[mb];
        }
    }

    __syncthreads();
    // the slices' sums, in their order
    for (int t = tid; t < windows * MB * 64; t += NW * 64) {
        const int frag = t >> 6, m = (frag % MB) * 16 + li, n = n_begin + (frag / MB) * 16 + lg * 4;
        const bool live = n < n_end && m < M;
        v4f sum = all[t];
#pragma unroll
        for (int j = 1; j < NW; j++) sum += all[j * apart + t];
        const size_t at = (size_t)(m0 + m) * (size_t)p.N + (size_t)n;
        if (live) store_c4(p, at, n, sum);
        // Sums that are not finite (all of a wavefront is here): P and 16 X meet as infinities where A has one, or where a group of finite rows passes fp32 by the 16 alone.  Such
        // values are taken and stored once more as the definition has them, the sum of A ((q - z) s), lanes along K: 16x28672x8192 25 us, with an infinity in one row 79, in all 780.  (Asking
        // costs 0.1 us a launch: 1x2048x2048 3.33 / 3.43, 16x28672x8192 level; in front of the stores 0.17.)
        const float mags = (fabsf(sum[0]) + fabsf(sum[1])) + (fabsf(sum[2]) + fabsf(sum[3]));
        for (uint64_t bad = __ballot(live && !(mags < __builtin_inff())); __builtin_expect(bad != 0, 0); bad &= bad - 1) {
            const int l = __builtin_ctzll(bad);
            const v4f d = plain_sums<BF16, GS, ZP>(p, (uint64_t)(m0 + __builtin_amdgcn_readlane(m, l)), __builtin_amdgcn_readlane(n, l), steps, groups, lane);
            if (lane == l) {
#pragma unroll
                for (int v = 0; v < 4; v++) sum[v] = fabsf(sum[v]) < __builtin_inff() ? sum[v] : d[v];
                store_c4(p, at, n, sum);
            }
        }
    }
}

// (ROWS below 16 MB: M <= ROWS)
template <bool BF16, int MB, int GS, bool ZP, int SPW, int SH, bool MANY, int ROWS = 16 * MB>
hipError_t go(W4Params p, hipStream_t stream) {
    const int steps = (p.K + 127) / 128;
    p.passes = (steps + W4_WAVES * SPW - 1) / (W4_WAVES * SPW);
    p.per = (steps + W4_WAVES * p.passes - 1) / (W4_WAVES * p.passes);
    // a workgroup has LDS for the sums of so many windows of 16 columns, which begin at a multiple of 8
    constexpr int PATCH = ROWS * SH * 256, windows = MANY ? (W4_LDS - W4_WAVES * PATCH) / (W4_WAVES * MB * 1024) : PATCH / (MB * 1024), most = 2 * windows;
    const long units = p.N / 8, cus = psg_cu_count(), rounds = (units + most * cus - 1) / (most * cus), wgs = units < cus * rounds ? units : cus * rounds;
    p.unit_q = (int)(units / wgs), p.unit_r = (int)(units % wgs);
    hipLaunchKernelGGL((k_w4a16<BF16, MB, GS, ZP, SPW, SH, MANY, ROWS>), dim3((unsigned)wgs, (unsigned)((p.M + MB * 16 - 1) / (MB * 16))), dim3(W4_WAVES * 64), 0, stream, p);
    return hipGetLastError();
}

// The steps of a wavefront's part of A are built to the number: a step too many is a window's MFMAs for nothing, at every window.  us with two or four for one or three / to the number:
// 1x28672x1024 7.6 / 5.9, 16x28672x2560 12.5 / 10.7, 4x4096x1024 3.3 / 3.1, 32x28672x1024 10.4 / 8.1, 8x18432x7168 19.3 / 16.4.
template <bool BF16, int GS, bool ZP>
hipError_t launch(const W4Params& p, hipStream_t stream) {
    const int per = ((p.K + 127) / 128 + W4_WAVES - 1) / W4_WAVES;  // steps of a wavefront
    const int64_t cus = psg_cu_count();
    // 17 to 32 rows read W once: where A fits the registers, 16 rows at a time / like this, 32x7168x2048 8.1 / 5.9, 32x4096x4096 8.6 / 6.8
    if (p.M > 16) {
        if (per == 1) return go<BF16, 2, GS, ZP, 1, 1, false>(p, stream);
        if (per == 2) return go<BF16, 2, GS, ZP, 2, 2, false>(p, stream);
        // of up to 24 rows three steps come through LDS at once, 24x2048x2560 in halves / like this 6.1 / 5.1, 20x6144x2560 in groups of 64 in passes / like this 7.8 / 6.4, 20x4096x2880 of 32 6.6 / 5.4;
        // four in halves, in groups of 64 in passes / like this 28x28672x4096 27.5 / 17.7, 28x8192x4096 8.7 / 8.3
        if constexpr (GS > 32 || !ZP) {
            if (per == 3 && p.M <= 24) return go<BF16, 2, GS, ZP, 3, 3, false, 24>(p, stream);
        }
        if constexpr (GS == 128 || (GS == 64 && !ZP)) {
            if (per <= 4) return go<BF16, 2, GS, ZP, 4, 2, false>(p, stream);
        }
        // longer rows in passes of two steps, which leave LDS for two windows a workgroup, 16 rows at a time / like this 32x8192x8192 22.9 / 16.0, 17x8192x5120 15.5 / 10.3, of up to 24 rows for four, passes of
        // one / of two 24x12288x6144 19.4 / 14.9, 17x16384x8192 28.1 / 22.9; or of one, for six, 16 rows at a time / of one 32x14336x4096 in groups of 32 20.2 / 16.6 (of two 18.7).  With still more columns 16 rows
        // at a time are level or better (32x28672x8192 47.7 / 55.8).
        if (p.N <= 32 * cus) return go<BF16, 2, GS, ZP, 2, 2, true>(p, stream);
        if (p.M <= 24 && p.N <= 64 * cus) return go<BF16, 2, GS, ZP, 2, 2, true, 24>(p, stream);
        if (p.N <= 96 * cus) return go<BF16, 2, GS, ZP, 1, 1, true>(p, stream);
    }
    if (per == 1) return go<BF16, 1, GS, ZP, 1, 1, false>(p, stream);
    if (per == 2) return go<BF16, 1, GS, ZP, 2, 2, false>(p, stream);
    if (per == 3) return go<BF16, 1, GS, ZP, 3, 3, false>(p, stream);
    if (per == 4) return go<BF16, 1, GS, ZP, 4, 4, false>(p, stream);
    // Five to eight steps in one pass, where the sums of their groups fit beside them: five come through LDS at once, of up to eight rows all of them, else three or four and again as many.  us in
    // passes of two / in halves / at once: 1x5120x5120 7.8 / 6.9 / 5.9, 16x13824x5120 13.5 / 11.5 / 10.3, 4x5120x6144 in groups of 64 8.4 / 8.1 / 7.4; 1x4096x7168 - / 6.2 / 5.6.  (Eight with 16 groups' sums spill: 4x5120x6144
    // in groups of 64 29; long rows of eight rows in passes of six or eight were level or spilled.)
    if constexpr (GS >= 64) {
        if (per == 5) return go<BF16, 1, GS, ZP, 5, 5, false>(p, stream);
        if (per == 6 && p.M <= 8) return go<BF16, 1, GS, ZP, 6, 6, false, 8>(p, stream);
        if (per == 6) return go<BF16, 1, GS, ZP, 6, 3, false>(p, stream);
    }
    if constexpr (GS == 128) {
        if (per == 7 && p.M <= 8) return go<BF16, 1, GS, ZP, 7, 7, false, 8>(p, stream);
        if (per == 8 && p.M <= 8) return go<BF16, 1, GS, ZP, 8, 8, false, 8>(p, stream);
        if (per <= 8) return go<BF16, 1, GS, ZP, 8, 4, false>(p, stream);
    }
    // Longer rows in as few passes of up to four steps as there are, which leave LDS for four windows a workgroup, three steps where that is what the passes come to or for eight windows, two for twelve.  us four / three:
    // 1x8192x9216 10.5 / 9.3, 16x20480x9216 27.5 / 23.5, 13x1536x8256 in groups of 32 10.3 / 8.7; two / three 3x18432x13824 32.4 / 28.7, 16x17408x16384 42.7 / 37.9, 16x13824x5120 in groups of 32 with zero
    // points 18.0 / 17.3; four / two 16x12288x7168 13.1 / 14.5, 9x3584x18944 12.8 / 14.4, 1x8192x28672 23.3 / 27.3; but groups of 32 with zero points, whose four steps take all registers, 2x8192x10240 16.9 / 14.9
    // (three 17.1).
    const int passes = (per + 3) / 4, each = (per + passes - 1) / passes;
    const bool all_registers = GS == 32 && ZP, wide = p.N > 64 * cus;
    if ((each == 3 || (wide && !all_registers)) && p.N <= 128 * cus) return go<BF16, 1, GS, ZP, 3, 3, true>(p, stream);
    if (wide || all_registers) return go<BF16, 1, GS, ZP, 2, 2, true>(p, stream);
    return go<BF16, 1, GS, ZP, 4, 4, true>(p, stream);
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
