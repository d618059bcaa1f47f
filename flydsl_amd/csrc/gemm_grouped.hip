// Products of rows grouped by expert with the experts' own weights, C[r, :] = A[r, :] W[e(r)]^T (times scales), the groups' ends on the device (gfx950): tiles of 16, 32 and
// 64 rows, for groups of few rows.  (Tiles of 128 rows: gemm_pair.hip.)
//
// Four wavefronts side by side along N, each 16 NR columns wide, or four slices of K for the same columns, whose sums meet in LDS; 128 bytes of K a step and slice.  A tile of rows goes through
// registers to a two-stage LDS tile (rows of 128 bytes, 16-byte pieces XORed with row / 2), W fragments go straight from the group's preshuffled weight into the operand registers,
// both asked for three steps ahead.
// Bound: the weights' way from memory, every group's read once by every tile of rows that it has (442 MB of 32 experts at 6.3 TB/s); with few tiles the steps' latency.
#include "gemm_tiled.h"
#include "group_tiles.h"

namespace {

// With block scales (KIND_FP8B) an MFMA's sum is scaled and added a step later, under the next step's MFMAs; the scales of a step stand in LDS beside A: 512 rows on 32 groups, 3584 x 4096, 75.1 us, 5.9 TB/s
// (one scale a row 74.6).  Its 64-row tile has 180 registers and two wavefronts a SIMD; for three it would spill.
// KS: K slices, 1 or 4: with four, the wavefronts have the same 16 NR columns and every fourth step each.  NT: W past the caches.
template <int KIND, int MR, int NR, int KS, bool NT>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(MR <= 2 ? 4 : KIND == KIND_FP8B ? 2 : 3))) k_grouped(A8W8Params p, GroupParams g) {
    using acc_t = typename Acc<KIND>::type;
    constexpr int BM = 16 * MR, CB = 4 / KS, TN = 16 * CB * NR, SETS = 4;  // (CB: column blocks side by side)
    constexpr int TILE = BM * TK;                                          // bytes of A a step; a stage holds KS of them
    constexpr int A_LOADS = (KS * BM * 8 + 255) / 256;                     // 16-byte pieces of a stage a thread
    constexpr bool SCALED = KIND == KIND_INT8 || KIND == KIND_FP8, BLOCKED = KIND == KIND_FP8B;
    constexpr int ROWB = TN * 2, GR = ROWB / 16;                           // bytes and 16-byte granules of a row of the tile of C
    constexpr int SUMS = KS > 1 ? 4 * MR * NR * 1024 : 0;
    __shared__ __attribute__((aligned(16))) uint8_t lds[2 * KS * TILE > SUMS ? 2 * KS * TILE : SUMS];
    __shared__ float s_scale[BLOCKED ? 2 * BM : 1];  // a stage's products of row and column scale
    const int tid = threadIdx.x, wave = wave_id(), lane = tid & 63, li = lane & 15, lg = lane >> 4;
    const int slice = KS > 1 ? wave : 0, block = KS > 1 ? 0 : wave;
    GroupTile t;
    if (!group_tile<BLOCKED>(g, p.M, BM, (int)blockIdx.x, (p.N + TN - 1) / TN, lane, t)) return;
    const int n0 = t.n_tile * TN;
    const uint32_t K = SCALED || BLOCKED ? (uint32_t)p.K : (uint32_t)p.K * 2u;  // bytes of a row
    const int KT = (int)((K + KS * TK - 1) / (KS * TK));

    // rows past the group's end and columns past N lie behind the descriptors' bounds or are redirected there, and read as zero
    const __amdgpu_buffer_rsrc_t ra = make_rsrc(p.a + (uint64_t)t.row * K, (uint64_t)(t.rows < BM ? t.rows : BM) * K);
    const __amdgpu_buffer_rsrc_t rb = make_rsrc(p.b + (uint64_t)t.e * (uint64_t)p.N * K, (uint64_t)p.N * K);
    uint32_t b_off[NR], a_off[A_LOADS];
    int a_lds[A_LOADS], a_k[A_LOADS];
#pragma unroll
    for (int ni = 0; ni < NR; ni++) {
        const int n = n0 + (ni * CB + block) * 16;  // the wavefronts of pass ni cover 16 CB columns in a row
        b_off[ni] = n < p.N ? (uint32_t)n * K + (uint32_t)lane * 16u : OOB;
    }
#pragma unroll
    for (int j = 0; j < A_LOADS; j++) {
        const int q = tid + 256 * j, sub = q / (BM * 8), row = q / 8 % BM, kc = q & 7;
        a_k[j] = sub * TK + kc * 16;
        a_off[j] = sub < KS ? (uint32_t)row * K + (uint32_t)a_k[j] : OOB;
        a_lds[j] = sub < KS ? sub * TILE + lds_off(row, kc) : -1;
    }
    v4i ar[SETS][A_LOADS], wlo[SETS][NR], whi[SETS][NR];
    // block scales of a stage: a row a thread, and that of the tile's columns, which lie in one block (rows past the group's end have others' scales, and zeros behind the array)
    static_assert(!BLOCKED || (KS == 1 && BM <= 64), "the scales of a stage are a wavefront's; K in slices is gemm_blockscale.hip's");
    float sar[SETS], sbr[SETS];
    const uint32_t KB = (K + TK - 1) / TK, NB = ((uint32_t)p.N + 127u) / 128u;
    const __amdgpu_buffer_rsrc_t rsa = make_rsrc(BLOCKED ? p.sa + t.row : nullptr, BLOCKED ? ((uint64_t)(KB - 1) * g.sa_stride + (uint32_t)(p.M - t.row)) * 4ull : 0ull);
    const __amdgpu_buffer_rsrc_t rsb = make_rsrc(BLOCKED ? p.sb + ((uint64_t)t.e * NB + (uint32_t)n0 / 128u) * KB : nullptr, BLOCKED ? KB * 4ull : 0ull);
    auto load_s = [&](int kt, int set) __attribute__((always_inline)) {
        if constexpr (BLOCKED) {
            const bool has = tid < BM && kt < KT;
            sar[set] = __int_as_float(buf_load4(rsa, has ? (uint32_t)tid * 4u : OOB, kt < KT ? (uint32_t)kt * 4u * g.sa_stride : 0u));
            sbr[set] = __int_as_float(buf_load4(rsb, has ? 0u : OOB, kt < KT ? (uint32_t)kt * 4u : 0u));
        }
    };
    auto store_s = [&](int stage, int set) __attribute__((always_inline)) {
        if constexpr (BLOCKED) {
            if (tid < BM) s_scale[stage * BM + tid] = sar[set] * sbr[set];
        }
    };
    __builtin_assume(KT > 0);
    auto load_a = [&](int kt, int set) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < A_LOADS; j++) ar[set][j] = buf_load16(ra, (uint32_t)kt * (KS * TK) + (uint32_t)a_k[j] < K ? a_off[j] : OOB, kt < KT ? (uint32_t)kt * (KS * TK) : 0u);  // (K ends on 64 bytes)
    };
    auto load_w = [&](int kt, int set) __attribute__((always_inline)) {
        const uint32_t s = (uint32_t)(kt * KS + slice);
        const bool lo = s * TK < K, hi = s * TK + 64u < K;
#pragma unroll
        for (int ni = 0; ni < NR; ni++) {
            wlo[set][ni] = (v4i)__builtin_amdgcn_raw_buffer_load_b128(rb, (int)(lo ? b_off[ni] : OOB), lo ? (int)(s * 2048u) : 0, NT ? 2 : 0);
            whi[set][ni] = (v4i)__builtin_amdgcn_raw_buffer_load_b128(rb, (int)(hi ? b_off[ni] : OOB), hi ? (int)(s * 2048u + 1024u) : 0, NT ? 2 : 0);
        }
    };
    auto store_a = [&](int stage, int set) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < A_LOADS; j++)
            if (a_lds[j] >= 0) *reinterpret_cast<v4i*>(&lds[stage * KS * TILE + a_lds[j]]) = ar[set][j];
    };
    acc_t acc[MR][NR];
#pragma unroll
    for (int mi = 0; mi < MR; mi++)
#pragma unroll
        for (int ni = 0; ni < NR; ni++) acc[mi][ni] = (acc_t){0, 0, 0, 0};
    // Block scales: what the last BEHIND MFMAs gave, added into the blocks' sums BEHIND MFMAs later, where it is there without a wait (that of a step's last ones in the next step).
    constexpr int BEHIND = MR * NR < 2 ? MR * NR : 2, SCALES = BEHIND / NR + 1 < MR ? BEHIND / NR + 1 : MR;
    v4f part[BEHIND] = {};
    float part_scale[SCALES] = {};
    auto add_part = [&](auto I) __attribute__((always_inline)) {
        if constexpr (BLOCKED) {
            constexpr int i = decltype(I)::value, mi = i / NR, ni = i % NR;
#pragma unroll
            for (int j = 0; j < 4; j++) acc[mi][ni][j] = __builtin_fmaf(part[i % BEHIND][j], part_scale[mi % SCALES], acc[mi][ni][j]);
            // (here, and not where the sums are used in the end: the compiler takes the additions of four steps behind the last branch and keeps what the MFMAs gave until then)
            asm volatile("" : "+v"(acc[mi][ni]));
        }
    };
    auto step = [&](int kt, auto I) __attribute__((always_inline)) {
        constexpr int S = decltype(I)::value & 1, set = decltype(I)::value % SETS;
        load_a(kt + 3, (set + 3) % SETS);
        load_s(kt + 3, (set + 3) % SETS);  // (in front of W, or the wait for the scales would be one for the W that is not due yet)
        load_w(kt + 3, (set + 3) % SETS);
        // (addresses in front, MFMAs behind: one that writes a register has two wait states to the vector instruction that wrote it last)
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("s_nop 1");
        const uint8_t* const mine = lds + (S * KS + slice) * TILE;
        if constexpr (BLOCKED) {
            // a step is a block: its products' sums by MFMAs that begin with zero, then times both scales into the sums of the blocks, behind the next MFMA
            v4i alo[2], ahi[2];
            static_for<MR * NR>([&](auto I) {
                constexpr int i = decltype(I)::value, mi = i / NR, ni = i % NR;
                if constexpr (ni == 0) alo[mi & 1] = *reinterpret_cast<const v4i*>(mine + lds_off(mi * 16 + li, lg)), ahi[mi & 1] = *reinterpret_cast<const v4i*>(mine + lds_off(mi * 16 + li, 4 + lg));
                add_part(std::integral_constant<int, (i + MR * NR - BEHIND) % (MR * NR)>{});
                if constexpr (ni == 0) part_scale[mi % SCALES] = s_scale[S * BM + mi * 16 + li];
                part[i % BEHIND] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(__builtin_shufflevector(wlo[set][ni], whi[set][ni], 0, 1, 2, 3, 4, 5, 6, 7),
                                                                                    __builtin_shufflevector(alo[mi & 1], ahi[mi & 1], 0, 1, 2, 3, 4, 5, 6, 7), (v4f){0.f, 0.f, 0.f, 0.f}, 0, 0, 0, 0, 0, 0);
            });
        }
#pragma unroll
        for (int mi = 0; mi < (BLOCKED ? 0 : MR); mi++) {
            const v4i alo = *reinterpret_cast<const v4i*>(mine + lds_off(mi * 16 + li, lg)), ahi = *reinterpret_cast<const v4i*>(mine + lds_off(mi * 16 + li, 4 + lg));
#pragma unroll
            for (int ni = 0; ni < NR; ni++) {
                const v4i b0 = wlo[set][ni], b1 = whi[set][ni];
                if constexpr (KIND == KIND_INT8) {
                    acc[mi][ni] = __builtin_amdgcn_mfma_i32_16x16x64_i8(b0, alo, acc[mi][ni], 0, 0, 0);
                    acc[mi][ni] = __builtin_amdgcn_mfma_i32_16x16x64_i8(b1, ahi, acc[mi][ni], 0, 0, 0);
                } else if constexpr (KIND == KIND_FP8) {
                    acc[mi][ni] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(__builtin_shufflevector(b0, b1, 0, 1, 2, 3, 4, 5, 6, 7), __builtin_shufflevector(alo, ahi, 0, 1, 2, 3, 4, 5, 6, 7),
                                                                                   acc[mi][ni], 0, 0, 0, 0, 0, 0);
                } else if constexpr (KIND == KIND_BF16) {
                    acc[mi][ni] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, b0), __builtin_bit_cast(v8bf, alo), acc[mi][ni], 0, 0, 0);
                    acc[mi][ni] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, b1), __builtin_bit_cast(v8bf, ahi), acc[mi][ni], 0, 0, 0);
                } else {
                    acc[mi][ni] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, b0), __builtin_bit_cast(v8h, alo), acc[mi][ni], 0, 0, 0);
                    acc[mi][ni] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, b1), __builtin_bit_cast(v8h, ahi), acc[mi][ni], 0, 0, 0);
                }
            }
        }
        store_a(S ^ 1, (set + 1) % SETS);
        store_s(S ^ 1, (set + 1) % SETS);
        __syncthreads();
    };

    static_for<3>([&](auto I) { load_w(decltype(I)::value, decltype(I)::value); });
    static_for<3>([&](auto I) { load_a(decltype(I)::value, decltype(I)::value); });
    static_for<3>([&](auto I) { load_s(decltype(I)::value, decltype(I)::value); });
    // the scales of the lane's rows and columns, under the loop
    float sa[MR];
    v4f sb[NR];
    if constexpr (SCALED) {
#pragma unroll
        for (int mi = 0; mi < MR; mi++) sa[mi] = p.sa[t.row + (mi * 16 + li < t.rows ? mi * 16 + li : 0)];
#pragma unroll
        for (int ni = 0; ni < NR; ni++) {
            const int n = n0 + (ni * CB + block) * 16 + lg * 4;
            sb[ni] = *reinterpret_cast<const v4f*>(p.sb + (size_t)t.e * (size_t)p.N + (n < p.N ? n : 0));
        }
    }
    store_a(0, 0);
    store_s(0, 0);
    __syncthreads();
    int kt = 0;
    for (; kt + SETS <= KT; kt += SETS) static_for<SETS>([&](auto I) { step(kt + decltype(I)::value, I); });
    static_for<SETS - 1>([&](auto I) {
        if (kt + decltype(I)::value < KT) step(kt + decltype(I)::value, I);
    });

    static_for<BEHIND>([&](auto I) { add_part(std::integral_constant<int, MR * NR - BEHIND + decltype(I)::value>{}); });

    auto finish = [&](acc_t r, int mi, int ni) __attribute__((always_inline)) {
        v4f x = {(float)r[0], (float)r[1], (float)r[2], (float)r[3]};
        if constexpr (SCALED) x = (v4f){(x[0] * sa[mi]) * sb[ni][0], (x[1] * sa[mi]) * sb[ni][1], (x[2] * sa[mi]) * sb[ni][2], (x[3] * sa[mi]) * sb[ni][3]};
        return p.out == OUT_BF16 ? pack4_out16<OUT_BF16>(x[0], x[1], x[2], x[3]) : pack4_out16<OUT_FP16>(x[0], x[1], x[2], x[3]);
    };
    if constexpr (KS > 1) {
        // the slices' sums through LDS (free behind the last barrier), added in their order, a fragment a wavefront; out 8 bytes a lane
        acc_t* const sums = reinterpret_cast<acc_t*>(lds);
#pragma unroll
        for (int mi = 0; mi < MR; mi++)
#pragma unroll
            for (int ni = 0; ni < NR; ni++) sums[((mi * NR + ni) * 4 + wave) * 64 + lane] = acc[mi][ni];
        __syncthreads();
#pragma unroll
        for (int f = 0; f < MR * NR; f++) {
            if (f % 4 != wave) continue;
            acc_t r = sums[f * 256 + lane];
#pragma unroll
            for (int j = 1; j < 4; j++) r += sums[(f * 4 + j) * 64 + lane];
            const int row = f / NR * 16 + li, n = n0 + f % NR * 16 + lg * 4;
            if (row < t.rows && n < p.N) *reinterpret_cast<v2i*>(static_cast<uint16_t*>(p.c) + (size_t)(t.row + row) * (size_t)p.N + n) = finish(r, f / NR, f % NR);
        }
    } else {
        // C through LDS (both stages are free behind the last barrier), out as whole rows of the tile
        static_assert(KS > 1 || BM * ROWB <= (int)sizeof(lds), "the tile of C fits the A stages");
#pragma unroll
        for (int mi = 0; mi < MR; mi++)
#pragma unroll
            for (int ni = 0; ni < NR; ni++) {
                const int row = mi * 16 + li, cb = ((ni * CB + block) * 16 + lg * 4) * 2;
                *reinterpret_cast<v2i*>(lds + row * ROWB + ((((cb >> 4) ^ row) & (GR - 1)) << 4) + (cb & 15)) = finish(acc[mi][ni], mi, ni);
            }
        __syncthreads();
        const int gr = tid & (GR - 1), n = n0 + gr * 8;
#pragma unroll
        for (int i = 0; i < (BM * GR + 255) / 256; i++) {
            const int row = tid / GR + i * (256 / GR);
            if (row < BM && row < t.rows && n < p.N)
                *reinterpret_cast<v4i*>(static_cast<uint16_t*>(p.c) + (size_t)(t.row + row) * (size_t)p.N + n) = *reinterpret_cast<const v4i*>(lds + row * ROWB + (((gr ^ row) & (GR - 1)) << 4));
        }
    }
}

template <int KIND, int MR, int NR, int KS, bool NT>
hipError_t launch(const A8W8Params& p, GroupParams g, hipStream_t stream) {
    constexpr int TN = 64 / KS * NR;
    g.most = (int)group_tiles_most(p.M, g.groups, 16 * MR);
    hipLaunchKernelGGL((k_grouped<KIND, MR, NR, KS, NT>), dim3((unsigned)g.most * (unsigned)((p.N + TN - 1) / TN)), dim3(256), 0, stream, p, g);
    return hipGetLastError();
}

// Whether W goes past the caches: where most groups are one tile, so that little is read twice, and two such products, as a layer has them at least, have more weights than the last-level
// cache (256 MB).  us through the caches / past them, fp8, 3584 x 4096 on 32 experts, by the rows that a group has for every row of its tile: tiles of 16, 1/2 83.8 / 77.8, 3/4 85.1 / 84.2, 1 90.3 / 96.2,
// 3/2 101 / 124; of 32, 1/2 86.2 / 81.1, 3/4 91.8 / 91.3, 1 97.5 / 107; of 64, 1/2 92.0 / 87.2, 3/4 101.4 / 102.0, 1 106 / 118; as many on fewer experts, W of 84 MB 16.6 / 18.3, 112 20.3 / 20.9, 140 27.5 / 27.3,
// 168 33.6 / 31.4; int8 2048 x 768 on 128, 2048 rows 45.8 / 40.9, 4200 49.9 / 45.5; bf16 2048 x 2048 on 64, 256 rows 99.8 / 91.0, 1100 107.4 / 99.6.
bool goes_past(const A8W8Params& p, const GroupParams& g, int bm, int bytes) {
    return 2ll * g.groups * p.N * p.K * bytes > 256ll << 20 && 4ll * p.M <= 3ll * bm * g.groups;
}

template <int KIND>
hipError_t launch_kind(const A8W8Params& p, const GroupParams& g, GroupedPlan plan, hipStream_t stream) {
    const bool past = goes_past(p, g, plan.bm, KIND == KIND_INT8 || KIND == KIND_FP8 || KIND == KIND_FP8B ? 1 : 2);
    switch (plan.bm) {
        case 16:
            if constexpr (KIND != KIND_FP8B) {  // (whose slices are in gemm_blockscale.hip)
                if (plan.sliced) return launch<KIND, 1, 1, 4, false>(p, g, stream);
            }
            return past ? launch<KIND, 1, 1, 1, true>(p, g, stream) : launch<KIND, 1, 1, 1, false>(p, g, stream);
        case 32: return past ? launch<KIND, 2, 1, 1, true>(p, g, stream) : launch<KIND, 2, 1, 1, false>(p, g, stream);
        default: return past ? launch<KIND, 4, 2, 1, true>(p, g, stream) : launch<KIND, 4, 2, 1, false>(p, g, stream);
    }
}

}  // namespace

// The tile, by its estimated time.  A step of K takes a workgroup that is alone on its CU `alone` us, and a CU `busy` us for every tile where it has many (fitted to 1 x 512 x 8192 bf16 with 40 rows and to
// 32768 rows on 32 experts, 4096 x 1536, fp8); the groups' last tiles are half empty on average.  Reading the weights takes every tile as long (5.3 TB/s).  Of the tiles that are within
// a tenth of the best, the largest that a group's rows fill: a group's weight is then read once.  Tiles of 16 rows with K in slices where that saves a quarter.  us, tiles of 16 in slices / 16 /
// 32 / 64 / 128 rows: bf16 40 rows on 1, 512 x 8192, 10.0 / 23.8 / 27.1 / 45 / 66, 300 on 4, 4096 x 2048, - / 24.8 / 18.8 / 17.0 / 21.9, 1500 on 17, 2816 x 1088, - / 47 / 38 / 33 / 28.6; fp8 16 on
// 1, 4096 x 4096, 7.0 / 8.3 / 9.0 / 16 / 24, 512 on 32, 3584 x 4096, 114 / 86 / 75 / 78 / 82; int8 4096 on 128, 2048 x 768, - / 63 / 51 / 44 / 51.
GroupedPlan psg_grouped_plan(int64_t rows, int groups, int N, int64_t kbytes) {
    struct Tile { int bm, tn; double alone, busy; };
    static constexpr Tile tiles[4] = {{16, 64, 0.186, 0.118}, {32, 64, 0.21, 0.146}, {64, 128, 0.35, 0.408}, {128, 256, 0.51, 1.137}};
    const double cus = psg_cu_count(), live = (double)(groups < rows ? groups : rows), steps = (double)((kbytes + TK - 1) / TK), weights = live * N * (double)kbytes / 5.3e6, mean = rows / live;
    auto estimate = [&](int bm, int tn, double n, double alone, double busy) {
        const double load = (rows / (double)bm + 0.5 * live) * ((N + tn - 1) / tn) * busy / cus;
        return n * (load > alone ? load : alone);
    };
    double t[4], best = 1e30;
    for (int i = 0; i < 4; i++) {
        const double e = estimate(tiles[i].bm, tiles[i].tn, steps, tiles[i].alone, tiles[i].busy);
        t[i] = e > weights ? e : weights;
        best = t[i] < best ? t[i] : best;
    }
    const double sliced = estimate(16, 16, (double)((kbytes + 4 * TK - 1) / (4 * TK)), 0.2, 0.346), whole = estimate(16, 64, steps, tiles[0].alone, tiles[0].busy);
    if (t[0] <= 1.1 * best && sliced < 0.75 * whole) return {16, true};
    const int fill = mean <= 8 ? 0 : mean <= 24 ? 1 : mean <= 48 ? 2 : 3;
    for (int i = fill; i > 0; i--)
        if (t[i] <= 1.1 * best) return {tiles[i].bm, false};
    return {16, false};
}

hipError_t psg_launch_grouped(const A8W8Params& p, const GroupParams& g, int kind, GroupedPlan plan, hipStream_t stream) {
    if (plan.bm == 128) return psg_launch_grouped_pair(p, g, kind, stream);
    switch (kind) {
        case KIND_INT8: return launch_kind<KIND_INT8>(p, g, plan, stream);
        case KIND_FP8: return launch_kind<KIND_FP8>(p, g, plan, stream);
        case KIND_FP8B: return launch_kind<KIND_FP8B>(p, g, plan, stream);
        case KIND_FP16: return launch_kind<KIND_FP16>(p, g, plan, stream);
        case KIND_BF16: return launch_kind<KIND_BF16>(p, g, plan, stream);
    }
    return hipErrorInvalidValue;
}
