// Products of rows grouped by expert with the experts' own weights, C[r, :] = A[r, :] W[e(r)]^T (times scales), the groups' ends on the device (gfx950): tiles of 16, 32 and
// 64 rows, for groups of few rows.  (Tiles of 128 rows: gemm_pair.hip.)
//
// Four wavefronts side by side along N, each 16 NR columns wide; 128 bytes of K a step.  A tile of rows goes through registers to a two-stage LDS tile (rows of 128 bytes,
// 16-byte pieces XORed with row / 2), W fragments go straight from the group's preshuffled weight into the operand registers, both asked for three steps ahead.
// Bound: the weights' way from memory.  Every group's weight is read once by every tile of rows that it has.
#include "gemm_tiled.h"
#include "group_tiles.h"

namespace {

// NT: W past the caches
template <int KIND, int MR, int NR, bool NT>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(MR <= 2 ? 4 : 3))) k_grouped(A8W8Params p, GroupParams g) {
    using acc_t = typename Acc<KIND>::type;
    constexpr int BM = 16 * MR, TN = 64 * NR, SETS = 4;
    constexpr int A_LOADS = (BM * 8 + 255) / 256;  // 16-byte pieces of a step's A tile a thread
    constexpr bool SCALED = KIND == KIND_INT8 || KIND == KIND_FP8;
    __shared__ __attribute__((aligned(16))) uint8_t lds[2][BM * TK];
    const int tid = threadIdx.x, wave = wave_id(), lane = tid & 63, li = lane & 15, lg = lane >> 4;
    GroupTile t;
    if (!group_tile(g, p.M, BM, (int)blockIdx.x, (p.N + TN - 1) / TN, lane, t)) return;
    const int n0 = t.n_tile * TN;
    const uint32_t K = SCALED ? (uint32_t)p.K : (uint32_t)p.K * 2u;  // bytes of a row
    const int KT = (int)((K + TK - 1) / TK);

    // rows past the group's end and columns past N lie behind the descriptors' bounds or are redirected there, and read as zero
    const __amdgpu_buffer_rsrc_t ra = make_rsrc(p.a + (uint64_t)t.row * K, (uint64_t)(t.rows < BM ? t.rows : BM) * K);
    const __amdgpu_buffer_rsrc_t rb = make_rsrc(p.b + (uint64_t)t.e * (uint64_t)p.N * K, (uint64_t)p.N * K);
    uint32_t b_off[NR], a_off[A_LOADS];
    int a_lds[A_LOADS];
#pragma unroll
    for (int ni = 0; ni < NR; ni++) {
        const int n = n0 + (ni * 4 + wave) * 16;  // the wavefronts of pass ni cover 64 columns in a row
        b_off[ni] = n < p.N ? (uint32_t)n * K + (uint32_t)lane * 16u : OOB;
    }
    const int kc = tid & 7;
#pragma unroll
    for (int j = 0; j < A_LOADS; j++) {
        const int row = (tid >> 3) + 32 * j;
        a_off[j] = row < BM ? (uint32_t)row * K + (uint32_t)kc * 16u : OOB;
        a_lds[j] = row < BM ? lds_off(row, kc) : -1;
    }
    v4i ar[SETS][A_LOADS], wlo[SETS][NR], whi[SETS][NR];
    __builtin_assume(KT > 0);
    auto load_a = [&](int kt, int set) __attribute__((always_inline)) {
        const bool in = (uint32_t)kt * TK + (uint32_t)kc * 16u < K;  // (K ends on 64 bytes)
#pragma unroll
        for (int j = 0; j < A_LOADS; j++) ar[set][j] = buf_load16(ra, in ? a_off[j] : OOB, kt < KT ? (uint32_t)kt * TK : 0u);
    };
    auto load_w = [&](int kt, int set) __attribute__((always_inline)) {
        const bool lo = kt < KT, hi = (uint32_t)kt * TK + 64u < K;
#pragma unroll
        for (int ni = 0; ni < NR; ni++) {
            wlo[set][ni] = (v4i)__builtin_amdgcn_raw_buffer_load_b128(rb, (int)(lo ? b_off[ni] : OOB), lo ? kt * 2048 : 0, NT ? 2 : 0);
            whi[set][ni] = (v4i)__builtin_amdgcn_raw_buffer_load_b128(rb, (int)(hi ? b_off[ni] : OOB), hi ? kt * 2048 + 1024 : 0, NT ? 2 : 0);
        }
    };
    auto store_a = [&](int stage, int set) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < A_LOADS; j++)
            if (a_lds[j] >= 0) *reinterpret_cast<v4i*>(&lds[stage][a_lds[j]]) = ar[set][j];
    };
    acc_t acc[MR][NR];
#pragma unroll
    for (int mi = 0; mi < MR; mi++)
#pragma unroll
        for (int ni = 0; ni < NR; ni++) acc[mi][ni] = (acc_t){0, 0, 0, 0};
    auto step = [&](int kt, auto I) __attribute__((always_inline)) {
        constexpr int S = decltype(I)::value & 1, set = decltype(I)::value % SETS;
        load_a(kt + 3, (set + 3) % SETS);
        load_w(kt + 3, (set + 3) % SETS);
        // (addresses in front, MFMAs behind: one that writes a register has two wait states to the vector instruction that wrote it last)
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("s_nop 1");
#pragma unroll
        for (int mi = 0; mi < MR; mi++) {
            const v4i alo = *reinterpret_cast<const v4i*>(&lds[S][lds_off(mi * 16 + li, lg)]), ahi = *reinterpret_cast<const v4i*>(&lds[S][lds_off(mi * 16 + li, 4 + lg)]);
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
        __syncthreads();
    };

    static_for<3>([&](auto I) { load_w(decltype(I)::value, decltype(I)::value); });
    static_for<3>([&](auto I) { load_a(decltype(I)::value, decltype(I)::value); });
    // the scales of the lane's rows and columns, under the loop
    float sa[MR];
    v4f sb[NR];
    if constexpr (SCALED) {
#pragma unroll
        for (int mi = 0; mi < MR; mi++) sa[mi] = p.sa[t.row + (mi * 16 + li < t.rows ? mi * 16 + li : 0)];
#pragma unroll
        for (int ni = 0; ni < NR; ni++) {
            const int n = n0 + (ni * 4 + wave) * 16 + lg * 4;
            sb[ni] = *reinterpret_cast<const v4f*>(p.sb + (size_t)t.e * (size_t)p.N + (n < p.N ? n : 0));
        }
    }
    store_a(0, 0);
    __syncthreads();
    int kt = 0;
    for (; kt + SETS <= KT; kt += SETS) static_for<SETS>([&](auto I) { step(kt + decltype(I)::value, I); });
    static_for<SETS - 1>([&](auto I) {
        if (kt + decltype(I)::value < KT) step(kt + decltype(I)::value, I);
    });

    // C through LDS (both stages are free behind the last barrier), out as whole rows of the tile
    constexpr int ROWB = TN * 2, GR = ROWB / 16;
    static_assert(BM * ROWB <= (int)sizeof(lds), "the tile of C fits the A stages");
    uint8_t* const out = &lds[0][0];
#pragma unroll
    for (int mi = 0; mi < MR; mi++)
#pragma unroll
        for (int ni = 0; ni < NR; ni++) {
            const acc_t r = acc[mi][ni];
            v4f x = {(float)r[0], (float)r[1], (float)r[2], (float)r[3]};
            if constexpr (SCALED) x = (v4f){(x[0] * sa[mi]) * sb[ni][0], (x[1] * sa[mi]) * sb[ni][1], (x[2] * sa[mi]) * sb[ni][2], (x[3] * sa[mi]) * sb[ni][3]};
            const int row = mi * 16 + li, cb = ((ni * 4 + wave) * 16 + lg * 4) * 2;
            *reinterpret_cast<v2i*>(out + row * ROWB + ((((cb >> 4) ^ row) & (GR - 1)) << 4) + (cb & 15)) =
                p.out == OUT_BF16 ? pack4_out16<OUT_BF16>(x[0], x[1], x[2], x[3]) : pack4_out16<OUT_FP16>(x[0], x[1], x[2], x[3]);
        }
    __syncthreads();
    const int gr = tid & (GR - 1), n = n0 + gr * 8;
#pragma unroll
    for (int i = 0; i < (BM * GR + 255) / 256; i++) {
        const int row = tid / GR + i * (256 / GR);
        if (row < BM && row < t.rows && n < p.N)
            *reinterpret_cast<v4i*>(static_cast<uint16_t*>(p.c) + (size_t)(t.row + row) * (size_t)p.N + n) = *reinterpret_cast<const v4i*>(out + row * ROWB + (((gr ^ row) & (GR - 1)) << 4));
    }
}

template <int KIND, int MR>
hipError_t launch(const A8W8Params& p, GroupParams g, hipStream_t stream) {
    constexpr int NR = 2, TN = 64 * NR;
    g.most = (int)group_tiles_most(p.M, g.groups, 16 * MR);
    const dim3 grid((unsigned)g.most * (unsigned)((p.N + TN - 1) / TN));
    hipLaunchKernelGGL((k_grouped<KIND, MR, NR, false>), grid, dim3(256), 0, stream, p, g);
    return hipGetLastError();
}

template <int KIND>
hipError_t launch_kind(const A8W8Params& p, const GroupParams& g, int bm, hipStream_t stream) {
    switch (bm) {
        case 16: return launch<KIND, 1>(p, g, stream);
        case 32: return launch<KIND, 2>(p, g, stream);
        default: return launch<KIND, 4>(p, g, stream);
    }
}

}  // namespace

// Rows of a tile, by the rows that a group has on average
int psg_grouped_tile(int64_t rows, int groups) {
    const int64_t mean = (rows + groups - 1) / groups;
    return mean <= 16 ? 16 : mean <= 48 ? 32 : mean <= 96 ? 64 : 128;
}

// bm: 16, 32, 64 or 128 (psg_grouped_tile)
hipError_t psg_launch_grouped(const A8W8Params& p, const GroupParams& g, int kind, int bm, hipStream_t stream) {
    if (bm == 128) return psg_launch_grouped_pair(p, g, kind, stream);
    switch (kind) {
        case KIND_INT8: return launch_kind<KIND_INT8>(p, g, bm, stream);
        case KIND_FP8: return launch_kind<KIND_FP8>(p, g, bm, stream);
        case KIND_FP16: return launch_kind<KIND_FP16>(p, g, bm, stream);
        case KIND_BF16: return launch_kind<KIND_BF16>(p, g, bm, stream);
    }
    return hipErrorInvalidValue;
}
