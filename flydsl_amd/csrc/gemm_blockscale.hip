// Block-scaled fp8 products of few tiles (gfx950): C[r, n] = sum over blocks b of 128 along K of sa[b, r] sb[n / 128, b] (A[r, b] W[n, b]^T), by tiles of 16 to 64 rows whose K is cut into eight slices; and which way such a product takes.
// (Few rows: gemm_a8w8_stream.hip.  Many tiles: gemm_grouped.hip, gemm_pair.hip, and the 128 x 128 tile of gemm_tiled8.h, which is built here.)
//
// With about a tile for every CU what counts is how soon its operands are there: a step of 128 bytes of K takes a workgroup that goes from step to step together a memory latency, whatever it
// multiplies.  Here the eight wavefronts of a workgroup have the same tile and every eighth step each, and nothing to do with each other until their sums meet in LDS: a wavefront asks for all of its
// step (A, W and the scales) by DMA into a piece of LDS of its own, waits, takes the fragments into registers, asks for its next step in their place and multiplies meanwhile.  That keeps 16 KB a
// wavefront on their way for tiles of 64 x 64, 128 KB a CU, without a barrier, without a register for what is on its way and with one wait that counts nothing.
// The order of the sums: a slice's blocks in theirs, then the slices in theirs.
// Bound: a CU's way to L2, 64 bytes a cycle.
#include <cmath>

#include "gemm_tiled.h"
#include "gemm_tiled8.h"
#include "group_tiles.h"
#include "lds_dma.h"

namespace {

constexpr int SLICES = 8;

template <int MR, int NR>
__global__ void __launch_bounds__(64 * SLICES) k_block_sliced(A8W8Params p, GroupParams g) {
    constexpr int BM = 16 * MR, TN = 16 * NR, A_BYTES = BM * TK, W_BYTES = TN * TK, PIECE = A_BYTES + W_BYTES + 512;  // (scales: 64 rows', and the columns' one 64 times)
    static_assert(128 % TN == 0 && BM <= 64, "a tile's columns lie in one block, its rows' scales are one DMA");
    static_assert(MR * NR * 1024 <= PIECE, "a wavefront's sums fit its piece");
    __shared__ __attribute__((aligned(1024))) uint8_t lds[SLICES * PIECE];
    const int tid = (int)threadIdx.x, wave = wave_id(), lane = tid & 63, li = lane & 15, lg = lane >> 4;
    GroupTile t;
    if (!group_tile<true>(g, p.M, BM, (int)blockIdx.x, (p.N + TN - 1) / TN, lane, t)) return;
    const int n0 = t.n_tile * TN;
    const uint32_t K = (uint32_t)p.K, KB = (K + TK - 1) / TK, NB = ((uint32_t)p.N + 127u) / 128u;
    const __amdgpu_buffer_rsrc_t ra = make_rsrc_uniform(p.a + (uint64_t)t.row * K, (uint64_t)(t.rows < BM ? t.rows : BM) * K);
    const __amdgpu_buffer_rsrc_t rb = make_rsrc_uniform(p.b + ((uint64_t)t.e * (uint32_t)p.N + (uint32_t)n0) * K, (uint64_t)(uint32_t)(p.N - n0) * K);
    const __amdgpu_buffer_rsrc_t rsa = make_rsrc_uniform(p.sa + t.row, ((uint64_t)(KB - 1) * g.sa_stride + (uint32_t)(p.M - t.row)) * 4ull);
    const __amdgpu_buffer_rsrc_t rsb = make_rsrc_uniform(p.sb + ((uint64_t)t.e * NB + (uint32_t)n0 / 128u) * KB, KB * 4ull);
    // (in a scalar register that the compiler cannot trace to the thread's number: it would keep every DMA's address in a vector register)
    uint32_t piece = (uint32_t)__builtin_amdgcn_readfirstlane((int)((uint32_t)(uintptr_t)lds + (uint32_t)wave * (uint32_t)PIECE));
    asm volatile("" : "+s"(piece));
    // a lane's 16-byte piece of its row in a DMA of eight rows, by the parity of the DMA (LDS rows are XORed with row / 2)
    const uint32_t kc[2] = {(uint32_t)((lane & 7) ^ (lane >> 4)) * 16u, (uint32_t)((lane & 7) ^ (lane >> 4) ^ 4) * 16u};
    uint32_t a_off[2 * MR], w_off[NR];
#pragma unroll
    for (int j = 0; j < 2 * MR; j++) a_off[j] = (uint32_t)(j * 8 + (lane >> 3)) * K + kc[j & 1];
#pragma unroll
    for (int ni = 0; ni < NR; ni++) w_off[ni] = n0 + ni * 16 < p.N ? (uint32_t)ni * 16u * K + (uint32_t)lane * 16u : OOB;
    // Step s of K.  What lies behind K, the group's rows or the columns is redirected behind the descriptors' bounds, or lies there, and reads as zero; rows past the group's end have others' scales.
    auto ask = [&](uint32_t s) __attribute__((always_inline)) {
        const bool in[2] = {s * TK + kc[0] < K, s * TK + kc[1] < K}, upper = s * TK + 64u < K;
#pragma unroll
        for (int j = 0; j < 2 * MR; j++) dma16(ra, piece + (uint32_t)j * 1024u, in[j & 1] ? a_off[j] : OOB, s * TK);
#pragma unroll
        for (int ni = 0; ni < NR; ni++) {
            dma16(rb, piece + (uint32_t)(A_BYTES + ni * 2048), w_off[ni], s * 2048u);
            dma16(rb, piece + (uint32_t)(A_BYTES + ni * 2048 + 1024), upper ? w_off[ni] : OOB, upper ? s * 2048u + 1024u : 0u);
        }
        dma4(rsa, piece + (uint32_t)(A_BYTES + W_BYTES), lane < BM ? (uint32_t)lane * 4u : OOB, s * g.sa_stride * 4u);
        dma4(rsb, piece + (uint32_t)(A_BYTES + W_BYTES + 256), 0u, s * 4u);
    };
    v4f acc[MR][NR];
#pragma unroll
    for (int mi = 0; mi < MR; mi++)
#pragma unroll
        for (int ni = 0; ni < NR; ni++) acc[mi][ni] = (v4f){0.f, 0.f, 0.f, 0.f};
    const uint8_t* const mine = lds + wave * PIECE;
    if ((uint32_t)wave < KB) ask((uint32_t)wave);
    for (uint32_t s = (uint32_t)wave; s < KB; s += SLICES) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // (the compiler does not know that the DMAs write LDS)
        v4i a[MR][2], w[NR][2];
        float scale[MR];
#pragma unroll
        for (int ni = 0; ni < NR; ni++)
#pragma unroll
            for (int h = 0; h < 2; h++) w[ni][h] = *reinterpret_cast<const v4i*>(mine + A_BYTES + ni * 2048 + h * 1024 + lane * 16);
        const float column = *reinterpret_cast<const float*>(mine + A_BYTES + W_BYTES + 256 + lane * 4);
#pragma unroll
        for (int mi = 0; mi < MR; mi++) {
#pragma unroll
            for (int h = 0; h < 2; h++) a[mi][h] = *reinterpret_cast<const v4i*>(mine + lds_off(mi * 16 + li, 4 * h + lg));
            scale[mi] = *reinterpret_cast<const float*>(mine + A_BYTES + W_BYTES + (mi * 16 + li) * 4) * column;
        }
        // everything is in registers before the next step's DMAs may write over it
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
        if (s + SLICES < KB) ask(s + SLICES);
        static_for<MR>([&](auto MI) {
            constexpr int mi = decltype(MI)::value;
            v4f part[NR];
#pragma unroll
            for (int ni = 0; ni < NR; ni++)
                part[ni] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(__builtin_shufflevector(w[ni][0], w[ni][1], 0, 1, 2, 3, 4, 5, 6, 7), __builtin_shufflevector(a[mi][0], a[mi][1], 0, 1, 2, 3, 4, 5, 6, 7),
                                                                            (v4f){0.f, 0.f, 0.f, 0.f}, 0, 0, 0, 0, 0, 0);
#pragma unroll
            for (int ni = 0; ni < NR; ni++)
#pragma unroll
                for (int i = 0; i < 4; i++) acc[mi][ni][i] = __builtin_fmaf(part[ni][i], scale[mi], acc[mi][ni][i]);
        });
    }
    // the slices' sums, every wavefront's in its own piece, added in their order, a fragment a wavefront; out 8 bytes a lane
    v4f* const sums = reinterpret_cast<v4f*>(lds + wave * PIECE);
#pragma unroll
    for (int mi = 0; mi < MR; mi++)
#pragma unroll
        for (int ni = 0; ni < NR; ni++) sums[(mi * NR + ni) * 64 + lane] = acc[mi][ni];
    __syncthreads();
    for (int f = wave; f < MR * NR; f += SLICES) {
        v4f part[SLICES], x;
#pragma unroll
        for (int j = 0; j < SLICES; j++) part[j] = reinterpret_cast<const v4f*>(lds + j * PIECE)[f * 64 + lane];
        x = part[0];
#pragma unroll
        for (int j = 1; j < SLICES; j++) x += part[j];
        const int row = f / NR * 16 + li, n = n0 + f % NR * 16 + lg * 4;
        if (row < t.rows && n < p.N)
            *reinterpret_cast<v2i*>(static_cast<uint16_t*>(p.c) + (size_t)(t.row + row) * (size_t)p.N + n) = p.out == OUT_BF16 ? pack4_out16<OUT_BF16>(x[0], x[1], x[2], x[3]) : pack4_out16<OUT_FP16>(x[0], x[1], x[2], x[3]);
    }
}

template <int MR, int NR>
hipError_t launch(const A8W8Params& p, GroupParams g, hipStream_t stream) {
    g.most = (int)group_tiles_most(p.M, g.groups, 16 * MR);
    hipLaunchKernelGGL((k_block_sliced<MR, NR>), dim3((unsigned)g.most * (unsigned)((p.N + 16 * NR - 1) / (16 * NR))), dim3(64 * SLICES), 0, stream, p, g);
    return hipGetLastError();
}

template <int STORE>
__global__ void __launch_bounds__(256, 2) k_block_square(A8W8Params p, GroupParams g) {
    tiled_dma<KIND_FP8B, STORE, 8, 4, 4, 3>(p, g);
}

}  // namespace

// The way of the least estimated time, in us.  Of `load` tiles a CU: a tile's steps when it is alone on its CU, longer as more CUs are at work; a CU's steps and tile ends where it has many (whole rounds of
// small tiles, up to four); W from memory.
// The constants are fitted to the times of 3,400 products of 1 to 32,768 rows on 1 to 128 groups (128 x 128 tiles to 6,000 others), which are not kept; on 4,800 more (profiles/block_scaled_times.csv, every way's
// time and the choice) it is 3.5 % slower than the best way dense and 2.8 % grouped, in the geometric mean (the choice for one scale a row, psg_grouped_plan, 15 and 7).  Slices with 16 x 64, 32 x 16, 64 x 16 and 64 x 32 tiles win 0.2 % more together and are not built.
// us, whole K on 16, 32, 64, 128 rows / slices on 16 x 16, 16 x 32, 32 x 32, 32 x 64, 64 x 64 / streamed: 346 x 352 x 11328 20.9, 23.3, 44.8, 69.7 / 12.4, 9.6, 11.7, 16.2, 22.3 / 19.1; 201 x 752 x 10624 21.9, 23.5, 41.9, 71.7 / 15.4,
// 14.0, 11.3, 15.5, 20.6 / 15.1; 775 x 624 x 13184 35.8, 31.5, 52.2, 94.9 / 41.0, 34.3, 26.1, 21.1, 28.4 / -; 127 x 5104 x 2944 12.7, 11.0, 15.1, 21.0 / 15.9, 13.3, 10.9, 12.0, 9.5 / -; 13 x 1616 x 16256 35.7, 38.1, 63.0, 129 /
// 15.3, 17.4, 18.1, 26.9, 30.6 / 10.4; 8 rows on 8, 1552 x 5504, 12.2, 13.6, 24.1, 33.6 / 6.5, 6.8, 7.3, 8.8, 10.7; 620 x 1760 x 832 7.7, 6.4, 7.2, 9.9 / 14.9, 9.9, 8.8, 10.0, 9.4.
BlockPlan psg_block_plan(int64_t rows, int groups, bool dense, int N, int K) {
    struct Way { int bm, tn; bool sliced, rounds; double start, alone, more, busy, end; };
    static constexpr Way ways[] = {
        {16, 64, false, true, 2.78, 0.199, 0.135, 0.173, 0.25},  {32, 64, false, true, 2.86, 0.228, 0.131, 0.202, 0.31}, {64, 128, false, false, 3.72, 0.449, 0.179, 0.425, 1.24},
        {128, 128, false, false, 4.28, 0.494, 0.152, 0.696, 1.77}, {128, 256, false, false, 3.99, 0.729, 0.762, 0.966, 2.51},
        {16, 16, true, true, 2.43, 0.471, 0.288, 0.397, 0.24},   {16, 32, true, true, 2.28, 0.597, 0.544, 0.629, 0.19},  {32, 32, true, true, 2.06, 0.718, 0.693, 0.851, 0.32},
        {32, 64, true, false, 2.66, 0.943, 1.030, 1.768, 0.74},  {64, 64, true, false, 2.93, 1.257, 1.492, 2.147, 1.16},
    };
    const int64_t live = groups < rows ? groups : rows, steps = (K + 127) / 128;
    BlockPlan best = {1, 8, false};
    double least = dense && rows <= 65535 * 64 ? psg_blockscale_stream_us((int)rows, N, K) : 1e30;
    for (const Way& w : ways) {
        const int64_t columns = (N + w.tn - 1) / w.tn;
        if (group_tiles_most(rows, groups, w.bm) * columns >= 1ll << 23) continue;  // (more than a launch holds)
        // (the groups' last tiles are half empty on average)
        double tiles = groups == 1 ? (double)((rows + w.bm - 1) / w.bm) : rows / (double)w.bm + 0.5 * live;
        if (tiles < live) tiles = (double)live;
        const double load = tiles * columns / psg_cu_count(), n = (double)(w.sliced ? (steps + 7) / 8 : steps);
        double t = n * (w.alone + w.more * (load < 1 ? load : 1));
        const double busy = (w.rounds && load <= 4 ? std::ceil(load) : load) * (n * w.busy + w.end);
        const double weights = (double)live * N * K / (w.sliced ? 8e6 : 10e6);
        t = t > busy ? t : busy;
        t = w.start + (t > weights ? t : weights);
        if (t < least) least = t, best = {w.bm, w.tn, w.sliced};
    }
    return best;
}

// Tiles of 128 x 128, K in one piece, for one or two tiles a CU; bf16 by STORE_C, fp16 by STORE_C_GENERIC.  us, these / 128 x 256 tiles / the best of the others: 1024 x 4096 x 4096 25.1 / 36.1 / 30.3,
// 700 x 5120 x 5120 29.2 / 43.8 / 34.6, 512 x 8192 x 8192 44.9 / 69.0 / 55.7, 512 x 7168 x 2048 15.2 / 21.3 / 17.2; of more tiles 2048 x 4096 x 4096 40.1 / 37.9, 8192 x 4096 x 4096 148 / 120, of fewer
// 256 x 4096 x 4096 23.4 / 36.1 / 12.7, 512 x 4096 x 4096 23.8 / 35.7 / 20.2.
hipError_t psg_launch_block_square(const A8W8Params& p, GroupParams g, hipStream_t stream) {
    g.most = (int)group_tiles_most(p.M, g.groups, 128);
    const dim3 grid((unsigned)g.most * (unsigned)((p.N + 127) / 128));
    if (p.out == OUT_BF16) hipLaunchKernelGGL((k_block_square<STORE_C>), grid, dim3(256), 0, stream, p, g);
    else hipLaunchKernelGGL((k_block_square<STORE_C_GENERIC>), grid, dim3(256), 0, stream, p, g);
    return hipGetLastError();
}

hipError_t psg_launch_block_sliced(const A8W8Params& p, const GroupParams& g, int bm, int tn, hipStream_t stream) {
    if (bm == 16) return tn == 16 ? launch<1, 1>(p, g, stream) : launch<1, 2>(p, g, stream);
    if (bm == 32) return tn == 32 ? launch<2, 2>(p, g, stream) : launch<2, 4>(p, g, stream);
    return launch<4, 4>(p, g, stream);
}
