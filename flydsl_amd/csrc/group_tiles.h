// Tiles of a product whose rows are grouped, the groups' ends known on the device only: which rows of which group a workgroup multiplies.
#pragma once
#include "psg_common.h"
#include "tile_order.h"

// Groups of rows: group e has rows [offsets[e], offsets[e + 1]) of A and C (clamped to the rows there are; none where the next offset is not above) and weight e.
struct GroupParams {
    const int32_t* offsets;  // [groups + 1]; nullptr: all rows are one group (block-scaled products only)
    int groups;
    int past;  // set by the launcher (128x256 tiles): C goes past the caches
    int most;  // set by the launcher: tiles along M that the grid was made for (offsets that go back may say more)
    // block-scaled products: A8W8Params::sa is [ceil(K / 128)][M], rows of sa_stride floats; sb [groups][ceil(N / 128)][ceil(K / 128)]
    uint32_t sa_stride;
};

// Rows of a tile (16, 32, 64 or 128), and whether K is cut into slices (16 rows only)
struct GroupedPlan {
    int bm;
    bool sliced;
};
GroupedPlan psg_grouped_plan(int64_t rows, int groups, int N, int64_t kbytes);
hipError_t psg_launch_grouped(const A8W8Params& p, const GroupParams& g, int kind, GroupedPlan plan, hipStream_t stream);
// How a block-scaled product is done: by tiles of bm rows and tn columns, with K in one piece or in slices, or (bm = 1) as a few rows against streamed weights
struct BlockPlan {
    int bm, tn;
    bool sliced;
};
BlockPlan psg_block_plan(int64_t rows, int groups, bool dense, int N, int K);
double psg_blockscale_stream_us(int M, int N, int K);
hipError_t psg_launch_block_square(const A8W8Params& p, GroupParams g, hipStream_t stream);
hipError_t psg_launch_block_sliced(const A8W8Params& p, const GroupParams& g, int bm, int tn, hipStream_t stream);
hipError_t psg_launch_blockscale_stream(const A8W8Params& p, const GroupParams& g, hipStream_t stream);
hipError_t psg_launch_grouped_pair(const A8W8Params& p, GroupParams g, int kind, hipStream_t stream);

// Upper bound of the tiles of `bm` rows that the rows of `groups` groups make, for the grid: a group's last tile may be almost empty, a group without rows makes none
inline int64_t group_tiles_most(int64_t rows, int64_t groups, int bm) { return (rows + (groups < rows ? groups : rows) * (bm - 1)) / bm; }

namespace {

struct GroupTile {
    int e;       // group
    int row;     // first row
    int rows;    // rows of the group from there on, more than `bm` of them where the tile is not its last
    int n_tile;  // tile along N
};

// sum over the lanes up to this one: inside rows of 16 by shifts, then the last lane of a row to the one behind it, of the first half to the second (by DPP: six exchanges through
// LDS would be half a microsecond in front of every tile)
__device__ __forceinline__ int sum_upto(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);  // row_shr:1
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);  // row_bcast:15 into rows 1 and 3
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);  // row_bcast:31 into rows 2 and 3
    return v;
}

// Workgroup `wg` of the launch -> its tile; false for the workgroups that the bound of the grid counts too many.  Every wavefront works it out by itself, a group a lane: no
// barrier; uniform.  Tiles are walked as in psg_tile_order, eight of them along M at a time, so that an XCD reads a group's weight once.
template <bool ONE = false>
__device__ __forceinline__ bool group_tile(const GroupParams& g, int M, int bm, int wg, int n_tiles, int lane, GroupTile& t) {
    if constexpr (ONE) {
        if (!g.offsets) {
            int m;
            psg_tile_order(wg, g.most, n_tiles, 8, &m, &t.n_tile);
            t.e = 0, t.row = m * bm, t.rows = M - t.row;
            return true;
        }
    }
    // of group base + lane: first row, rows, and its tiles with those of the lanes in front of it
    auto look = [&](int base, int& row, int& rows, int& upto) __attribute__((always_inline)) {
        const int e = base + lane;
        const int a = g.offsets[e < g.groups ? e : g.groups], b = g.offsets[e + 1 < g.groups ? e + 1 : g.groups];
        row = a < 0 ? 0 : a < M ? a : M;
        const int end = b < 0 ? 0 : b < M ? b : M;
        rows = end > row ? end - row : 0;
        upto = (int)((unsigned)(rows + bm - 1) / (unsigned)bm);
        upto = sum_upto(upto);
    };
    int row, rows, upto, total = 0;
    look(0, row, rows, upto);
    total = __builtin_amdgcn_readlane(upto, 63);
    for (int base = 64; base < g.groups; base += 64) {
        int r, n, u;
        look(base, r, n, u);
        total += __builtin_amdgcn_readlane(u, 63);
    }
    total = total < g.most ? total : g.most;
    if (wg >= total * n_tiles) return false;
    int m;
    psg_tile_order(wg, total, n_tiles, 8, &m, &t.n_tile);
    int base = 0, before = 0;
    for (;;) {
        const uint64_t at = __ballot(before + upto > m);
        if (at) {
            const int l = __builtin_ctzll(at);
            const int mine = (int)((unsigned)(__builtin_amdgcn_readlane(rows, l) + bm - 1) / (unsigned)bm);
            const int in = m - (before + __builtin_amdgcn_readlane(upto, l) - mine);
            t.e = base + l;
            t.row = __builtin_amdgcn_readlane(row, l) + in * bm;
            t.rows = __builtin_amdgcn_readlane(rows, l) - in * bm;
            return true;
        }
        before += __builtin_amdgcn_readlane(upto, 63);
        base += 64;
        if (base >= g.groups) return false;  // (not reached: m is below the sum of all tiles)
        look(base, row, rows, upto);
    }
}

}  // namespace
