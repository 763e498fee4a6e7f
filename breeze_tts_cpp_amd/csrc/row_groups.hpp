// Rows grouped by the weights they use: the device side of what
// qlin_route / qlin_group_rows write and the grouped products read.
//   offsets [groups + 1]  the slots [offsets[g], offsets[g + 1]) hold group g's rows
//   order   [slots]       the row (or choice) each slot came from
// Both live on the device, so a launch is sized by the host's upper bound
// and each workgroup finds its tile from the offsets.
#pragma once
#include "qlin_device.hpp"

namespace qlin {
namespace {

// Inclusive prefix sum over the 64 lanes: row shifts inside each 16, then the
// last lane of a 16 / 32 added to the next (lanes without a source add 0).
__device__ __forceinline__ int wave_scan(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, true);   // row_shr:1
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, true);   // row_shr:2
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, true);   // row_shr:4
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, true);   // row_shr:8
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);  // row_bcast:15
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);  // row_bcast:31
    return v;
}

// The same with the maximum in place of the sum (values from 0 on; unsigned, so that
// the exchange folds into the maximum).
__device__ __forceinline__ int wave_scan_max(uint32_t v) {
    v = max(v, uint32_t(__builtin_amdgcn_update_dpp(0, int(v), 0x111, 0xF, 0xF, true)));
    v = max(v, uint32_t(__builtin_amdgcn_update_dpp(0, int(v), 0x112, 0xF, 0xF, true)));
    v = max(v, uint32_t(__builtin_amdgcn_update_dpp(0, int(v), 0x114, 0xF, 0xF, true)));
    v = max(v, uint32_t(__builtin_amdgcn_update_dpp(0, int(v), 0x118, 0xF, 0xF, true)));
    v = max(v, uint32_t(__builtin_amdgcn_update_dpp(0, int(v), 0x142, 0xA, 0xF, false)));
    v = max(v, uint32_t(__builtin_amdgcn_update_dpp(0, int(v), 0x143, 0xC, 0xF, false)));
    return int(v);
}

// One tile of a grouped product: `rows` slots from `begin` of group `group`,
// column tile `column`.
struct RowTile {
    int group, begin, rows, column;
};

// The tile of workgroup `index`: the groups' row tiles of at most `height`
// slots times `columns` column tiles, numbered group by group, each column
// tile's row tiles in a run (they share the group's weights there). The
// hardware places workgroup i on XCD i % 8: every 256 workgroups (a round of the
// CUs) take 256 tiles, each XCD 32 in a run that share its L2; the rest of the
// tiles is numbered XCD-major. (All tiles XCD-major puts whole groups on one XCD,
// and groups differ in size: a 4096-token prefill over 32 experts 5% slower.) False past the last tile.
// Bad offsets cannot lead out of the arrays, nor two groups to one slot: each is
// held to [0, slots] and to the largest before it, so that a slot belongs to the
// first group that claims it and the tiles are no more than the launch's bound.
// Same result in every lane of the workgroup.
__device__ __forceinline__ bool find_tile(const int *__restrict__ offsets, int groups, int slots,
                                          int height, int columns, int index, RowTile &tile) {
    const int lane = threadIdx.x & 63;
    // Rows of the groups [g0, g0 + 64), one a lane, after offsets up to `largest`.
    auto load = [&](int g0, int &largest, int &begin) {
        const int g = g0 + lane;
        const int from = offsets[min(g, groups)], to = offsets[min(g + 1, groups)];
        begin = max(wave_scan_max(uint32_t(min(max(from, 0), slots))), largest);
        largest = __builtin_amdgcn_readlane(begin, 63);
        return max(min(to, slots) - begin, 0);
    };
    int first_begin = 0, first_largest = 0;
    const int first_rows = load(0, first_largest, first_begin);
    int mine = (first_rows + height - 1) / height;
    for (int g0 = 64, largest = first_largest; g0 < groups; g0 += 64) {
        int begin;
        mine += (load(g0, largest, begin) + height - 1) / height;
    }
    const int total = __builtin_amdgcn_readlane(wave_scan(mine), 63) * columns;
    if (index >= total) return false;
    const int whole = total & ~255;
    const int at = index < whole ? (index & ~255) + (index % 8) * 32 + index % 256 / 8
                                 : whole + xcd_major(index - whole, total - whole);
    int before = 0;  // row tiles of the groups before this run of 64
    for (int g0 = 0, largest = first_largest; g0 < groups; g0 += 64) {
        int begin = first_begin;
        const int rows = g0 ? load(g0, largest, begin) : first_rows;
        const int tiles = (rows + height - 1) / height;
        const int upto = before + wave_scan(tiles);
        const uint64_t past = __ballot(upto * columns > at);
        if (past) {
            const int l = __builtin_ctzll(past);
            const int n = __builtin_amdgcn_readlane(tiles, l);
            const int in = at - (__builtin_amdgcn_readlane(upto, l) - n) * columns;
            const int row = in % n * height;
            tile.group = g0 + l;
            tile.column = in / n;
            tile.begin = __builtin_amdgcn_readlane(begin, l) + row;
            tile.rows = min(height, __builtin_amdgcn_readlane(rows, l) - row);
            return true;
        }
        before = __builtin_amdgcn_readlane(upto, 63);
    }
    return false;
}

}  // namespace
}  // namespace qlin
