// Shared pieces of the microscaled 4-bit kernels (mx4.hip, mx4_gemm.hip): the
// scale's value and where the rows of a group lie in the padded places of a
// matrix quantised along its columns.
#pragma once

#include "rhp_common.h"

namespace rhp {
namespace {

constexpr int kMx4Many = RHP_MAX_GROUPS_PER_LAUNCH;   // matrices a quantising launch

// The scale with exponent code e (0 .. 254): a power of two, the lowest one subnormal.
__device__ __forceinline__ float mx4_scale(uint32_t e) { return __uint_as_float(e ? e << 23 : 0x00400000u); }

// Lane g of the wave: the padded rows (multiples of 128) of the groups before
// g and of group g, whose rows are [first, first + count) of the matrix.
// Offsets that leave [0, rows] or descend are cut: no row outside the matrix.
struct Mx4Groups {
    int first, count, pad_begin, pad;
    int total;   // padded rows of all groups
    int before;  // rows ahead of the groups
    int last;    // the first row behind them
};
__device__ __forceinline__ Mx4Groups mx4_groups(const int32_t* offsets, int G, int64_t rows) {
    static_assert(RHP_MAX_GROUPS_PER_LAUNCH <= 64, "one group per lane");
    const int lane = static_cast<int>(threadIdx.x & 63), R = static_cast<int>(rows);
    Mx4Groups m{0, 0, 0, 0, 0, 0, 0};
    if (lane < G) {
        m.first = min(max(offsets[lane], 0), R);
        m.count = max(min(offsets[lane + 1], R) - m.first, 0);
    }
    m.pad = (m.count + 127) / 128 * 128;
    int end = m.pad;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int v = __shfl_up(end, d);
        if (lane >= d) end += v;
    }
    m.pad_begin = end - m.pad;
    m.total = __builtin_amdgcn_readlane(end, 63);
    m.before = __builtin_amdgcn_readfirstlane(m.first);
    m.last = min(max(offsets[G], 0), R);
    return m;
}

// Rows [r0, r1) of the matrix at padded places [pos, pos + 128): those of the
// group there; past the groups' places the rows behind the last group, then
// those ahead of the first (which no group's product reads), 128 at a time.
// (rows + 127 (G + 2)) / 128 tiles reach all of them.
struct Mx4Tile {
    int64_t r0, r1;
    bool in_group;
};
__device__ __forceinline__ Mx4Tile mx4_tile(const int32_t* offsets, int G, int64_t rows, int pos) {
    const Mx4Groups m = mx4_groups(offsets, G, rows);
    if (pos >= m.total) {
        const int64_t past = pos - m.total, behind = (rows - m.last + 127) / 128 * 128;
        if (past < behind) return {m.last + past, rows, false};
        return {past - behind, m.before, false};
    }
    const int g = __ffsll(static_cast<unsigned long long>(__ballot(pos < m.pad_begin + m.pad))) - 1;
    const int first = __builtin_amdgcn_readlane(m.first, g);
    return {first + static_cast<int64_t>(pos - __builtin_amdgcn_readlane(m.pad_begin, g)),
            first + static_cast<int64_t>(__builtin_amdgcn_readlane(m.count, g)), true};
}

}  // namespace
}  // namespace rhp
