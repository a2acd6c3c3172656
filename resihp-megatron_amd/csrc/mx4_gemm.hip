// Grouped products of operands in microscaled 4-bit floating point, for gfx950.
//
// The grouped products are those of the expert FFN (resihp/runtime/
// moe.py:82-83, 96-100, 164-167) with both operands quantised along the
// reduction (mx4.hip):
//   row groups   y[t, n]  = sum_k a[t, k]  w_g[n, k]   token rows t of group g
//   K groups     dW_g[o, i] = sum_t aT[o, t] bT[i, t]  t over group g's padded places
// with a[t, k] = code * 2^scale of each operand.  A 32 x 32 x 64 product is one
// v_mfma_scale_f32_32x32x64_f8f6f4 on e2m1 codes with a scale a lane: lane L
// holds row L % 32 and the 32 values of block L / 32, so a lane's operand is
// the 16 bytes of one block and its scale that block's.  Products of codes and
// scales are exact; sums are float; the bfloat16 output is rounded once.
//
// A block computes 256 x 256 outputs on eight waves of 128 x 64; one block a CU.
// Measured on 16384 rows of 8 groups, of 2048 each / ragged (1356 to 4126): 28672 x
// 4096 in 1.06 / 1.09 ms (3.6, 3.5 PFLOP/s), the product back, 4096 x 28672, in 0.91 /
// 1.03 (4.2, 3.7), the weights' gradient in 1.32 / 1.35 (2.9, 2.8).
// The matrix cores alone, on random codes in registers, hold 5.9 PFLOP/s of this
// shape (9.2 on zeros: the clock falls with the power) and 7.25 of 16 x 16 x 128, and a
// further 4096 of K runs at 4.9 PFLOP/s (ragged 4.6); the rest is the first loads and
// the stores of a tile, which no other block covers (forward without its stores -16 %,
// without its loads -18 %).  Built and timed against it on these three: blocks that walk
// their tiles with the next one's loads under the stores, on either product, four waves
// of 128 x 128 and four stages of 128 places, none faster by more than 2 %; blocks that
// start at different times, no difference.  16 x 16 x 128 in this kernel's structure was
// not built.  Few rows take gg_mx4_short_kernel.

#include <type_traits>

#include "gemm_common.h"
#include "mx4_common.h"

namespace rhp {
namespace {

// A K step is 256 codes, one 128-byte line a row: an operand tile of 256 rows
// is 32 KB and its scales 2 KB (two words a row).  Two stages; the loads of a
// step have a whole step to land.
constexpr int kM4K = 256;
constexpr int kM4Blocks = kM4K / 32;
constexpr int kM4Tile = kTile * kM4K / 2;
constexpr int kM4Scales = kTile * kM4Blocks;
constexpr int kM4Stage = 2 * (kM4Tile + kM4Scales);
constexpr int kM4PerWave = kM4Tile / 1024 / kWaves;
constexpr int kM4Lds = 2 * kM4Stage > kEpBytes ? 2 * kM4Stage : kEpBytes;
static_assert(kM4Lds <= 163840, "two stages");
constexpr int kFmtE2m1 = 4;   // MFMA operand format code

typedef int i32x8_t __attribute__((ext_vector_type(8)));

struct Mx4Gemm {
    Params p;            // a[0], b[0]: codes; lda, ldb: bytes a row; K: blocks of 32 of a row
    const uint8_t* ys;   // scales of a
    const uint8_t* xs;   // scales of b
    int64_t x_codes, x_scales;   // bytes from one group's weight to the next
    int64_t y_rows, x_rows;      // rows of the operands (words between their scales' 128-blocks)
};

// 4 bytes per lane from the buffer at voff + soff into LDS at lds + 4 * lane.
__device__ __forceinline__ void dma4(const Rsrc& r, uint32_t voff, uint32_t soff, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %3\n\tbuffer_load_dword %0, %1, %2 offen lds"
                 :
                 : "v"(voff), "s"(r.d), "s"(__builtin_amdgcn_readfirstlane(soff)),
                   "s"(__builtin_amdgcn_readfirstlane(lds))
                 : "memory");
}

template <int MODE, int EPI>
__global__ __launch_bounds__(kThreadsMfma) void gg_mx4_kernel(Mx4Gemm q) {
    const Params& p = q.p;
    __shared__ __align__(1024) uint8_t lds[kM4Lds];
    Tile t;
    if (find_tile<MODE>(p, x_per_tile<EPI>(), kTile, blockIdx.x, &t) != kTileOk) return;
    t.g = __builtin_amdgcn_readfirstlane(t.g);
    t.x0 = __builtin_amdgcn_readfirstlane(t.x0);
    t.x_lim = __builtin_amdgcn_readfirstlane(t.x_lim);
    t.y0 = __builtin_amdgcn_readfirstlane(t.y0);
    t.y_lim = __builtin_amdgcn_readfirstlane(t.y_lim);
    t.row0 = __builtin_amdgcn_readfirstlane(static_cast<int>(t.row0));
    const int g = t.g;
    const int L = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wx = wave & 1, wy = wave >> 1;

    // Blocks of 32 to sum over, and the first of them in the operands' rows (a multiple of four).
    int blocks = p.K, first = 0;
    if constexpr (MODE == kWgrad) {
        const Mx4Groups m = mx4_groups(p.offsets, p.G, p.rows_cap);
        blocks = (__builtin_amdgcn_readlane(m.count, g) + 31) / 32;
        first = __builtin_amdgcn_readlane(m.pad_begin, g) / 32;
        blocks = min(blocks, max(0, p.K - first));   // p.K: blocks of all places
    }
    const int nk = (blocks + kM4Blocks - 1) / kM4Blocks;
    const int words = (blocks + 3) / 4;

    const uint32_t lda = static_cast<uint32_t>(p.lda), ldb = static_cast<uint32_t>(p.ldb);
    const int64_t yfirst = tile_first_row<MODE>(t);
    const Rsrc ry = make_dma_rsrc(static_cast<const uint8_t*>(p.a[0]) + yfirst * p.lda,
                                  static_cast<int64_t>(min(t.y_lim, kTile)) * p.lda);
    const uint8_t* X = static_cast<const uint8_t*>(p.b[0]) + (MODE == kWgrad ? 0 : g * q.x_codes);
    const Rsrc rx = make_dma_rsrc(X, q.x_rows * p.ldb);
    const int64_t all_words = (static_cast<int64_t>(p.K) + 3) / 4;
    const Rsrc rys = make_dma_rsrc(q.ys, all_words * q.y_rows * 4);
    const Rsrc rxs = make_dma_rsrc(q.xs + (MODE == kWgrad ? 0 : g * q.x_scales), all_words * q.x_rows * 4);

    const auto y_row = [&](int r) { return min(r, t.y_lim - 1); };
    const auto x_row = [&](int r) {
        if (is_swiglu_fwd(EPI)) {
            // 256 weight rows = [gate 64 | up 64] for each half of 128 activation columns.
            const int half = r >> 7, qq = r & 127;
            int col = t.x0 + half * 64 + (qq & 63);
            col = col < p.f ? col : 0;
            return qq < 64 ? col : p.f + col;
        }
        const int n = t.x0 + r;
        return n < p.N ? n : 0;
    };
    // Lane L of load j of wave w fills 16 bytes of row 8 (8 j + w) + L / 8: the block that belongs at place L % 8
    // (k64_off); it is the same for every j.
    const int chunk = (L & 7) ^ ((wave & 1) * 4 + (L >> 4));
    uint32_t vx[kM4PerWave], vy[kM4PerWave];
#pragma unroll
    for (int j = 0; j < kM4PerWave; ++j) {
        const int row = (j * kWaves + wave) * 8 + (L >> 3);
        vx[j] = static_cast<uint32_t>(x_row(row)) * ldb + chunk * 16;
        vy[j] = static_cast<uint32_t>(y_row(row)) * lda + chunk * 16;
    }
    // Scales: wave w loads word w % 2 of the step's two for rows 64 (w / 2) .. + 63 of both operands.
    const int srow = 64 * (wave >> 1) + L;
    const uint32_t vxs = static_cast<uint32_t>(x_row(srow)) * 4;
    const uint32_t vys = static_cast<uint32_t>(yfirst + y_row(srow)) * 4;

    const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(lds));
    // Quarter n of this wave's loads of step `step`: blocks past the last (all of them, past the last step) read as
    // zeros, and so do their scales (a scale that is not this group's must not meet zero codes: it may be NaN).
    auto issue = [&](int step, int n) {
        const uint32_t base = lds0 + (step & 1) * kM4Stage + wave * 1024;
        const uint32_t soff = static_cast<uint32_t>(first * 16 + step * (kM4K / 2));
        const uint32_t off = chunk < blocks - step * kM4Blocks ? 0u : kOutOfRange;
        if (n < 2) {
#pragma unroll
            for (int j = 2 * n; j < 2 * n + 2; ++j) dma16(ry, vy[j] | off, soff, base + kM4Tile + j * kWaves * 1024);
        } else {
#pragma unroll
            for (int j = 2 * (n - 2); j < 2 * (n - 2) + 2; ++j) dma16(rx, vx[j] | off, soff, base + j * kWaves * 1024);
            const int word = 2 * step + (wave & 1);
            const uint32_t sbase = lds0 + (step & 1) * kM4Stage + 2 * kM4Tile + (wave & 1) * 1024 + (wave >> 1) * 256;
            const uint32_t soffs = word < words ? static_cast<uint32_t>(first / 4 + word) * 4u : 0u;
            const uint32_t out = word < words ? 0u : kOutOfRange;
            if (n == 2)
                dma4(rxs, vxs | out, soffs * static_cast<uint32_t>(q.x_rows), sbase);
            else
                dma4(rys, vys | out, soffs * static_cast<uint32_t>(q.y_rows), sbase + kM4Scales);
        }
    };
    constexpr int kLoads = 2 * kM4PerWave + 2;   // of a step, a wave
    auto wait_lds = [](auto n_c) {               // vmcnt(n) lgkmcnt(0)
        constexpr int n = decltype(n_c)::value;
        __builtin_amdgcn_s_waitcnt(0x0070 | (n & 15) | ((n >> 4) << 14));
    };
    auto barrier = [] {
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };

    Acc32<kWaveY> acc;
    acc.zero();
    static_assert(kFragY == 2, "six fragments: X 0 to 3, Y 0 and 1");
    typedef i32x4_t FragSet[6];
    typedef uint32_t ScaleSet[6][2];
    // A fragment's rows are 32 apart, whole turns of the places' pattern: fragment i of the wave's X rows lies at
    // px + 4096 i (its scales at sx + 128 i), of its Y rows at py + 4096 j; block b turns the place by 32 b bytes.
    const int half = L >> 5;
    const uint32_t lane_place = k64_off(L & 31, half);
    const uint32_t px = static_cast<uint32_t>(wx * 128 * 128), py = static_cast<uint32_t>(kM4Tile + wy * kWaveY * 128);
    const uint32_t sx = static_cast<uint32_t>(2 * kM4Tile + (wx * 128 + (L & 31)) * 4);
    const uint32_t sy = static_cast<uint32_t>(2 * kM4Tile + kM4Scales + (wy * kWaveY + (L & 31)) * 4);
    constexpr int order[6] = {0, 4, 5, 1, 2, 3};   // as the MFMAs use them: X0, Y0, Y1, X1, X2, X3
    auto read_one = [&](FragSet& f, int stage, int b, int i) {
        const uint8_t* at = lds + (stage * kM4Stage + (i < 4 ? px : py) + (lane_place ^ static_cast<uint32_t>(b << 5)));
        f[i] = *reinterpret_cast<const i32x4_t*>(at + (i & 3) * 4096);
    };
    auto read_frags = [&](FragSet& f, int stage, int b) {
#pragma unroll
        for (int i = 0; i < 6; ++i) read_one(f, stage, b, order[i]);
    };
    // The words of a step's scales, to be shifted so that bytes 0 and 2 are this lane's blocks of the two k64.
    auto read_scale = [&](ScaleSet& s, int stage, int i) {
        const uint8_t* at = lds + (stage * kM4Stage + (i < 4 ? sx : sy));
#pragma unroll
        for (int k = 0; k < 2; ++k) s[i][k] = *reinterpret_cast<const uint32_t*>(at + (i & 3) * 128 + k * 1024);
    };
    auto wide = [](i32x4_t v) { return __builtin_shufflevector(v, v, 0, 1, 2, 3, -1, -1, -1, -1); };
    auto mfma = [&](const FragSet& f, const ScaleSet& s, auto b_c, int i, int j) {
        constexpr int b = decltype(b_c)::value, sel = (b & 1) * 2;
        acc.v[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wide(f[i]), wide(f[4 + j]), acc.v[i][j], kFmtE2m1,
                                                                   kFmtE2m1, sel, s[i][b >> 1], sel, s[4 + j][b >> 1]);
    };
    auto mfmas = [&](const FragSet& f, const ScaleSet& s, auto b_c) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < kFragY; ++j) mfma(f, s, b_c, i, j);
    };
    using Three = std::integral_constant<int, 3>;

    if (nk > 0) {
#pragma unroll
        for (int n = 0; n < 8; ++n) issue(n / 4, n % 4);
        wait_lds(std::integral_constant<int, kLoads>());
        barrier();
        const bool idle = wy * kWaveY >= t.y_lim;
        if (idle) {
            for (int kt = 0; kt < nk; ++kt) {
                wait_lds(std::integral_constant<int, 0>());
                barrier();
#pragma unroll
                for (int n = 0; n < 4; ++n) issue(kt + 2, n);
            }
        } else {
            FragSet fa, fb;
            ScaleSet sc, sn;
            read_frags(fa, 0, 0);
#pragma unroll
            for (int i = 0; i < 6; ++i) read_scale(sn, 0, i);
            __builtin_amdgcn_s_waitcnt(0xc07f);   // lgkmcnt(0)
            for (int kt = 0; kt < nk; ++kt) {
                const int stage = kt & 1;
#pragma unroll
                for (int i = 0; i < 6; ++i)
#pragma unroll
                    for (int k = 0; k < 2; ++k) sc[i][k] = sn[i][k] >> (8 * half);
                read_frags(fb, stage, 1);
                mfmas(fa, sc, std::integral_constant<int, 0>());
                interleave_reads<0, 8, 6>();
                read_frags(fa, stage, 2);
                mfmas(fb, sc, std::integral_constant<int, 1>());
                interleave_reads<0, 8, 6>();
                read_frags(fb, stage, 3);
                mfmas(fa, sc, std::integral_constant<int, 2>());
                interleave_reads<0, 8, 6>();
                // The next step's loads have landed, every read of this stage is done.
                wait_lds(std::integral_constant<int, 0>());
                barrier();
                // The last block's products between the reads of the next step's first block (past the last step:
                // zeros) and the loads of the step after it.
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                    if (n < 2) {
                        read_one(fa, stage ^ 1, 0, order[2 * n]);
                        read_one(fa, stage ^ 1, 0, order[2 * n + 1]);
                        read_scale(sn, stage ^ 1, order[2 * n]);
                        read_scale(sn, stage ^ 1, order[2 * n + 1]);
                    } else {
                        read_one(fa, stage ^ 1, 0, order[n + 2]);
                        read_scale(sn, stage ^ 1, order[n + 2]);
                    }
                    mfma(fb, sc, Three(), n, 0);
                    mfma(fb, sc, Three(), n, 1);
                    issue(kt + 2, n);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
        }
        wait_loads_all();   // the zeros past the last step
        lds_barrier();      // and the reads of them
    }
    epilogue<MODE, EPI, kThreadsMfma, kWaveY>(p, t, lds, acc, wx, wy, L);
}

// Short products: few rows a group, where a tile of 256 rows is mostly empty, or
// (the weights' gradients) few steps of K, where nothing covers the loads'
// latency and the stores of the one block of a CU.  A block computes 256 columns by 128 rows on
// four waves of 128 x 64, and two blocks share a CU: one's loads and stores run
// under the other's products.  It reads a half more bytes a product.  A K step is 128 codes, 64 bytes
// a row; three stages, so a step's loads have two steps to land.
//
// us of gg_mx4_kernel / this one, with ragged groups around the mean:
//   rows a group    64 groups, 2816 x 2048                    8 groups, 28672 x 4096
//                   forward   back      weights' gradient     forward     back        weights' gradient
//     32 (8: 16)    50 / 37   43 / 37   228 / 207             123 / 105   164 / 155    516 / 425
//     96 (8: 64)    56 / 48   50 / 51   232 / 211             136 / 120   169 / 162    530 / 443
//    128            62 / 56   53 / 53   244 / 228             148 / 161   182 / 170    545 / 485
//    256            93 / 97   86 / 89   277 / 263             200 / 212   211 / 274    610 / 575
//   1024           294 / 301 271 / 287  445 / 436             570 / 642   593 / 694    950 / 902
//   2048                                                     1108 / 1234 1027 / 1210  1374 / 1394
// so it takes row-grouped products of up to 96 rows a group and weights' gradients of up to 1024.  The
// latter's stores alone take 121 us of the 64 groups' 738 MB (6.1 TB/s); a tile's loads, which its one step waits
// for, are what is left.  Tiles of a group on one XCD: 211 -> 215 at 96 rows, 902 -> 1016 at 1024.
constexpr int kShortRows = 96, kShortSum = 1024;   // mean rows of a group: of a row-grouped product, of a weights' gradient
constexpr int kS4Waves = 4, kS4Threads = 64 * kS4Waves;
constexpr int kS4X = 256, kS4Y = 128;
constexpr int kS4K = 128, kS4Blocks = kS4K / 32;
constexpr int kS4TileX = kS4X * kS4K / 2, kS4TileY = kS4Y * kS4K / 2;   // bytes of codes
constexpr int kS4ScaleX = kS4X * 4, kS4ScaleY = 1024;   // Y's 512 bytes take the room of a whole load
constexpr int kS4Stage = kS4TileX + kS4TileY + kS4ScaleX + kS4ScaleY;
constexpr int kS4Stages = 3;
constexpr int kS4Lds = kS4Stages * kS4Stage;
static_assert(2 * kS4Lds <= 163840 && 64 * kEpPitchF * 4 <= kS4Lds, "two blocks a CU");

// Position of 16-byte chunk c (0..3) of row r in a stage of 64-byte rows: c ^ ((r >> 2) & 3), so the 16 rows of one
// ds_read_b128 hit 16 distinct bank slots.
__device__ __forceinline__ uint32_t s4_off(int row, int chunk) {
    return static_cast<uint32_t>(row * 64 + ((chunk ^ ((row >> 2) & 3)) << 4));
}

template <int MODE, int EPI>
__global__ __launch_bounds__(kS4Threads, 2) void gg_mx4_short_kernel(Mx4Gemm q) {
    const Params& p = q.p;
    __shared__ __align__(1024) uint8_t lds[kS4Lds];
    Tile t;
    if (find_tile<MODE>(p, x_per_tile<EPI>(), kS4Y, blockIdx.x, &t) != kTileOk) return;
    t.g = __builtin_amdgcn_readfirstlane(t.g);
    t.x0 = __builtin_amdgcn_readfirstlane(t.x0);
    t.x_lim = __builtin_amdgcn_readfirstlane(t.x_lim);
    t.y0 = __builtin_amdgcn_readfirstlane(t.y0);
    t.y_lim = __builtin_amdgcn_readfirstlane(t.y_lim);
    t.row0 = __builtin_amdgcn_readfirstlane(static_cast<int>(t.row0));
    const int g = t.g;
    const int L = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wx = wave & 1, wy = wave >> 1;

    // Blocks of 32 to sum over, and the first of them in the operands' rows (a multiple of four).
    int blocks = p.K, first = 0;
    if constexpr (MODE == kWgrad) {
        const Mx4Groups m = mx4_groups(p.offsets, p.G, p.rows_cap);
        blocks = (__builtin_amdgcn_readlane(m.count, g) + 31) / 32;
        first = __builtin_amdgcn_readlane(m.pad_begin, g) / 32;
        blocks = min(blocks, max(0, p.K - first));   // p.K: blocks of all places
    }
    const int nk = (blocks + kS4Blocks - 1) / kS4Blocks;

    const uint32_t lda = static_cast<uint32_t>(p.lda), ldb = static_cast<uint32_t>(p.ldb);
    const int64_t yfirst = tile_first_row<MODE>(t);
    const Rsrc ry = make_dma_rsrc(static_cast<const uint8_t*>(p.a[0]) + yfirst * p.lda,
                                  static_cast<int64_t>(min(t.y_lim, kS4Y)) * p.lda);
    const uint8_t* X = static_cast<const uint8_t*>(p.b[0]) + (MODE == kWgrad ? 0 : g * q.x_codes);
    const Rsrc rx = make_dma_rsrc(X, q.x_rows * p.ldb);
    const int64_t all_words = (static_cast<int64_t>(p.K) + 3) / 4;
    const Rsrc rys = make_dma_rsrc(q.ys, all_words * q.y_rows * 4);
    const Rsrc rxs = make_dma_rsrc(q.xs + (MODE == kWgrad ? 0 : g * q.x_scales), all_words * q.x_rows * 4);

    const auto y_row = [&](int r) { return min(r, t.y_lim - 1); };
    const auto x_row = [&](int r) {
        if (is_swiglu_fwd(EPI)) {
            // 256 weight rows = [gate 64 | up 64] for each half of 128 activation columns.
            const int half = r >> 7, qq = r & 127;
            int col = t.x0 + half * 64 + (qq & 63);
            col = col < p.f ? col : 0;
            return qq < 64 ? col : p.f + col;
        }
        const int n = t.x0 + r;
        return n < p.N ? n : 0;
    };
    // Lane L of load j of wave w fills 16 bytes of row 16 (4 j + w) + L / 4: the block that belongs at place L % 4
    // (s4_off); it is the same for every j.
    const int chunk = (L & 3) ^ (L >> 4);
    constexpr int kLoadsX = kS4TileX / 1024 / kS4Waves, kLoadsY = kS4TileY / 1024 / kS4Waves;
    uint32_t vx[kLoadsX], vy[kLoadsY];
#pragma unroll
    for (int j = 0; j < kLoadsX; ++j)
        vx[j] = static_cast<uint32_t>(x_row((j * kS4Waves + wave) * 16 + (L >> 2))) * ldb + chunk * 16;
#pragma unroll
    for (int j = 0; j < kLoadsY; ++j)
        vy[j] = static_cast<uint32_t>(y_row((j * kS4Waves + wave) * 16 + (L >> 2))) * lda + chunk * 16;
    // Scales: waves 0 and 2 load the step's words of X, 1 and 3 of Y (the same bytes twice, so that every wave has as
    // many loads), four rows a lane.  Rows past the tile: those that follow, or zeros; their outputs are dropped.
    const bool sx_wave = (wave & 1) == 0;
    const uint32_t vs = sx_wave ? static_cast<uint32_t>(x_row(4 * L)) * 4
                                : L < kS4Y / 4 ? static_cast<uint32_t>(static_cast<int>(yfirst) + 4 * L) * 4 : kOutOfRange;
    const Rsrc rs = sx_wave ? rxs : rys;
    const uint32_t s_rows = static_cast<uint32_t>(sx_wave ? q.x_rows : q.y_rows);

    const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(lds));
    // Load n of this wave's of step `step` into stage `stage`: blocks past the last (all of them, past the last step)
    // read as zeros, and so do their scales (a scale that is not this group's must not meet zero codes: it may be NaN).
    constexpr int kLoads = kLoadsX + kLoadsY + 1;
    auto issue = [&](int step, int stage, int n) {
        const uint32_t base = lds0 + stage * kS4Stage + wave * 1024;
        const uint32_t soff = static_cast<uint32_t>(first * 16 + step * (kS4K / 2));
        const uint32_t off = chunk < blocks - step * kS4Blocks ? 0u : kOutOfRange;
        if (n < kLoadsY) {
            dma16(ry, vy[n] | off, soff, base + kS4TileX + n * kS4Waves * 1024);
        } else if (n < kLoadsY + kLoadsX) {
            dma16(rx, vx[n - kLoadsY] | off, soff, base + (n - kLoadsY) * kS4Waves * 1024);
        } else {
            const bool have = step < nk;
            dma16(rs, vs | (have ? 0u : kOutOfRange), (have ? static_cast<uint32_t>(first / 4 + step) * 4u : 0u) * s_rows,
                  lds0 + stage * kS4Stage + kS4TileX + kS4TileY + (sx_wave ? 0 : kS4ScaleX));
        }
    };
    auto wait_lds = [](auto n_c) {               // vmcnt(n) lgkmcnt(0)
        constexpr int n = decltype(n_c)::value;
        __builtin_amdgcn_s_waitcnt(0x0070 | (n & 15) | ((n >> 4) << 14));
    };
    auto barrier = [] {
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };

    Acc16<64> acc;
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc.v[i][j] = f32x4_t{};
    // A step is one k128 block of eight slots: X fragment i (16 rows) with the four Y fragments.  X fragments and their
    // scales come three slots ahead into a ring of four.  Lane L of a fragment has row L % 16 and the 32 codes of block
    // L / 16, and that block's scale.  Rows 16 apart are whole turns of the places' pattern: fragment i of the wave's X
    // rows lies at px + 1024 i (its scales at sx + 64 i), of its Y rows at py + 1024 j.
    struct Frag {
        i32x4_t v;
        uint32_t s;
    };
    const int quad = L >> 4;
    const uint32_t place = s4_off(L & 15, quad);
    const uint32_t px = static_cast<uint32_t>(wx * 128 * 64) + place, py = static_cast<uint32_t>(kS4TileX + wy * 64 * 64) + place;
    const uint32_t sx = static_cast<uint32_t>(kS4TileX + kS4TileY + (wx * 128 + (L & 15)) * 4 + quad);
    const uint32_t sy = static_cast<uint32_t>(kS4TileX + kS4TileY + kS4ScaleX + (wy * 64 + (L & 15)) * 4 + quad);
    auto read_x = [&](int stage, int i) {
        Frag f;
        f.v = *reinterpret_cast<const i32x4_t*>(lds + (stage * kS4Stage + px) + i * 1024);
        f.s = lds[(stage * kS4Stage + sx) + i * 64];
        return f;
    };
    auto read_y = [&](int stage, int j) {
        Frag f;
        f.v = *reinterpret_cast<const i32x4_t*>(lds + (stage * kS4Stage + py) + j * 1024);
        f.s = lds[(stage * kS4Stage + sy) + j * 64];
        return f;
    };
    auto wide = [](i32x4_t v) { return __builtin_shufflevector(v, v, 0, 1, 2, 3, -1, -1, -1, -1); };
    auto mfmas = [&](const Frag& x, const Frag (&y)[4], int i) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            acc.v[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wide(x.v), wide(y[j].v), acc.v[i][j], kFmtE2m1,
                                                                        kFmtE2m1, 0, x.s, 0, y[j].s);
    };
    using Pending = std::integral_constant<int, (kS4Stages - 2) * kLoads>;   // the steps past the next stay in flight

    if (nk > 0) {
#pragma unroll
        for (int n = 0; n < kS4Stages * kLoads; ++n) issue(n / kLoads, n / kLoads, n % kLoads);
        wait_lds(std::integral_constant<int, (kS4Stages - 1) * kLoads>());
        barrier();
        const bool idle = wy * 64 >= t.y_lim;   // such a wave only keeps the loads and the barriers going
        Frag xr[4], yr[2][4];
        if (!idle) {
#pragma unroll
            for (int j = 0; j < 4; ++j) yr[0][j] = read_y(0, j);
#pragma unroll
            for (int n = 0; n < 3; ++n) xr[n] = read_x(0, n);
        }
        int stage = 0;
        const auto step = [&](int kt, auto c_c) {
            constexpr int c = decltype(c_c)::value;
            const int next = stage + 1 == kS4Stages ? 0 : stage + 1;
            if (!idle) {
#pragma unroll
                for (int n = 0; n < 5; ++n) {
                    xr[(n + 3) & 3] = read_x(stage, n + 3);
                    mfmas(xr[n & 3], yr[c], n);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            // The next step's loads have landed, every read of this stage is done.
            wait_lds(Pending());
            barrier();
            // The last three slots between the reads of the next step's first fragments and the loads into this stage.
#pragma unroll
            for (int n = 5; n < 8; ++n) {
                if (!idle) {
                    if (n < 7) {
                        yr[c ^ 1][2 * (n - 5)] = read_y(next, 2 * (n - 5));
                        yr[c ^ 1][2 * (n - 5) + 1] = read_y(next, 2 * (n - 5) + 1);
                    }
                    mfmas(xr[n & 3], yr[c], n);
                    xr[(n - 5) & 3] = read_x(next, n - 5);
                }
#pragma unroll
                for (int i = 0; i < kLoads; ++i)
                    if (i * 3 / kLoads == n - 5) issue(kt + kS4Stages, stage, i);
                __builtin_amdgcn_sched_barrier(0);
            }
            stage = next;
        };
        for (int kt = 0; kt < nk; kt += 2) {   // past the last step all is zeros
            step(kt, std::integral_constant<int, 0>());
            step(kt + 1, std::integral_constant<int, 1>());
        }
        wait_loads_all();   // the zeros past the last step
    }
    // 64 rows at a time through LDS (they fit beside another block's), so that rows leave in 512 contiguous bytes.
    t.y_lim = min(t.y_lim, kS4Y);
    float* ep = reinterpret_cast<float*>(lds);
#pragma unroll
    for (int part = 0; part < 2; ++part) {
        if (64 * part >= t.y_lim) break;
        AuxHalf<EPI, kS4Threads, 64> aux;
        load_aux_half<MODE, EPI, kS4Threads, 64>(p, t, 64 * part, aux);
        lds_barrier();   // every read of what the stage held is done
        if (wy == part) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    *reinterpret_cast<f32x4_t*>(ep + (16 * j + (L & 15)) * kEpPitchF + wx * 128 + 16 * i + 4 * quad) =
                        acc.v[i][j];
        }
        lds_barrier();
        epilogue_half<MODE, EPI, kS4Threads, false, 64>(p, t, ep, 64 * part, aux);
    }
}

// ------------------------------------------------------------------ bfloat16 rows

// Products of bfloat16 token rows with weights in 4 bits: serving, from one
// token on.  With few rows the weights' bytes are all that counts (17 / 32 of a byte
// a weight), so they go from memory straight into registers, every byte once
// a row tile, are made bfloat16 there (exactly: two codes a conversion) and
// multiplied by v_mfma_f32_16x16x32_bf16: lane L holds weight row L % 16, and of
// 128 reduction places block L / 16 whole, 16 bytes, whose four words make
// four products over places 8 i .. + 7 of every block; token rows (the
// product's columns) are read to match.  A wave has NT x 16 weight rows and 16
// token rows; the block's WK waves share the reduction in turns of 256 places (a
// 128-byte line of codes a weight row) and add their sums through LDS in wave order.
//
// Which kernel, by the mean rows of a group (us of fc1 + fc2, SwiGLU, the
// experts of 4096 x 14336 or 2048 x 1408; "few" is this kernel, the others mx4_tile_kernel):
//   8 experts  rows a group  1: few  71 +  41, 32-row tiles  79 +  45
//                            2:     113 +  54               113 +  47
//                           12:     145 +  83               118 +  49, 64-row tiles 122 +  77
//                           32:     275 + 141               137 +  80               132 +  86
//                           64:     485 + 252               216 + 132               183 + 112
//   64 experts               1:      22 +  14                23 +  11
//                            3:      40 +  24                36 +  17
//                           24:      87 +  42                49 +  26                44 +  25
// so few for one, tiles of 32 rows up to 32, then of 64.  A long reduction is shared by eight waves:
// one token's fc2 23 -> 19 us of 14336 places, while its fc1 of 4096 takes 39 us so and 31 on four; in 32-row
// tiles two waves a column share: fc2 68 -> 49 us of 12 rows, 74 -> 53 of 24.  64-row tiles do not share: 181 -> 235 us of 128.
constexpr int kRowsWaves = 4, kRowsThreads = 64 * kRowsWaves, kRowsK = 256;
constexpr int kRowsLongK = 8192;
constexpr int kRowsFew = 1, kRowsTile32 = 32;   // mean rows of a group

struct Mx4Rows {
    const uint16_t* x;          // [rows, K]
    const int32_t* offsets;     // [G + 1]
    const uint8_t *codes, *scales;   // G weights of N (SwiGLU: 2 N) rows
    uint16_t* out;              // [rows, N]
    int64_t rows;
    int G, N, K, blocks;        // blocks: of 32 of a weight row
    int64_t w_codes, w_scales;  // bytes from one weight to the next
    int w_rows;                 // rows of a weight
};

// A block's group (-1: none is left), first row, rows from there on, and first column.  Row tiles of a weight's rows are
// neighbours (on one XCD), so that they share its bytes in the L2.
struct RowsBlock {
    int g, n0, r_lim;
    int64_t row0;
};
__device__ __forceinline__ RowsBlock rows_block(const Mx4Rows& p, int tile_rows, int tile_cols) {
    const int L = threadIdx.x & 63;
    int g_first = 0, g_rows = 0;
    if (L < p.G) {
        g_first = min(max(p.offsets[L], 0), static_cast<int>(p.rows));
        g_rows = max(min(p.offsets[L + 1], static_cast<int>(p.rows)) - g_first, 0);
    }
    const uint32_t ncb = static_cast<uint32_t>((p.N + tile_cols - 1) / tile_cols);
    const uint32_t g_tiles = static_cast<uint32_t>((g_rows + tile_rows - 1) / tile_rows) * ncb;
    uint32_t g_end = g_tiles;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint32_t v = __shfl_up(g_end, d);
        if (L >= d) g_end += v;
    }
    const uint32_t total = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(g_end), 63));
    if (blockIdx.x >= total) return {-1, 0, 0, 0};
    uint32_t id = xcd_remap(blockIdx.x, total);
    const int g = __ffsll(static_cast<unsigned long long>(__ballot(g_end > id))) - 1;
    id -= static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(g_end - g_tiles), g & 63));
    if (g < 0 || id >= static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(g_tiles), g)))
        return {-1, 0, 0, 0};   // groups that overlap so far that their tiles' number wraps
    const int n_rows = __builtin_amdgcn_readlane(g_rows, g);
    const uint32_t rt_n = static_cast<uint32_t>((n_rows + tile_rows - 1) / tile_rows);
    const int r0 = static_cast<int>(id % rt_n) * tile_rows;
    return {g, static_cast<int>(id / rt_n) * tile_cols, n_rows - r0,
            __builtin_amdgcn_readlane(g_first, g) + static_cast<int64_t>(r0)};
}

// Lane L has columns 4 (L / 16) .. + 3 of row L % 16 of each 16 x 16 tile; SwiGLU: gate tiles, then up tiles.
template <int NT, int RT, int EPI>
__device__ __forceinline__ void rows_store(const Mx4Rows& p, const f32x4_t (&acc)[NT][RT], int n0, int64_t row0, int r_lim,
                                           int q, int m) {
    constexpr bool kGlu = EPI == kEpiSwigluAct;
    constexpr int kCols = kGlu ? NT / 2 : NT;
#pragma unroll
    for (int n = 0; n < kCols; ++n)
#pragma unroll
        for (int j = 0; j < RT; ++j) {
            const int col = n0 + 16 * n + 4 * q;
            if (16 * j + m >= r_lim || col >= p.N) continue;
            float v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                v[e] = acc[n][j][e];
                if constexpr (kGlu) v[e] = silu_f(v[e]) * acc[n + kCols][j][e];
                if constexpr (EPI == kEpiGeluAct) v[e] = gelu_f(v[e]);
            }
            store_bf16x4(p.out + (row0 + 16 * j + m) * p.N + col, v[0], v[1], v[2], v[3]);
        }
}

template <int NT, int RT, int WK, int EPI>
__global__ __launch_bounds__(64 * WK) void mx4_rows_kernel(Mx4Rows p) {
    constexpr bool kGlu = EPI == kEpiSwigluAct;
    constexpr int kCols = kGlu ? NT / 2 : NT;   // 16-wide output tiles
    static_assert(!kGlu || NT % 2 == 0, "gate and up tiles in pairs");
    __shared__ float4 part[WK - 1][NT * RT][64];
    const int L = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

    const RowsBlock at = rows_block(p, 16 * RT, 16 * kCols);
    if (at.g < 0) return;
    const int n0 = at.n0, r_lim = at.r_lim, g = at.g;
    const int64_t row0 = at.row0;

    const int q = L >> 4, m = L & 15;
    const uint8_t* codes = p.codes + g * p.w_codes;
    const uint32_t* scales = reinterpret_cast<const uint32_t*>(p.scales + g * p.w_scales);
    int w_row[NT];
#pragma unroll
    for (int i = 0; i < NT; ++i) {
        const int c = n0 + 16 * (i % kCols) + m;
        w_row[i] = min(c, p.N - 1) + (i >= kCols ? p.N : 0);   // past the last column: its values are dropped
    }
    const uint16_t* xr[RT];
#pragma unroll
    for (int j = 0; j < RT; ++j) xr[j] = p.x + (row0 + 16 * j + m) * p.K;   // rows past the tile's are not read

    f32x4_t acc[NT][RT] = {};
    struct Turn {
        u32x4v_t w[NT][2];
        uint32_t s[NT][2];
    };
    // Of the 256 places from k on this lane's two blocks; past the weight's blocks codes of zero under scale 1.
    const auto load_w = [&](Turn& t, int k) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const int b = k / 32 + 4 * c + q;
            const bool have = b < p.blocks;
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                t.w[i][c] = u32x4v_t{0u, 0u, 0u, 0u};
                t.s[i][c] = 127u << (8 * q);
                if (have) {
                    t.w[i][c] = *reinterpret_cast<const u32x4v_t*>(codes + (static_cast<int64_t>(w_row[i]) * p.blocks + b) * 16);
                    t.s[i][c] = scales[static_cast<int64_t>(b >> 2) * p.w_rows + w_row[i]];
                }
            }
        }
    };
    Turn cur, nxt;
    int k = wave * kRowsK;
    load_w(cur, k);
    for (; k < p.K; k += WK * kRowsK) {
        load_w(nxt, k + WK * kRowsK);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            u32x4v_t xv[RT][4];
#pragma unroll
            for (int j = 0; j < RT; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int at = k + 128 * c + 32 * q + 8 * i;
                    xv[j][i] = u32x4v_t{0u, 0u, 0u, 0u};
                    if (at < p.K && 16 * j + m < r_lim) xv[j][i] = *reinterpret_cast<const u32x4v_t*>(xr[j] + at);
                }
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const uint32_t e = cur.s[n][c] >> (8 * q) & 255u;
                const float s = e == 255u ? __builtin_nanf("") : mx4_scale(e);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t w = cur.w[n][c][i];
                    u32x4v_t v;
                    v[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 0));
                    v[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 1));
                    v[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 2));
                    v[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 3));
#pragma unroll
                    for (int j = 0; j < RT; ++j)
                        acc[n][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, v),
                                                                            __builtin_bit_cast(bf16x8_t, xv[j][i]),
                                                                            acc[n][j], 0, 0, 0);
                }
            }
        }
        cur = nxt;
    }
    // Wave 0 adds the others' sums and stores: lane L has columns 4 (L / 16) .. + 3 of row L % 16 of each tile.
    if (wave > 0) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int j = 0; j < RT; ++j)
                part[wave - 1][n * RT + j][L] = make_float4(acc[n][j][0], acc[n][j][1], acc[n][j][2], acc[n][j][3]);
    }
    __syncthreads();
    if (wave > 0) return;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < RT; ++j)
#pragma unroll
            for (int w = 0; w < WK - 1; ++w) {
                const float4 v = part[w][n * RT + j][L];
                acc[n][j][0] += v.x, acc[n][j][1] += v.y, acc[n][j][2] += v.z, acc[n][j][3] += v.w;
            }
    rows_store<NT, RT, EPI>(p, acc, n0, row0, r_lim, q, m);
}

// More rows: the token rows go through LDS, 128 places a step, for four waves
// that each have NT x 16 weight rows of their own and all RT x 16 token rows, so
// a weight is read and made bfloat16 once a row tile and a token row once a
// block.  Two stages; the next step's rows and weights are on their way while one is
// multiplied.  The places of a lane's products are those of mx4_rows_kernel.  The reduction runs in
// one piece, or in two (WK) on twice the waves, every other step each.  64 rows of the 64 experts above 37 + 18 us
// (197 + 98 MB of weights: 5.3 TB/s); 1024 rows of the 8: 272 + 180 us, one
// conversion a matrix instruction.  Weights two steps ahead: 64 rows of the
// 8 experts 118 -> 112 us, but 512 rows 189 -> 260, its registers cost a wave a SIMD; not kept.
constexpr int kTileK = 128;

template <int NT, int RT, int WK, int EPI>
__global__ __launch_bounds__(WK * kRowsThreads) void mx4_tile_kernel(Mx4Rows p) {
    constexpr bool kGlu = EPI == kEpiSwigluAct;
    constexpr int kCols = kGlu ? NT / 2 : NT;   // 16-wide output tiles a wave
    constexpr int kStage = 16 * RT * kTileK * 2, kLoads = RT;   // bytes; 1 KB loads a wave (4 rows each)
    static_assert(kLoads * kRowsWaves * 1024 == kStage, "the waves' loads fill a stage");
    constexpr int kJoin = WK > 1 ? kRowsWaves * NT * RT * 64 * 16 : 0;   // bytes of one share's sums
    __shared__ __align__(1024) uint8_t lds_all[WK * 2 * kStage > kJoin ? WK * 2 * kStage : kJoin];
    const int L = threadIdx.x & 63, all_wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wave = all_wave % kRowsWaves, share = all_wave / kRowsWaves;
    uint8_t* lds = lds_all + share * 2 * kStage;
    const RowsBlock at = rows_block(p, 16 * RT, 16 * kCols * kRowsWaves);
    if (at.g < 0) return;
    const int n0 = at.n0 + wave * 16 * kCols, r_lim = at.r_lim;
    const int64_t row0 = at.row0;
    const int q = L >> 4, m = L & 15;
    const uint8_t* codes = p.codes + at.g * p.w_codes;
    const uint32_t* scales = reinterpret_cast<const uint32_t*>(p.scales + at.g * p.w_scales);
    int w_row[NT];
#pragma unroll
    for (int i = 0; i < NT; ++i) {
        const int c = n0 + 16 * (i % kCols) + m;
        w_row[i] = min(c, p.N - 1) + (i >= kCols ? p.N : 0);   // past the last column: its values are dropped
    }
    // 256 bytes of a token row a step, 16-byte chunk c at place c ^ (row % 16): the 16 rows of a fragment meet all
    // banks.  Load j of wave w fills rows 4 (4 j + w) .. + 3, lane L place L % 16 of row L / 16 of them.
    const Rsrc rx = make_dma_rsrc(p.x + row0 * p.K, static_cast<int64_t>(min(r_lim, 16 * RT)) * p.K * 2);
    uint32_t vo[kLoads];
    int kc[kLoads];   // the chunk's first place
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
        const int row = 4 * (kRowsWaves * j + wave) + q;
        kc[j] = 8 * ((L & 15) ^ (row & 15));
        vo[j] = row < r_lim ? static_cast<uint32_t>(row) * static_cast<uint32_t>(p.K * 2) + kc[j] * 2 : kOutOfRange;
    }
    const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(lds));
    const auto load_x = [&](int k, int stage) {
#pragma unroll
        for (int j = 0; j < kLoads; ++j)
            dma16(rx, vo[j] | (k + kc[j] < p.K ? 0u : kOutOfRange), static_cast<uint32_t>(k) * 2,
                  lds0 + stage * kStage + (kRowsWaves * j + wave) * 1024);
    };
    struct Codes {
        u32x4v_t w[NT];
        uint32_t s[NT];
    };
    const auto load_w = [&](Codes& t, int k) {
        const int b = k / 32 + q;
        const bool have = b < p.blocks;
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            t.w[i] = u32x4v_t{0u, 0u, 0u, 0u};
            t.s[i] = 127u << (8 * q);
            if (have) {
                t.w[i] = *reinterpret_cast<const u32x4v_t*>(codes + (static_cast<int64_t>(w_row[i]) * p.blocks + b) * 16);
                t.s[i] = scales[static_cast<int64_t>(b >> 2) * p.w_rows + w_row[i]];
            }
        }
    };
    // Fragment (i, j): row 16 j + m, chunk 4 q + i of the stage.
    const auto read_x = [&](int stage, int slot) {
        const int i = slot / RT, j = slot % RT;
        return *reinterpret_cast<const u32x4v_t*>(lds + stage * kStage + (16 * j + m) * 256 + (((4 * q + i) ^ m) << 4));
    };
    f32x4_t acc[NT][RT] = {};
    Codes cur, nxt;
    load_x(share * kTileK, 0);
    load_w(cur, share * kTileK);
    int stage = 0;
    for (int k0 = 0; k0 < p.K; k0 += WK * kTileK, stage ^= 1) {
        const int k = k0 + share * kTileK;   // past K: zeros
        __builtin_amdgcn_s_waitcnt(0x0F70);   // vmcnt(0): this step's rows, and its weights
        __syncthreads();                      // all waves' rows; the other stage has been read
        load_x(k + WK * kTileK, stage ^ 1);
        load_w(nxt, k + WK * kTileK);
        u32x4v_t ring[4];
#pragma unroll
        for (int n = 0; n < 3; ++n) ring[n] = read_x(stage, n);
        float s[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const uint32_t e = cur.s[n] >> (8 * q) & 255u;
            s[n] = e == 255u ? __builtin_nanf("") : mx4_scale(e);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            u32x4v_t v[NT];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const uint32_t w = cur.w[n][i];
                v[n][0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s[n], 0));
                v[n][1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s[n], 1));
                v[n][2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s[n], 2));
                v[n][3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s[n], 3));
            }
#pragma unroll
            for (int j = 0; j < RT; ++j) {
                const int slot = i * RT + j;
                if (slot + 3 < 4 * RT) ring[(slot + 3) & 3] = read_x(stage, slot + 3);
#pragma unroll
                for (int n = 0; n < NT; ++n)
                    acc[n][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, v[n]),
                                                                        __builtin_bit_cast(bf16x8_t, ring[slot & 3]),
                                                                        acc[n][j], 0, 0, 0);
            }
        }
        cur = nxt;
    }
    wait_loads_all();   // no load into LDS outlives the block
    if constexpr (WK == 2) {
        // The second share's sums go to the first, wave by wave.
        float4(*part)[64] = reinterpret_cast<float4(*)[64]>(lds_all) + wave * NT * RT;
        __syncthreads();
        if (share == 1) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int j = 0; j < RT; ++j)
                    part[n * RT + j][L] = make_float4(acc[n][j][0], acc[n][j][1], acc[n][j][2], acc[n][j][3]);
        }
        __syncthreads();
        if (share == 1) return;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int j = 0; j < RT; ++j) {
                const float4 v = part[n * RT + j][L];
                acc[n][j][0] += v.x, acc[n][j][1] += v.y, acc[n][j][2] += v.z, acc[n][j][3] += v.w;
            }
    }
    rows_store<NT, RT, EPI>(p, acc, n0, row0, r_lim, q, m);
}

template <int MODE, int EPI>
int launch_mx4(const Mx4Gemm& q, int64_t nb, hipStream_t s) {
    hipLaunchKernelGGL((gg_mx4_kernel<MODE, EPI>), dim3(static_cast<unsigned>(nb)), dim3(kThreadsMfma), 0, s, q);
    return check_launch("gg_mx4_kernel");
}
template <int MODE, int EPI>
int launch_short(const Mx4Gemm& q, int64_t nb, hipStream_t s) {
    hipLaunchKernelGGL((gg_mx4_short_kernel<MODE, EPI>), dim3(static_cast<unsigned>(nb)), dim3(kS4Threads), 0, s, q);
    return check_launch("gg_mx4_short_kernel");
}

int64_t blocks_of(int64_t len) { return (len + 31) / 32; }
int64_t words_of(int64_t len) { return (len + 127) / 128; }

}  // namespace
}  // namespace rhp

using namespace rhp;

extern "C" int rhp_mx4_gemm(int epi, int G, const int32_t* offsets, int64_t rows, int N, int K, const void* a_codes,
                            const void* a_scales, const void* w_codes, const void* w_scales, void* out, void* act_out,
                            const void* aux, hipStream_t stream) {
    clear_error();
    RHP_REQUIRE(G >= 1 && G <= kMaxG, "rhp_mx4_gemm: 1 to 64 groups per call");
    RHP_REQUIRE(epi >= kEpiStore && epi <= kEpiGeluBwd, "rhp_mx4_gemm: the epilogue must be 0 to 4");
    RHP_REQUIRE(rows >= 0 && N >= 1 && N < (1 << 30) && K >= 1, "rhp_mx4_gemm: bad sizes");
    RHP_REQUIRE(N % 8 == 0, "rhp_mx4_gemm: N must be a multiple of 8");
    if (rows == 0) return 0;
    const bool fwd = epi == kEpiSwigluFwd || epi == kEpiGeluFwd, bwd = epi == kEpiSwigluBwd || epi == kEpiGeluBwd;
    RHP_REQUIRE(offsets && a_codes && a_scales && w_codes && w_scales && (out || fwd), "rhp_mx4_gemm: null pointer");
    RHP_REQUIRE((act_out != nullptr) == fwd && (aux != nullptr) == bwd,
                "rhp_mx4_gemm: forward activations write act_out, backward ones read aux, others neither");
    RHP_REQUIRE(aligned16(a_codes) && aligned16(a_scales) && aligned16(w_codes) && aligned16(w_scales) &&
                    aligned16(out) && aligned16(act_out) && aligned16(aux),
                "rhp_mx4_gemm: operands and outputs must be 16-byte aligned");
    const int64_t kb = blocks_of(K), lim = int64_t(1) << 31;
    const int64_t w_rows = epi == kEpiSwigluFwd ? 2 * int64_t(N) : N;
    const int64_t wide = epi == kEpiSwigluFwd || epi == kEpiSwigluBwd ? 2 * int64_t(N) : N;   // columns of out and aux
    RHP_REQUIRE(rows < lim - kTile && kTile * kb * 16 < lim && w_rows * kb * 16 < lim && wide * 2 * kTile < lim &&
                    words_of(K) * rows * 4 < lim && words_of(K) * w_rows * 4 < lim,
                "rhp_mx4_gemm: a weight, 256 rows of every operand and all scales of either must each stay below 2 GiB");
    Mx4Gemm q{};
    q.p.a[0] = a_codes;
    q.p.b[0] = w_codes;
    for (int g = 0; g < G; ++g) {
        q.p.c[g] = out;
        q.p.c2[g] = act_out;
        q.p.aux[g] = aux;
    }
    q.p.offsets = offsets;
    q.p.G = G;
    q.p.rows_from_offsets = 1;
    q.p.N = N;
    q.p.K = static_cast<int>(kb);
    q.p.lda = q.p.ldb = static_cast<int>(kb * 16);
    q.p.ldc = q.p.ldaux = static_cast<int>(wide);
    q.p.ldc2 = N;
    q.p.f = N;
    q.p.rows_cap = static_cast<int>(rows);
    q.ys = static_cast<const uint8_t*>(a_scales);
    q.xs = static_cast<const uint8_t*>(w_scales);
    q.x_codes = w_rows * kb * 16;
    q.x_scales = words_of(K) * w_rows * 4;
    q.y_rows = rows;
    q.x_rows = w_rows;
    const bool brief = rows <= int64_t(kShortRows) * G;
    const int xt = epi == kEpiSwigluFwd ? x_per_tile<kEpiSwigluFwd>() : kTile, yt = brief ? kS4Y : kTile;
    const int64_t nb = ((rows + yt - 1) / yt + G) * ((N + xt - 1) / xt);
    RHP_REQUIRE(nb < lim, "rhp_mx4_gemm: too many tiles");
    const auto go = [&](auto e) {
        return brief ? launch_short<kFwd, decltype(e)::value>(q, nb, stream) : launch_mx4<kFwd, decltype(e)::value>(q, nb, stream);
    };
    using std::integral_constant;
    switch (epi) {
        case kEpiSwigluFwd: return out ? go(integral_constant<int, kEpiSwigluFwd>()) : go(integral_constant<int, kEpiSwigluAct>());
        case kEpiGeluFwd: return out ? go(integral_constant<int, kEpiGeluFwd>()) : go(integral_constant<int, kEpiGeluAct>());
        case kEpiSwigluBwd: return go(integral_constant<int, kEpiSwigluBwd>());
        case kEpiGeluBwd: return go(integral_constant<int, kEpiGeluBwd>());
        default: return go(integral_constant<int, kEpiStore>());
    }
}

extern "C" int rhp_mx4_wgrad(int G, const int32_t* offsets, int64_t rows, int M, int N, const void* a_codes,
                             const void* a_scales, const void* b_codes, const void* b_scales, void* out,
                             hipStream_t stream) {
    clear_error();
    RHP_REQUIRE(G >= 1 && G <= kMaxG, "rhp_mx4_wgrad: 1 to 64 groups per call");
    RHP_REQUIRE(rows >= 0 && M >= 1 && N >= 1, "rhp_mx4_wgrad: bad sizes");
    RHP_REQUIRE(N % 8 == 0, "rhp_mx4_wgrad: N must be a multiple of 8");
    RHP_REQUIRE(offsets && out && aligned16(out), "rhp_mx4_wgrad: null pointer or unaligned output");
    const int64_t len = rhp_mx4_padded_rows(rows, G), kb = blocks_of(len), lim = int64_t(1) << 31;
    RHP_REQUIRE(len == 0 || (a_codes && a_scales && b_codes && b_scales), "rhp_mx4_wgrad: null pointer");
    RHP_REQUIRE(aligned16(a_codes) && aligned16(a_scales) && aligned16(b_codes) && aligned16(b_scales),
                "rhp_mx4_wgrad: operands must be 16-byte aligned");
    RHP_REQUIRE(rows < lim - 64 * 128 && (kTile + 1) * kb * 16 < lim && (N + int64_t(1)) * kb * 16 < lim &&
                    words_of(len) * std::max(M, N) * 4 < lim && int64_t(N) * 2 * kTile < lim,
                "rhp_mx4_wgrad: the operands' codes of b, 256 rows of a's and the scales must stay below 2 GiB");
    Mx4Gemm q{};
    q.p.a[0] = a_codes;
    q.p.b[0] = b_codes;
    for (int g = 0; g < G; ++g) q.p.c[g] = static_cast<uint16_t*>(out) + static_cast<int64_t>(g) * M * N;
    q.p.offsets = offsets;
    q.p.G = G;
    q.p.rows_from_offsets = 1;
    q.p.N = N;
    q.p.K = static_cast<int>(kb);
    q.p.Mo = M;
    q.p.lda = q.p.ldb = static_cast<int>(kb * 16);
    q.p.ldc = N;
    q.p.rows_cap = static_cast<int>(rows);
    q.ys = static_cast<const uint8_t*>(a_scales);
    q.xs = static_cast<const uint8_t*>(b_scales);
    q.y_rows = M;
    q.x_rows = N;
    const bool brief = rows <= int64_t(kShortSum) * G;
    const int64_t xt = (N + kTile - 1) / kTile, yt = brief ? (M + kS4Y - 1) / kS4Y : (M + kTile - 1) / kTile;
    const int64_t nb = wgrad_blocks(G, xt * yt);
    RHP_REQUIRE(nb < lim, "rhp_mx4_wgrad: too many tiles");
    return brief ? launch_short<kWgrad, kEpiStore>(q, nb, stream) : launch_mx4<kWgrad, kEpiStore>(q, nb, stream);
}

namespace {

template <int EPI>
int rows_gemm(const Mx4Rows& p, hipStream_t stream) {
    const int64_t busy = std::min<int64_t>(p.G, p.rows), mean = (p.rows + busy - 1) / busy;
    constexpr bool kGlu = EPI == kEpiSwigluAct;
    using std::integral_constant;
    // f(columns a wave's 16-wide tiles, row tiles): launches the kernel for blocks of `waves` waves along the columns.
    const auto grid = [&](int rows, int cols) { return std::min(p.rows, (p.rows + rows - 1) / rows + p.G) * ((p.N + cols - 1) / cols); };
    const auto few = [&](auto nt, auto rt) {
        constexpr int NT = decltype(nt)::value, RT = decltype(rt)::value;
        const int64_t nb = grid(16 * RT, 16 * (kGlu ? NT / 2 : NT));
        RHP_REQUIRE(nb < (int64_t(1) << 31), "rhp_mx4_rows_gemm: too many tiles");
        if (p.K >= kRowsLongK)
            hipLaunchKernelGGL((mx4_rows_kernel<NT, RT, 8, EPI>), dim3(static_cast<unsigned>(nb)), dim3(512), 0, stream, p);
        else
            hipLaunchKernelGGL((mx4_rows_kernel<NT, RT, 4, EPI>), dim3(static_cast<unsigned>(nb)), dim3(256), 0, stream, p);
        return check_launch("mx4_rows_kernel");
    };
    const auto many = [&](auto nt, auto rt) {
        constexpr int NT = decltype(nt)::value, RT = decltype(rt)::value;
        const int64_t nb = grid(16 * RT, 16 * kRowsWaves * (kGlu ? NT / 2 : NT));
        RHP_REQUIRE(nb < (int64_t(1) << 31), "rhp_mx4_rows_gemm: too many tiles");
        if constexpr (RT == 2) {
            if (p.K >= kRowsLongK) {
                hipLaunchKernelGGL((mx4_tile_kernel<NT, RT, 2, EPI>), dim3(static_cast<unsigned>(nb)), dim3(2 * kRowsThreads), 0, stream, p);
                return check_launch("mx4_tile_kernel");
            }
        }
        hipLaunchKernelGGL((mx4_tile_kernel<NT, RT, 1, EPI>), dim3(static_cast<unsigned>(nb)), dim3(kRowsThreads), 0, stream, p);
        return check_launch("mx4_tile_kernel");
    };
    // As many columns a wave as leave some two blocks a CU, or four of the first kernel, where many groups are empty: the
    // more, the less often the token rows are read.  One token's fc2 18 us on one 16-wide tile, 27 on four, 4 tokens' 41 on
    // two, 54 on four; 16 tokens' fc1 111 on one or two, 115 on four, 128 tokens' 151 and 137.
    const auto tiles16 = [&](int rows) {
        return std::min(p.rows, busy * ((mean + rows - 1) / rows)) * ((p.w_rows + 15) / 16);
    };
    const auto with_few = [&](auto rt) {
        const int64_t tiles = tiles16(16 * decltype(rt)::value);
        if (tiles >= 4 * 1024) return few(integral_constant<int, 4>(), rt);
        if (kGlu || tiles >= 2 * 1024) return few(integral_constant<int, 2>(), rt);
        return few(integral_constant<int, kGlu ? 2 : 1>(), rt);
    };
    const auto with_many = [&](auto rt) {
        const int64_t tiles = tiles16(16 * decltype(rt)::value) / kRowsWaves;
        if (tiles >= 4 * 512) return many(integral_constant<int, 4>(), rt);
        if (kGlu || tiles >= 2 * 512) return many(integral_constant<int, 2>(), rt);
        return many(integral_constant<int, kGlu ? 2 : 1>(), rt);
    };
    if (mean <= kRowsFew) return with_few(integral_constant<int, 1>());
    if (mean <= kRowsTile32) return with_many(integral_constant<int, 2>());
    return with_many(integral_constant<int, 4>());
}

}  // namespace

extern "C" int rhp_mx4_rows_gemm(int G, const int32_t* offsets, int64_t rows, int N, int K, int act, const void* x,
                                 const void* w_codes, const void* w_scales, void* out, hipStream_t stream) {
    clear_error();
    RHP_REQUIRE(G >= 1 && G <= kMaxG, "rhp_mx4_rows_gemm: 1 to 64 groups per call");
    RHP_REQUIRE(rows >= 0 && N >= 1 && K >= 1, "rhp_mx4_rows_gemm: bad sizes");
    RHP_REQUIRE(N % 8 == 0 && K % 8 == 0, "rhp_mx4_rows_gemm: N and K must be multiples of 8");
    RHP_REQUIRE(act == -1 || act == RHP_ACT_GELU || act == RHP_ACT_SWIGLU, "rhp_mx4_rows_gemm: unknown activation");
    if (rows == 0) return 0;
    RHP_REQUIRE(offsets && x && w_codes && w_scales && out, "rhp_mx4_rows_gemm: null pointer");
    RHP_REQUIRE(aligned16(x) && aligned16(w_codes) && aligned16(w_scales) && aligned16(out),
                "rhp_mx4_rows_gemm: operands and output must be 16-byte aligned");
    const int64_t w_rows = act == RHP_ACT_SWIGLU ? 2 * int64_t(N) : N, lim = int64_t(1) << 31;
    RHP_REQUIRE(rows < lim - 4096 && w_rows < lim - 4096 && K < (1 << 23),
                "rhp_mx4_rows_gemm: too many rows, or more than 2^23 columns");
    Mx4Rows p{};
    p.x = static_cast<const uint16_t*>(x);
    p.offsets = offsets;
    p.codes = static_cast<const uint8_t*>(w_codes);
    p.scales = static_cast<const uint8_t*>(w_scales);
    p.out = static_cast<uint16_t*>(out);
    p.rows = rows;
    p.G = G;
    p.N = N;
    p.K = K;
    p.blocks = static_cast<int>(blocks_of(K));
    p.w_codes = w_rows * p.blocks * 16;
    p.w_scales = words_of(K) * w_rows * 4;
    p.w_rows = static_cast<int>(w_rows);
    if (act == RHP_ACT_SWIGLU) return rows_gemm<kEpiSwigluAct>(p, stream);
    if (act == RHP_ACT_GELU) return rows_gemm<kEpiGeluAct>(p, stream);
    return rows_gemm<kEpiStore>(p, stream);
}
