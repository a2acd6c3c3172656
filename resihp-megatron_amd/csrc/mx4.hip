// Microscaled 4-bit floating point (e2m1 elements, one power of two for 32
// neighbours) for gfx950: quantisation along the rows of a matrix, along its
// columns, or both in one pass, and the way back.
//
// The reference keeps only the fp8-style amax state of resihp/runtime/
// reference_model.py:44-46; the 4-bit format is the OCP microscaling one.
//
//   scale  s = 2^(floor(log2(max |v|)) - 2)   of the block's 32 values, at least 2^-127
//   code   the nearest of 0 .5 1 1.5 2 3 4 6 to |v| / s, ties to the even code,
//          6 past it; bit 3 is the sign
// A block with an infinity or a NaN has the scale NaN (255): every value of it
// is NaN.  All of it is exact: v / s is a shift of the exponent, done by the
// conversion instruction (checked on this GPU for every scale, at and between
// all rounding borders, subnormals among them).
//
// Layout of a quantised matrix of R rows with C values along the blocks (Mx4):
//   codes  [R][ceil(C / 32) * 16] bytes, value c in the low (even c) or high
//          nibble of byte c / 2; the rest of a last block is zero codes
//   scales [ceil(C / 128)][R][4] bytes: the exponent + 127 of the four blocks of
//          128 values, so that the four scales a matrix instruction's operand
//          row needs are one word and neighbouring rows' words are contiguous;
//          blocks past the last are 0
// Along columns the matrix is the transposed one: R = columns, C = rows; with
// row groups (experts), each group's rows start at a multiple of 128, zeros
// between, in C = ((rows + 127 G) / 128) * 128 places.

#include <algorithm>

#include "mx4_common.h"

namespace rhp {
namespace {

constexpr int kQTile = 128;   // rows and columns of a block's tile
constexpr int kQThreads = 256;

struct Mx4QuantParams {
    const void* x[kMx4Many];    // one matrix, or many alike
    const int32_t* offsets;     // [G + 1] row groups of the one matrix, or null
    int G;
    int64_t rows;
    int cols;
    uint8_t *row_codes, *row_scales;   // or null
    uint8_t *col_codes, *col_scales;   // or null
    int64_t col_len;            // C of the columns' layout: rows, or the padded rows of the groups
    uint32_t tiles_x, tiles_y, tiles;   // column tiles, row tiles, and both of all matrices
};

// Eight neighbouring values of a row as float (zeros past the row).
template <class S> struct Eight;
template <> struct Eight<bf16> {
    uint32_t u[4];
    __device__ __forceinline__ void load(const bf16* p, int have) {
        if (have >= 8) {
            typedef uint32_t V __attribute__((ext_vector_type(4)));
            typedef V Vu __attribute__((aligned(2)));
            const V v = __builtin_nontemporal_load(reinterpret_cast<const Vu*>(p));
#pragma unroll
            for (int i = 0; i < 4; ++i) u[i] = v[i];
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t lo = 2 * i < have ? p[2 * i].bits : 0u, hi = 2 * i + 1 < have ? p[2 * i + 1].bits : 0u;
                u[i] = lo | hi << 16;
            }
        }
    }
    __device__ __forceinline__ uint4 word4(int) const { return make_uint4(u[0], u[1], u[2], u[3]); }
    // The largest magnitude, as the bits of a float (infinities and NaN past all finite ones).
    __device__ __forceinline__ uint32_t top() const {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) m = pk_max_u16(m, u[i] & 0x7fff7fffu);
        return max(m << 16, m & 0xffff0000u);
    }
    __device__ __forceinline__ uint32_t codes(float scale) const {
        uint32_t c = 0;
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2_hw_t, u[0]), scale, 0);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2_hw_t, u[1]), scale, 1);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2_hw_t, u[2]), scale, 2);
        return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2_hw_t, u[3]), scale, 3);
    }
    static __device__ __forceinline__ uint32_t pk_max_u16(uint32_t a, uint32_t b) {
        typedef unsigned short U __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(U, a), __builtin_bit_cast(U, b)));
    }
};
template <> struct Eight<float> {
    float v[8];
    __device__ __forceinline__ void load(const float* p, int have) {
        if (have >= 8) {
            typedef float V __attribute__((ext_vector_type(4)));
            typedef V Vu __attribute__((aligned(4)));
            const V a = __builtin_nontemporal_load(reinterpret_cast<const Vu*>(p));
            const V b = __builtin_nontemporal_load(reinterpret_cast<const Vu*>(p + 4));
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[i] = a[i];
                v[4 + i] = b[i];
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = i < have ? p[i] : 0.0f;
        }
    }
    __device__ __forceinline__ uint4 word4(int q) const {
        return make_uint4(__float_as_uint(v[4 * q]), __float_as_uint(v[4 * q + 1]), __float_as_uint(v[4 * q + 2]),
                          __float_as_uint(v[4 * q + 3]));
    }
    __device__ __forceinline__ uint32_t top() const {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
        return m;
    }
    __device__ __forceinline__ uint32_t codes(float scale) const {
        uint32_t c = 0;
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[0], v[1], scale, 0);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[2], v[3], scale, 1);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[4], v[5], scale, 2);
        return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[6], v[7], scale, 3);
    }
};

// Code (exponent + 127) of the block's scale from the bits of its largest magnitude; 255 where that is not finite.
__device__ __forceinline__ uint32_t scale_code(uint32_t top) {
    return top >= 0x7f800000u ? 255u : static_cast<uint32_t>(max(static_cast<int>(top >> 23) - 2, 0));
}

template <int kCtrl> __device__ __forceinline__ uint32_t dpp_u32(uint32_t v) {
    return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), kCtrl, 0xf, 0xf, true));
}

// One block: 128 rows by 128 columns.  Four neighbouring lanes hold a block of
// 32 along a row, eight values a lane: its maximum takes two lane exchanges,
// its codes leave as one word a lane, whole rows of 64 bytes.  For the columns
// the raw tile goes through LDS, with the words of the row blocks b = 0 .. 3
// turned by 16 b, so that the lanes that read four row blocks of 16 columns at
// once meet 64 banks; a thread then has whole blocks of a column and stores 16
// bytes, four threads 64 of a line.  Bound by HBM: both directions of 8 x 28672 x 4096
// bfloat16 557 us (2.9 GB, 5.2 TB/s), of 64 x 2816 x 2048 228, of 16384 x 28672 rows
// 333 and of 16384 x 4096 40.5; 8 x 28672 x 4096 float32 906 (5.2 TB/s).  Rows alone, columns alone:
// bfloat16 551, 453 us, float32 857, 799.  Tiles in plain order, whose neighbours' halves of a
// line meet in no L2, take 702 and 369 us of the first and third.
template <class S, bool kRows, bool kCols>
__global__ __launch_bounds__(kQThreads) void mx4_quantize_kernel(Mx4QuantParams p) {
    constexpr int kW = sizeof(S) / 2;   // half words an element
    __shared__ __align__(16) uint32_t tile[kCols ? kQTile : 1][kCols ? 64 * kW : 4];
    __shared__ uint32_t sc[kRows ? kQTile : 1];
    const int t = threadIdx.x, lane = t & 63, w = t >> 6;
    // Neighbouring tiles on one XCD, whose L2 then joins the 64 bytes that each has of a line: pairs of row tiles, column
    // by column.
    const uint32_t id = xcd_remap(blockIdx.x, p.tiles), per = p.tiles_x * p.tiles_y;
    const int64_t mat = id / per;
    const uint32_t in = id % per, band = in / (2 * p.tiles_x), rest = in % (2 * p.tiles_x);
    const uint32_t high = min(2u, p.tiles_y - 2 * band);
    const uint32_t tx = rest / high, ty = 2 * band + rest % high;
    const int c0 = static_cast<int>(tx) * kQTile;
    const S* x = static_cast<const S*>(p.x[mat]);

    // The tile's rows [r0, r1) of the matrix, and its first place k0 along the columns' blocks.
    int64_t r0, r1, k0;
    k0 = static_cast<int64_t>(ty) * kQTile;
    bool in_group = true, cols_here = kCols;
    if (p.offsets) {
        const Mx4Tile at = mx4_tile(p.offsets, p.G, p.rows, static_cast<int>(k0));
        r0 = at.r0;
        r1 = at.r1;
        in_group = at.in_group;                        // past the groups: zeros to the end of the places
        cols_here = kCols && k0 + kQTile <= p.col_len;
    } else {
        r0 = k0;
        r1 = p.rows;
    }

    const int col = c0 + 8 * (lane & 15);
    Eight<S> v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int64_t row = r0 + 32 * w + 4 * i + (lane >> 4);
        v[i].load(x + row * p.cols + col, row < r1 ? p.cols - col : 0);
    }
    if constexpr (kRows) {
        const int pitch = (p.cols + 31) / 32 * 16;
        uint8_t* out = p.row_codes + mat * p.rows * pitch;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int rr = 32 * w + 4 * i + (lane >> 4);
            uint32_t m = v[i].top();
            m = max(m, dpp_u32<0xB1>(m));   // quad_perm [1,0,3,2]
            m = max(m, dpp_u32<0x4E>(m));   // quad_perm [2,3,0,1]
            const uint32_t e = scale_code(m);
            const uint32_t c = e == 255u ? 0u : v[i].codes(mx4_scale(e));
            if (r0 + rr < r1 && (col & ~31) < p.cols)
                *reinterpret_cast<uint32_t*>(out + (r0 + rr) * pitch + col / 2) = c;
            if ((lane & 3) == 0) reinterpret_cast<uint8_t*>(&sc[rr])[(lane & 15) >> 2] = static_cast<uint8_t>(e);
        }
    }
    if constexpr (kCols) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int rr = 32 * w + 4 * i + (lane >> 4);
#pragma unroll
            for (int q = 0; q < kW; ++q)
                *reinterpret_cast<uint4*>(&tile[rr][(4 * kW * (lane & 15) + 4 * q) ^ (16 * w)]) = v[i].word4(q);
        }
    }
    __syncthreads();
    if constexpr (kRows) {
        if (t < kQTile && r0 + t < r1)
            reinterpret_cast<uint32_t*>(p.row_scales)[(mat * ((p.cols + 127) / 128) + tx) * p.rows + r0 + t] = sc[t];
    }
    if constexpr (kCols) {
        if (!cols_here) return;
        const int64_t pitch = (p.col_len + 31) / 32 * 16;
        uint8_t* out = p.col_codes + mat * p.cols * pitch;
        uint32_t* scales = reinterpret_cast<uint32_t*>(p.col_scales) +
                           (mat * ((p.col_len + 127) / 128) + k0 / 128) * p.cols;
        const int b = t & 3;   // row block
        const bool store = k0 + 32 * b < p.col_len;
        const auto emit = [&](int c, uint32_t top, auto codes_of) {
            const uint32_t e = scale_code(top);
            uint4 q = make_uint4(0u, 0u, 0u, 0u);
            if (e != 255u) q = codes_of(mx4_scale(e));
            if (c < p.cols && store) *reinterpret_cast<uint4*>(out + c * pitch + (k0 + 32 * b) / 2) = q;
            uint32_t s = e << (8 * b);
            s |= dpp_u32<0xB1>(s);
            s |= dpp_u32<0x4E>(s);
            return s;
        };
        if constexpr (sizeof(S) == 2) {
            const int pair = t >> 2;
            uint32_t u[32], m = 0;
#pragma unroll
            for (int i = 0; i < 32; ++i) {
                u[i] = in_group ? tile[32 * b + i][pair ^ (16 * b)] : 0u;
                m = Eight<bf16>::pk_max_u16(m, u[i] & 0x7fff7fffu);
            }
            const int c = c0 + 2 * pair;
            uint32_t s[2];
#pragma unroll
            for (int half = 0; half < 2; ++half)
                s[half] = emit(c + half, half ? m & 0xffff0000u : m << 16, [&](float scale) {
                    uint32_t o[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        Eight<bf16> e8;
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            e8.u[j] = __builtin_amdgcn_perm(u[8 * k + 2 * j + 1], u[8 * k + 2 * j],
                                                            half ? 0x07060302u : 0x05040100u);
                        o[k] = e8.codes(scale);
                    }
                    return make_uint4(o[0], o[1], o[2], o[3]);
                });
            if (b < 2 && c + b < p.cols) scales[c + b] = b ? s[1] : s[0];
        } else {
#pragma unroll
            for (int part = 0; part < 2; ++part) {
                const int cc = 64 * part + (t >> 2);
                float u[32];
                uint32_t m = 0;
#pragma unroll
                for (int i = 0; i < 32; ++i) {
                    u[i] = in_group ? __uint_as_float(tile[32 * b + i][cc ^ (16 * b)]) : 0.0f;
                    m = max(m, __float_as_uint(u[i]) & 0x7fffffffu);
                }
                const uint32_t s = emit(c0 + cc, m, [&](float scale) {
                    uint32_t o[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        Eight<float> e8;
#pragma unroll
                        for (int j = 0; j < 8; ++j) e8.v[j] = u[8 * k + j];
                        o[k] = e8.codes(scale);
                    }
                    return make_uint4(o[0], o[1], o[2], o[3]);
                });
                if (b == 0 && c0 + cc < p.cols) scales[c0 + cc] = s;
            }
        }
    }
}

// Values of codes: eight of a row a thread.  16384 x 4096 in bfloat16 27.6 us (6.1 TB/s).
template <class S>
__global__ __launch_bounds__(256) void mx4_dequantize_kernel(const uint8_t* __restrict__ codes,
                                                             const uint8_t* __restrict__ scales, uint32_t R, int C,
                                                             uint32_t total, S* __restrict__ out) {
    const uint32_t i = blockIdx.x * 256u + threadIdx.x;
    if (i >= total) return;
    const uint32_t per_row = static_cast<uint32_t>((C + 7) / 8);
    const uint32_t row = i / per_row;                    // of all matrices
    const int c = static_cast<int>(i - row * per_row) * 8;
    const uint32_t mat = row / R;
    const int pitch = (C + 31) / 32 * 16;
    const uint32_t q = *reinterpret_cast<const uint32_t*>(codes + static_cast<int64_t>(row) * pitch + c / 2);
    const int64_t word = (static_cast<int64_t>(mat) * ((C + 127) / 128) + c / 128) * R + (row - mat * R);
    const uint32_t e = scales[word * 4 + (c >> 5 & 3)];
    const float s = e == 255u ? __builtin_nanf("") : mx4_scale(e);
    S* o = out + static_cast<int64_t>(row) * C + c;
    if constexpr (sizeof(S) == 2) {
        const bf16x2_hw_t v[4] = {__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, s, 0),
                                  __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, s, 1),
                                  __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, s, 2),
                                  __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, s, 3)};
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = e == 255u ? 0x7fc07fc0u : __builtin_bit_cast(uint32_t, v[j]);
        if (c + 8 <= C) {
            typedef uint32_t V __attribute__((ext_vector_type(4)));
            typedef V Vu __attribute__((aligned(2)));
            *reinterpret_cast<Vu*>(o) = V{w[0], w[1], w[2], w[3]};
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (c + j < C) o[j].bits = static_cast<uint16_t>(w[j / 2] >> (16 * (j & 1)));
        }
    } else {
        const f32x2_hw_t v[4] = {__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, s, 0),
                                 __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, s, 1),
                                 __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, s, 2),
                                 __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, s, 3)};
        float w[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j] = e == 255u ? __builtin_nanf("") : v[j / 2][j & 1];
        if (c + 8 <= C) {
            typedef float V __attribute__((ext_vector_type(4)));
            typedef V Vu __attribute__((aligned(4)));
            *reinterpret_cast<Vu*>(o) = V{w[0], w[1], w[2], w[3]};
            *reinterpret_cast<Vu*>(o + 4) = V{w[4], w[5], w[6], w[7]};
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (c + j < C) o[j] = w[j];
        }
    }
}

template <class S>
int launch_quantize(const Mx4QuantParams& p, dim3 grid, hipStream_t s) {
    const bool r = p.row_codes != nullptr, c = p.col_codes != nullptr;
    if (r && c)
        hipLaunchKernelGGL((mx4_quantize_kernel<S, true, true>), grid, dim3(kQThreads), 0, s, p);
    else if (r)
        hipLaunchKernelGGL((mx4_quantize_kernel<S, true, false>), grid, dim3(kQThreads), 0, s, p);
    else
        hipLaunchKernelGGL((mx4_quantize_kernel<S, false, true>), grid, dim3(kQThreads), 0, s, p);
    return check_launch("mx4_quantize_kernel");
}

}  // namespace
}  // namespace rhp

using namespace rhp;

extern "C" int64_t rhp_mx4_padded_rows(int64_t rows, int G) {
    return rows < 0 || G < 1 ? 0 : (rows + 127 * static_cast<int64_t>(G)) / 128 * 128;
}

extern "C" int rhp_mx4_quantize(int n, const void* const* x, int dtype, int64_t rows, int cols, const int32_t* offsets,
                                int G, void* row_codes, void* row_scales, void* col_codes, void* col_scales,
                                hipStream_t stream) {
    clear_error();
    RHP_REQUIRE(dtype == RHP_BF16 || dtype == RHP_F32,
                std::string("rhp_mx4_quantize: unsupported dtype ") + dtype_name(dtype));
    RHP_REQUIRE(n >= 0 && rows >= 0 && rows < (int64_t(1) << 31) - 16384 && cols >= 1 && cols < INT32_MAX - 256,
                "rhp_mx4_quantize: bad sizes");
    RHP_REQUIRE(!offsets || (n == 1 && G >= 1 && G <= RHP_MAX_GROUPS_PER_LAUNCH),
                "rhp_mx4_quantize: row groups are 1 to 64 of one matrix");
    if (n == 0 || (rows == 0 && (!offsets || !col_codes))) return 0;
    RHP_REQUIRE(x && (row_codes || col_codes), "rhp_mx4_quantize: null pointer");
    RHP_REQUIRE((!row_codes || row_scales) && (!col_codes || col_scales), "rhp_mx4_quantize: codes without scales");
    RHP_REQUIRE(aligned16(row_codes) && aligned16(row_scales) && aligned16(col_codes) && aligned16(col_scales),
                "rhp_mx4_quantize: codes and scales must be 16-byte aligned");
    // With groups a last tile each of the G, of the rows behind them and of those ahead.
    const int64_t tiles = offsets ? (rows + 127 * (static_cast<int64_t>(G) + 2)) / 128 : (rows + 127) / 128;
    const int64_t ct = (static_cast<int64_t>(cols) + 127) / 128;
    const size_t bytes = dtype_bytes(dtype);
    RHP_REQUIRE(ct * tiles * std::min(n, kMx4Many) < (int64_t(1) << 24), "rhp_mx4_quantize: too many tiles");
    Mx4QuantParams p{};
    p.offsets = offsets;
    p.G = G;
    p.rows = rows;
    p.cols = cols;
    p.col_len = offsets ? rhp_mx4_padded_rows(rows, G) : rows;
    const int64_t row_bytes = rows * ((static_cast<int64_t>(cols) + 31) / 32 * 16), row_words = ct * rows;
    const int64_t col_bytes = cols * ((p.col_len + 31) / 32 * 16), col_words = (p.col_len + 127) / 128 * cols;
    for (int i0 = 0; i0 < n; i0 += kMx4Many) {
        const int m = std::min(kMx4Many, n - i0);
        for (int i = 0; i < m; ++i) {
            p.x[i] = x[i0 + i];
            RHP_REQUIRE(rows == 0 || (p.x[i] && reinterpret_cast<uintptr_t>(p.x[i]) % bytes == 0),
                        "rhp_mx4_quantize: a matrix is null or not aligned to its elements");
        }
        if (row_codes) {
            p.row_codes = static_cast<uint8_t*>(row_codes) + i0 * row_bytes;
            p.row_scales = static_cast<uint8_t*>(row_scales) + i0 * row_words * 4;
        }
        if (col_codes) {
            p.col_codes = static_cast<uint8_t*>(col_codes) + i0 * col_bytes;
            p.col_scales = static_cast<uint8_t*>(col_scales) + i0 * col_words * 4;
        }
        p.tiles_x = static_cast<uint32_t>(ct);
        p.tiles_y = static_cast<uint32_t>(tiles);
        p.tiles = static_cast<uint32_t>(ct * tiles * m);
        const dim3 grid(p.tiles);
        const int rc = dtype == RHP_F32 ? launch_quantize<float>(p, grid, stream) : launch_quantize<bf16>(p, grid, stream);
        if (rc) return rc;
    }
    return 0;
}

extern "C" int rhp_mx4_dequantize(const void* codes, const void* scales, int64_t n, int64_t rows, int cols, int dtype,
                                  void* out, hipStream_t stream) {
    clear_error();
    RHP_REQUIRE(dtype == RHP_BF16 || dtype == RHP_F32,
                std::string("rhp_mx4_dequantize: unsupported dtype ") + dtype_name(dtype));
    RHP_REQUIRE(n >= 0 && rows >= 0 && cols >= 1 && cols < INT32_MAX - 256, "rhp_mx4_dequantize: bad sizes");
    if (n == 0 || rows == 0) return 0;
    RHP_REQUIRE(codes && scales && out, "rhp_mx4_dequantize: null pointer");
    RHP_REQUIRE(aligned16(codes) && aligned16(scales) && reinterpret_cast<uintptr_t>(out) % dtype_bytes(dtype) == 0,
                "rhp_mx4_dequantize: codes and scales must be 16-byte aligned, the output to its elements");
    const int64_t per_row = (static_cast<int64_t>(cols) + 7) / 8;
    RHP_REQUIRE(n < (int64_t(1) << 31) && rows < (int64_t(1) << 31) && n * rows < (int64_t(1) << 32) &&
                    n * rows * per_row < (int64_t(1) << 32) - 256,
                "rhp_mx4_dequantize: at most 2^35 values");
    const uint32_t total = static_cast<uint32_t>(n * rows * per_row);
    const dim3 grid((total + 255u) / 256u);
    const uint8_t *q = static_cast<const uint8_t*>(codes), *s = static_cast<const uint8_t*>(scales);
    if (dtype == RHP_F32)
        hipLaunchKernelGGL(mx4_dequantize_kernel<float>, grid, dim3(256), 0, stream, q, s, static_cast<uint32_t>(rows),
                           cols, total, static_cast<float*>(out));
    else
        hipLaunchKernelGGL(mx4_dequantize_kernel<bf16>, grid, dim3(256), 0, stream, q, s, static_cast<uint32_t>(rows),
                           cols, total, static_cast<bf16*>(out));
    return check_launch("mx4_dequantize_kernel");
}
