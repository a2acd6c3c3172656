// Backward of the router's logits under a gradient of all of them, for gfx950:
// what the router's losses send into the tokens and the router's weight.
//
// logits = x W^T (resihp/runtime/moe.py:76), so with dl = dlogits [T, E]:
//   dx [T, h] = dl W       dW [E, h] = dl^T x
// (The gradient of the selected logits alone takes rhp_token_bwd and
// rhp_router_wgrad, which read k experts a token, not E.)
//
// With bfloat16 tokens x is read once and dx written once (67 MB each at 16384 x
// 2048), for 2 T E h operations each.  In float
// matrix instructions those would take four times as long as the bytes, so the float
// operands are split into bfloat16 terms, v = t0 + t1 (+ t2) with t0 and t1 the
// upper 8 bits of what is left (exact, by truncation) and the last rounded:
//   dW  three terms of dl, all 24 bits, times x, which is bfloat16: exact products
//   dx  two terms of dl and of W (the last rounded: 2^-16 of a factor left out at most), the
//       product of the two small ones, each below 2^-7 of its factor, left out too: at most 2^-14 +
//       2^-15 of |dl| |W|, against the 2^-8 of dx's own rounding
// An infinite dl or W gives NaN (its second term is inf - inf).  Float32 and
// float64 tokens, and rows that are not multiples of 8, take plain tiles of
// fused multiply-adds.  dW is summed over slices of the tokens and then over the
// slices, in an order that the sizes alone decide.

#include <algorithm>
#include <type_traits>

#include "rhp_common.h"

namespace rhp {
namespace {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));

constexpr int kDenseMaxE = 1024;
constexpr int kChunkE = 64;        // experts that a dW block takes (128: its accumulators spill)

// ------------------------------------------------------------------ plain tiles

constexpr int kPlainTile = 64, kPlainK = 16, kPlainThreads = 256;

// C[m, n] = sum_k A(m, k) B(k, n) over k in [k0, k1): 64 x 64 a block, 4 x 4 a thread.  kTransA: a is [K, M].
// Bound by the fused multiply-adds and their reads from LDS, eight for sixteen; dW has 64 experts a tile, however few
// there are, and too few blocks where there are few.  us of dx, dW with the sum over the slices (a library product of the
// same: dx, dW), where the tokens' bytes alone take 22, 90 and 45 in float32:
//   16384 x 2048 by 64 experts    float32  93, 421 (60, 126)     float64 171, 563 (100, 1770)
//   32768 x 4096 by 8                     163, 1796 (128, 280)           265, 2234 (180, 3546)
//   32768 x 2048 by 128                   357, 1906 (171, 228)           652, 2380 (332, 3518)
//   16384 x 2044 by 64, bfloat16 tokens    88, 429
template <class A, class S, class O, bool kTransA>
__global__ __launch_bounds__(kPlainThreads) void router_plain_kernel(const A* __restrict__ a, const S* __restrict__ b,
                                                                     int64_t M, int N, int64_t K, int64_t lda,
                                                                     int slices, O* __restrict__ out) {
    __shared__ A as[kPlainK][kPlainTile + 1], bs[kPlainK][kPlainTile + 1];
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const int64_t m0 = static_cast<int64_t>(blockIdx.y) * kPlainTile;
    const int n0 = blockIdx.x * kPlainTile;
    const int64_t k0 = K * blockIdx.z / slices, k1 = K * (blockIdx.z + 1) / slices;
    A acc[4][4] = {};
    for (int64_t k = k0; k < k1; k += kPlainK) {
        for (int i = threadIdx.x; i < kPlainK * kPlainTile; i += kPlainThreads) {
            const int kk = kTransA ? i / kPlainTile : i % kPlainK, mm = kTransA ? i % kPlainTile : i / kPlainK;
            as[kk][mm] = k + kk < k1 && m0 + mm < M ? a[kTransA ? (k + kk) * lda + m0 + mm : (m0 + mm) * lda + k + kk] : A(0);
            const int kb = i / kPlainTile, nn = i % kPlainTile;
            bs[kb][nn] = k + kb < k1 && n0 + nn < N ? static_cast<A>(Elem<S>::ld(b, (k + kb) * N + n0 + nn)) : A(0);
        }
        __syncthreads();
#pragma unroll
        for (int kk = 0; kk < kPlainK; ++kk)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] += as[kk][ty + 16 * i] * bs[kk][tx + 16 * j];
        __syncthreads();
    }
    out += static_cast<int64_t>(blockIdx.z) * M * N;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (m0 + ty + 16 * i < M && n0 + tx + 16 * j < N)
                Elem<O>::st(out, (m0 + ty + 16 * i) * N + n0 + tx + 16 * j, acc[i][j]);
}

// The sum of `slices` partial results of n values each.
template <class A>
__global__ __launch_bounds__(256) void router_slices_kernel(const A* __restrict__ part, int64_t n, int slices,
                                                            A* __restrict__ out) {
    const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (i >= n) return;
    A sum = part[i];
#pragma unroll 8
    for (int s = 1; s < slices; ++s) sum += part[s * n + i];
    out[i] = sum;
}

// ------------------------------------------------------------------ bfloat16 tokens

// Eight floats as bfloat16 terms: all but the last the upper bits of what is left, the last rounded.
template <int TERMS> __device__ __forceinline__ void split8(const float (&v)[8], u32x4_t (&t)[TERMS]) {
    float r[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = v[i];
#pragma unroll
    for (int n = 0; n < TERMS; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (n + 1 == TERMS) {
                t[n][i] = pack_bf16x2(r[2 * i], r[2 * i + 1]);
            } else {
                const uint32_t a = __float_as_uint(r[2 * i]), b = __float_as_uint(r[2 * i + 1]);
                t[n][i] = __builtin_amdgcn_perm(b, a, 0x07060302u);
                r[2 * i] -= __uint_as_float(a & 0xffff0000u);
                r[2 * i + 1] -= __uint_as_float(b & 0xffff0000u);
            }
        }
}
__device__ __forceinline__ f32x16_t mfma_bf16(u32x4_t a, u32x4_t b, f32x16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}

// A barrier for what the block shares in LDS: __syncthreads would also wait for the loads and stores in flight.
__device__ __forceinline__ void lds_sync() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0xC07F);   // lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// dx: a wave holds W's terms for 64 columns and up to 16 KS experts in registers
// and the block walks the tokens, 64 at a time, whose terms of dl its threads make
// once and share through LDS (one wave's own: the splits took longer than the
// products).  Lane L of a 32 x 32 x 16 product has column L % 32 (as the product's rows) and
// experts 8 (L / 32) .. + 7 of W, and token L % 32 and the same experts of dl.
// The results are turned through LDS, so that a row leaves in 128 contiguous
// bytes.  More than 128 experts: W's terms are made again for every 64 tokens.
// 16384 x 2048 by 64 experts 28 us (2.5 TB/s; a block's splits, products and stores follow
// one another, two blocks a CU cover them), 16384 x 4096 by 8 experts 25 (5.4
// TB/s), 32768 x 2048 by 128 experts 107 (the products' three terms; from 65 experts on the
// block's 84 KB of LDS leave room for one a CU, so nothing covers them).  Every wave with
// splits of its own took 64 us of the first.
constexpr int kDxThreads = 256, kDxWaves = kDxThreads / 64, kDxTokens = 64;
constexpr int kDxPitch = 72;   // halves a staged row of 64: 16-byte pieces, banks turned by 4 a row

template <int KS>
__global__ __launch_bounds__(kDxThreads) void router_dx_kernel(const float* __restrict__ dl, const float* __restrict__ w,
                                                               int64_t T, int h, int E, int tiles,
                                                               bf16* __restrict__ dx) {
    constexpr int kItems = kDxTokens * 2 * KS / kDxThreads;   // eight experts of a token each, of a thread
    static_assert(kItems * kDxThreads == kDxTokens * 2 * KS || KS == 1, "whole shares");
    __shared__ __align__(16) uint16_t stage[kDxWaves][32][kDxPitch];
    __shared__ u32x4_t terms[2][2][KS][2][64];   // [buffer][32 tokens][16 experts][term][lane]
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
    const int h0 = (blockIdx.x * kDxWaves + wave) * 64;
    const bool vec = (E & 3) == 0;
    u32x4_t wt[2][KS][2];
    const auto load_w = [&](int e0) {
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                const int col = h0 + 32 * m + (lane & 31);
                float v[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int e = e0 + 16 * ks + 8 * half + j;
                    v[j] = e < E && col < h ? w[static_cast<int64_t>(e) * h + col] : 0.0f;
                }
                split8<2>(v, wt[m][ks]);
                __builtin_amdgcn_sched_barrier(0);   // a fragment's loads at a time
            }
    };
    // Item i: token i % 64, experts 8 (i / 64) .. + 7.
    constexpr int kMine = kItems > 0 ? kItems : 1;
    const auto load_d = [&](float (&v)[kMine][8], int64_t tile, int e0) {
#pragma unroll
        for (int n = 0; n < kMine; ++n) {
            const int i = threadIdx.x + kDxThreads * n;
            const int64_t t = tile * kDxTokens + (i & 63);
            const int e = e0 + 8 * (i >> 6);
            const float* p = dl + t * E + e;
            const bool have = t < T && i < kDxTokens * 2 * KS;
#pragma unroll
            for (int j = 0; j < 8; j += 4) {
                if (vec) {
                    float4 q = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (have && e + j < E) q = *reinterpret_cast<const float4*>(p + j);
                    v[n][j] = q.x, v[n][j + 1] = q.y, v[n][j + 2] = q.z, v[n][j + 3] = q.w;
                } else {
#pragma unroll
                    for (int k = 0; k < 4; ++k) v[n][j + k] = have && e + j + k < E ? p[j + k] : 0.0f;
                }
            }
        }
    };
    const auto put_d = [&](const float (&v)[kMine][8], int buffer) {
#pragma unroll
        for (int n = 0; n < kMine; ++n) {
            const int i = threadIdx.x + kDxThreads * n;
            if (i >= kDxTokens * 2 * KS) break;
            const int t = i & 63, e8 = i >> 6;
            u32x4_t d[2];
            split8<2>(v[n], d);
#pragma unroll
            for (int k = 0; k < 2; ++k) terms[buffer][t >> 5][e8 >> 1][k][(t & 31) + 32 * (e8 & 1)] = d[k];
        }
    };
    const bool again = E > 16 * KS;
    const int64_t all = (T + kDxTokens - 1) / kDxTokens;
    const int64_t first = static_cast<int64_t>(blockIdx.y) * tiles, last = min(all, first + tiles);
    float v[kMine][8];
    load_d(v, first, 0);
    if (!again) load_w(0);
    put_d(v, 0);
    lds_sync();
    int buffer = 0;
    for (int64_t tile = first; tile < last; ++tile) {
        f32x16_t acc[2][2] = {};
        for (int e0 = 0; e0 < E; e0 += 16 * KS, buffer ^= 1) {
            // The next 64 tokens' (or experts') gradients are on their way under the products.
            const bool more = e0 + 16 * KS < E;
            load_d(v, more ? tile : tile + 1, more ? e0 + 16 * KS : 0);
            if (again) load_w(e0);
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    const u32x4_t d0 = terms[buffer][s][ks][0][lane], d1 = terms[buffer][s][ks][1][lane];
#pragma unroll
                    for (int m = 0; m < 2; ++m) {
                        acc[s][m] = mfma_bf16(wt[m][ks][1], d0, acc[s][m]);
                        acc[s][m] = mfma_bf16(wt[m][ks][0], d1, acc[s][m]);
                        acc[s][m] = mfma_bf16(wt[m][ks][0], d0, acc[s][m]);
                    }
                }
            put_d(v, buffer ^ 1);
            lds_sync();
        }
        // The stage is the wave's own: its accesses to LDS are in order, no barrier is needed.
#pragma unroll
        for (int s = 0; s < 2; ++s) {
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    *reinterpret_cast<uint2*>(&stage[wave][lane & 31][32 * m + 8 * q + 4 * half]) =
                        make_uint2(pack_bf16x2(acc[s][m][4 * q], acc[s][m][4 * q + 1]),
                                   pack_bf16x2(acc[s][m][4 * q + 2], acc[s][m][4 * q + 3]));
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = 8 * i + (lane >> 3), c = 8 * (lane & 7);
                const int64_t t = tile * kDxTokens + 32 * s + r;
                if (t < T && h0 + c < h)
                    *reinterpret_cast<uint4*>(dx + t * h + h0 + c) = *reinterpret_cast<const uint4*>(&stage[wave][r][c]);
            }
            __builtin_amdgcn_wave_barrier();
        }
    }
}

// dW: a block takes 128 columns and a slice of the tokens, MT x 32 experts.  Its
// eight waves are two along the columns and four along the tokens, 32 tokens a turn each.  x goes
// straight from memory into the products: lane L reads the two columns
// 2 (L % 32), + 1 of tokens 8 (L / 32) .. + 7, and the even columns make one product, the odd ones the
// other.  dl's terms are made once a block and read from LDS by both column waves.
// The four token waves' sums are added through LDS, in their order.  A turn waits for
// memory, so its loads are issued two turns ahead, through buffer views, whose 32-bit
// offsets leave the registers for them: 16384 x 2048 by 64 experts 32 us with the sum over the
// slices (36 one turn ahead), 16384 x 4096 by 8 33, 32768 x 2048 by 128 80.
constexpr int kDwThreads = 512, kDwCols = 128, kDwTokens = 128;

template <int MT>
__global__ __launch_bounds__(kDwThreads) void router_dw_kernel(const float* __restrict__ dl, const bf16* __restrict__ x,
                                                               int64_t T, int h, int E, int slices,
                                                               float* __restrict__ out) {
    // Terms of dl: [token wave][32 experts][16 tokens][term][lane].
    __shared__ __align__(16) union {
        u32x4_t d[4][MT][2][3][64];
        float sum[4][MT * 2 * 16 / 4][128];   // a quarter of the accumulators of the waves that give theirs away
    } lds;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
    const int wh = wave & 1, wk = wave >> 1;
    const int e0 = blockIdx.z * kChunkE;
    const int col = blockIdx.x * kDwCols + 64 * wh + 2 * (lane & 31);
    const int64_t turns = (T + kDwTokens - 1) / kDwTokens;
    const int64_t first = turns * blockIdx.y / slices, last = turns * (blockIdx.y + 1) / slices;
    f32x16_t acc[MT][2] = {};
    struct Turn {
        uint32_t x[2][8];
        float d[MT][8];
    };
    // A thread's share of dl's terms: item i = thread + 512 n of the turn is expert i % (32 MT), tokens 8 (i / (32 MT)) .. + 7.
    const auto load = [&](Turn& v, int64_t turn) {
        const int64_t t0 = turn * kDwTokens;
        const int left = static_cast<int>(min(T - t0, static_cast<int64_t>(kDwTokens)));   // tokens of the turn
        // Views of the turn's rows: rows past the last read zeros, and 32-bit offsets spare registers.
        const __amdgpu_buffer_rsrc_t xr = __builtin_amdgcn_make_buffer_rsrc(const_cast<bf16*>(x + t0 * h), 0, left * h * 2, 0x00020000);
        const __amdgpu_buffer_rsrc_t dr = __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(dl + t0 * E), 0, left * E * 4, 0x00020000);
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
            const int at = col < h ? ((32 * wk + 16 * ks + 8 * half) * h + col) * 2 : INT32_MIN;   // past every view
#pragma unroll
            for (int j = 0; j < 8; ++j) v.x[ks][j] = __builtin_amdgcn_raw_buffer_load_b32(xr, at, j * h * 2, 0);
        }
#pragma unroll
        for (int n = 0; n < MT; ++n) {
            const int i = threadIdx.x + kDwThreads * n;
            const int e = e0 + i % (32 * MT);
            const int at = e < E ? (8 * (i / (32 * MT)) * E + e) * 4 : INT32_MIN;
#pragma unroll
            for (int j = 0; j < 8; ++j)
                v.d[n][j] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(dr, at, j * E * 4, 0));
        }
    };
    // One turn from v, into which the turn after the next is loaded under its products.
    const auto work = [&](Turn& v, int64_t turn) {
        lds_sync();   // the turn before has read dl's terms
#pragma unroll
        for (int n = 0; n < MT; ++n) {
            const int i = threadIdx.x + kDwThreads * n;
            const int e = i % (32 * MT), t8 = i / (32 * MT);   // t8: eight tokens of 128
            u32x4_t d[3];
            split8<3>(v.d[n], d);
#pragma unroll
            for (int k = 0; k < 3; ++k) lds.d[t8 >> 2][e >> 5][(t8 >> 1) & 1][k][(e & 31) + 32 * (t8 & 1)] = d[k];
        }
        u32x4_t b[2][2];
#pragma unroll
        for (int ks = 0; ks < 2; ++ks)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                b[ks][0][i] = __builtin_amdgcn_perm(v.x[ks][2 * i + 1], v.x[ks][2 * i], 0x05040100u);
                b[ks][1][i] = __builtin_amdgcn_perm(v.x[ks][2 * i + 1], v.x[ks][2 * i], 0x07060302u);
            }
        if (turn + 2 < last) load(v, turn + 2);
        lds_sync();
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int ks = 0; ks < 2; ++ks)
#pragma unroll
                for (int k = 2; k >= 0; --k) {
                    const u32x4_t a = lds.d[wk][m][ks][k][lane];
                    acc[m][0] = mfma_bf16(a, b[ks][0], acc[m][0]);
                    acc[m][1] = mfma_bf16(a, b[ks][1], acc[m][1]);
                }
    };
    Turn even, odd;
    if (first < last) load(even, first);
    if (first + 1 < last) load(odd, first + 1);
    for (int64_t turn = first; turn < last; turn += 2) {
        work(even, turn);
        if (turn + 1 < last) work(odd, turn + 1);
    }
    // The token waves' sums: 1 to 3 give theirs to wave 0, a quarter of the registers at a time.
    constexpr int kN = MT * 2 * 16;
    const int slot = wh * 64 + lane;
#pragma unroll
    for (int part = 0; part < 4; ++part) {
        lds_sync();
        if (wk > 0) {
#pragma unroll
            for (int i = 0; i < kN / 4; ++i) {
                const int n = part * (kN / 4) + i;
                lds.sum[wk][i][slot] = acc[n / 32][n / 16 % 2][n % 16];
            }
        }
        lds_sync();
        if (wk == 0) {
#pragma unroll
            for (int i = 0; i < kN / 4; ++i) {
                const int n = part * (kN / 4) + i;
                float v = acc[n / 32][n / 16 % 2][n % 16];
                for (int k = 1; k < 4; ++k) v += lds.sum[k][i][slot];
                acc[n / 32][n / 16 % 2][n % 16] = v;
            }
        }
    }
    if (wk != 0 || col >= h) return;
    out += static_cast<int64_t>(blockIdx.y) * E * h;
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int e = e0 + 32 * m + 8 * (i / 4) + 4 * half + i % 4;
            if (e < E) *reinterpret_cast<float2*>(out + static_cast<int64_t>(e) * h + col) = make_float2(acc[m][0][i], acc[m][1][i]);
        }
}

// ------------------------------------------------------------------ host

bool dense_fast(int x_dtype, int h) { return x_dtype == RHP_BF16 && h % 8 == 0; }

// Slices of the tokens that dW is summed in: about a block a CU.
int dw_slices(int64_t T, int h, int E, int x_dtype) {
    int64_t blocks, most;
    if (dense_fast(x_dtype, h)) {
        blocks = static_cast<int64_t>((h + kDwCols - 1) / kDwCols) * ((E + kChunkE - 1) / kChunkE);
        most = (T + kDwTokens - 1) / kDwTokens;
    } else {
        blocks = static_cast<int64_t>((h + kPlainTile - 1) / kPlainTile) * ((E + kPlainTile - 1) / kPlainTile);
        most = (T + 63) / 64;
    }
    return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({(256 + blocks - 1) / blocks, most, 64})));
}

template <class A, class S>
int dense_plain(const void* dl, const void* x, const void* w, int64_t T, int h, int E, int slices, void* dx, void* dw,
                void* ws, hipStream_t stream) {
    const unsigned nb = static_cast<unsigned>((h + kPlainTile - 1) / kPlainTile);
    if (dx) {
        hipLaunchKernelGGL((router_plain_kernel<A, A, S, false>), dim3(nb, static_cast<unsigned>((T + kPlainTile - 1) / kPlainTile), 1),
                           dim3(kPlainThreads), 0, stream, static_cast<const A*>(dl), static_cast<const A*>(w), T, h,
                           static_cast<int64_t>(E), static_cast<int64_t>(E), 1, static_cast<S*>(dx));
        if (int rc = check_launch("router_plain_kernel")) return rc;
    }
    if (dw) {
        A* out = static_cast<A*>(slices > 1 ? ws : dw);
        hipLaunchKernelGGL((router_plain_kernel<A, S, A, true>),
                           dim3(nb, static_cast<unsigned>((E + kPlainTile - 1) / kPlainTile), static_cast<unsigned>(slices)),
                           dim3(kPlainThreads), 0, stream, static_cast<const A*>(dl), static_cast<const S*>(x),
                           static_cast<int64_t>(E), h, T, static_cast<int64_t>(E), slices, out);
        if (int rc = check_launch("router_plain_kernel")) return rc;
    }
    return 0;
}

int dense_bf16(const float* dl, const bf16* x, const float* w, int64_t T, int h, int E, int slices, bf16* dx, float* dw,
               float* ws, hipStream_t stream) {
    if (dx && T) {
        // Two blocks a CU at most; a block walks `tiles` tiles of 64 tokens with W in registers.
        const int64_t all = (T + kDxTokens - 1) / kDxTokens, cols = (h + 255) / 256;
        const int64_t tiles = std::max<int64_t>(1, (all * cols + 511) / 512);
        const dim3 grid(static_cast<unsigned>(cols), static_cast<unsigned>((all + tiles - 1) / tiles));
        const auto go = [&](auto ks) {
            hipLaunchKernelGGL((router_dx_kernel<decltype(ks)::value>), grid, dim3(kDxThreads), 0, stream, dl, w, T, h, E,
                               static_cast<int>(tiles), dx);
            return check_launch("router_dx_kernel");
        };
        using std::integral_constant;
        const int rc = E <= 16   ? go(integral_constant<int, 1>())
                       : E <= 32 ? go(integral_constant<int, 2>())
                       : E <= 64 ? go(integral_constant<int, 4>())
                                 : go(integral_constant<int, 8>());
        if (rc) return rc;
    }
    if (dw) {
        const dim3 grid(static_cast<unsigned>((h + kDwCols - 1) / kDwCols), static_cast<unsigned>(slices),
                        static_cast<unsigned>((E + kChunkE - 1) / kChunkE));
        const auto go = [&](auto mt) {
            hipLaunchKernelGGL((router_dw_kernel<decltype(mt)::value>), grid, dim3(kDwThreads), 0, stream, dl, x, T, h, E,
                               slices, slices > 1 ? ws : dw);
            return check_launch("router_dw_kernel");
        };
        using std::integral_constant;
        return E <= 32 ? go(integral_constant<int, 1>()) : go(integral_constant<int, 2>());
    }
    return 0;
}

template <class A> int dense_sum(const void* ws, int64_t n, int slices, void* dw, hipStream_t stream) {
    hipLaunchKernelGGL(router_slices_kernel<A>, dim3(static_cast<unsigned>((n + 255) / 256)), dim3(256), 0, stream,
                       static_cast<const A*>(ws), n, slices, static_cast<A*>(dw));
    return check_launch("router_slices_kernel");
}

}  // namespace
}  // namespace rhp

using namespace rhp;

extern "C" size_t rhp_router_logits_bwd_workspace_bytes(int64_t T, int h, int E, int x_dtype) {
    if (T < 0 || h < 1 || E < 1) return 0;
    const int s = dw_slices(T, h, E, x_dtype);
    return s > 1 ? static_cast<size_t>(s) * E * h * (x_dtype == RHP_F64 ? 8 : 4) : 0;
}

extern "C" int rhp_router_logits_bwd(const void* dlogits, const void* x, int x_dtype, const void* router_w, int r_dtype,
                                     int64_t T, int h, int E, void* dx, void* dw, void* workspace,
                                     size_t workspace_bytes, hipStream_t stream) {
    clear_error();
    RHP_REQUIRE(x_dtype == RHP_F64 || x_dtype == RHP_F32 || x_dtype == RHP_BF16,
                std::string("rhp_router_logits_bwd: unsupported dtype ") + dtype_name(x_dtype));
    RHP_REQUIRE(r_dtype == (x_dtype == RHP_F64 ? RHP_F64 : RHP_F32),
                "rhp_router_logits_bwd: a float64 model needs a float64 router, others a float32 router");
    RHP_REQUIRE(T >= 0 && T < (int64_t(1) << 31) - 64 && h >= 1 && E >= 1 && E <= kDenseMaxE,
                "rhp_router_logits_bwd: need T >= 0, h >= 1 and 1 <= E <= 1024");
    RHP_REQUIRE(h <= (1 << 22), "rhp_router_logits_bwd: rows of at most 2^22 columns");
    RHP_REQUIRE((!dw && !dx) || T == 0 || dlogits, "rhp_router_logits_bwd: null pointer");
    RHP_REQUIRE(!dx || T == 0 || (router_w && dx != dlogits), "rhp_router_logits_bwd: dx needs the router's weight");
    RHP_REQUIRE(!dw || T == 0 || x, "rhp_router_logits_bwd: dw needs the tokens");
    RHP_REQUIRE(aligned16(dlogits) && aligned16(x) && aligned16(router_w) && aligned16(dx) && aligned16(dw),
                "rhp_router_logits_bwd: tensors must be 16-byte aligned");
    const int slices = dw_slices(T, h, E, x_dtype);
    RHP_REQUIRE(!dw || slices == 1 ||
                    (workspace && aligned16(workspace) &&
                     workspace_bytes >= rhp_router_logits_bwd_workspace_bytes(T, h, E, x_dtype)),
                "rhp_router_logits_bwd: workspace smaller than rhp_router_logits_bwd_workspace_bytes(), null or unaligned");
    RHP_REQUIRE(T <= int64_t(65535) * 32 || !dx || dense_fast(x_dtype, h),
                "rhp_router_logits_bwd: at most 2 M tokens of these types");
    int rc;
    if (dense_fast(x_dtype, h))
        rc = dense_bf16(static_cast<const float*>(dlogits), static_cast<const bf16*>(x), static_cast<const float*>(router_w),
                        T, h, E, slices, static_cast<bf16*>(dx), static_cast<float*>(dw), static_cast<float*>(workspace), stream);
    else if (x_dtype == RHP_BF16)
        rc = dense_plain<float, bf16>(dlogits, x, router_w, T, h, E, slices, T ? dx : nullptr, dw, workspace, stream);
    else if (x_dtype == RHP_F32)
        rc = dense_plain<float, float>(dlogits, x, router_w, T, h, E, slices, T ? dx : nullptr, dw, workspace, stream);
    else
        rc = dense_plain<double, double>(dlogits, x, router_w, T, h, E, slices, T ? dx : nullptr, dw, workspace, stream);
    if (rc || !dw || slices == 1) return rc;
    const int64_t n = static_cast<int64_t>(E) * h;
    return x_dtype == RHP_F64 ? dense_sum<double>(workspace, n, slices, dw, stream)
                              : dense_sum<float>(workspace, n, slices, dw, stream);
}
