// Layer norm for gfx950: the normalisation in front of the MoE layer, forward
// and backward with the reduction of the weight's and bias's gradients.
//
// Reference: the pre-norm residual block of resihp/runtime/reference_model.py:
// 195-234 (out = x + f(norm(x))); here f is the MoE layer of
// resihp/runtime/moe.py:90-101.
//
//   mean = sum(x) / h      rstd = 1 / sqrt(sum((x - mean)^2) / h + eps)
//   y    = (x - mean) * rstd * w + b
// and with g = dy * w, xh = (x - mean) * rstd:
//   dx   = rstd * (g - sum(g) / h - xh * sum(g * xh) / h) (+ the residual's gradient)
//   dw   = sum over rows of dy * xh      db = sum over rows of dy
//
// Statistics are float (double for double rows) and so are sums, but those over
// the columns of rows past the registers, which are double; a bfloat16 result is
// rounded once, when it is stored.  The variance is that of the centred
// values, so a large mean does not swamp it.  Nothing uses atomics: every sum
// has an order fixed by the sizes, so results are reproducible bit for bit.
//
// Both directions are bound by HBM: a row is read once (the backward reads dy,
// x and the residual's gradient) and written once, some ten operations an
// element.  16384 x 4096 bfloat16: forward 46 us (268 MB, 5.8 TB/s), backward
// with the residual's gradient 95 us and 4.5 us for the sum of its partial
// rows (537 MB and 2 x 8.4 MB, 5.6 TB/s); a non-temporal copy reaches 6.0.

#include <algorithm>
#include <initializer_list>
#include <type_traits>

#include "rhp_common.h"

namespace rhp {
namespace {

constexpr int kNormThreads = 256;
constexpr int kNormWaves = kNormThreads / 64;

__device__ __forceinline__ float rsqrt_t(float x) { return 1.0f / __builtin_sqrtf(x); }
__device__ __forceinline__ double rsqrt_t(double x) { return 1.0 / __builtin_sqrt(x); }

template <int kCtrl> __device__ __forceinline__ float dpp(float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), kCtrl, 0xf, 0xf, true));
}
// Sum over neighbouring lanes (8, 16, 32 or 64 of them), in all of them.
template <int kLanes> __device__ __forceinline__ float lane_sum(float v) {
    v += dpp<0xB1>(v);                           // quad_perm [1,0,3,2]
    v += dpp<0x4E>(v);                           // quad_perm [2,3,0,1]
    v += dpp<0x141>(v);                          // row_half_mirror: the other four of eight
    if constexpr (kLanes > 8) v += dpp<0x140>(v);   // row_mirror: the other eight of sixteen
    if constexpr (kLanes > 16) v += __shfl_xor(v, 16, 64);
    if constexpr (kLanes > 32) v += __shfl_xor(v, 32, 64);
    return v;
}
template <int kLanes> __device__ __forceinline__ double lane_sum(double v) {
#pragma unroll
    for (int d = kLanes / 2; d >= 1; d >>= 1) v += __shfl_xor(v, d, 64);
    return v;
}

// ------------------------------------------------------------------ chunks of 16 bytes

// A vector access needs no alignment beyond its element's, and costs the same
// where it is aligned.
typedef uint32_t Q __attribute__((ext_vector_type(4)));
typedef Q Qu __attribute__((aligned(2)));
template <class S> constexpr int kVec = 16 / static_cast<int>(sizeof(S));

template <class S> struct Chunk {
    Q q;
    __device__ __forceinline__ void load(const S* p) { q = __builtin_nontemporal_load(reinterpret_cast<const Qu*>(p)); }
    __device__ __forceinline__ typename Elem<S>::acc at(int j) const {
        if constexpr (sizeof(S) == 8)
            return __hiloint2double(static_cast<int>(q[2 * j + 1]), static_cast<int>(q[2 * j]));
        else if constexpr (sizeof(S) == 4)
            return __uint_as_float(q[j]);
        else
            return __uint_as_float(j & 1 ? q[j / 2] & 0xffff0000u : q[j / 2] << 16);
    }
};
template <class S> __device__ __forceinline__ void store_chunk(S* p, const typename Elem<S>::acc* v) {
    Q q;
    if constexpr (sizeof(S) == 8) {
        q = {static_cast<uint32_t>(__double2loint(v[0])), static_cast<uint32_t>(__double2hiint(v[0])),
             static_cast<uint32_t>(__double2loint(v[1])), static_cast<uint32_t>(__double2hiint(v[1]))};
    } else if constexpr (sizeof(S) == 4) {
        q = {__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])};
    } else {
        q = {pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7])};
    }
    *reinterpret_cast<Qu*>(p) = q;
}
// N elements from p on, with the ordinary cache policy: what is read again.
template <int N, class W> __device__ __forceinline__ void load_again(const W* p, typename Elem<W>::acc* v) {
    constexpr int M = kVec<W>;
    static_assert(M <= N && N % M == 0, "whole chunks");
#pragma unroll
    for (int k = 0; k < N; k += M) {
        Chunk<W> c;
        c.q = *reinterpret_cast<const Qu*>(p + k);
#pragma unroll
        for (int j = 0; j < M; ++j) v[k + j] = c.at(j);
    }
}

// ------------------------------------------------------------------ rows of any length

// One block a row, any h: the row is read again for every pass, from the
// caches.  For float64, and for rows that are too short or too long for
// registers (below).  3355 rows of 20000 bfloat16: forward 78 us, 3.5 TB/s;
// backward with the residual's gradient 186 us, which reads dy and x a second
// time for the columns' sums.  float64, 16384 rows of 4096: 298 and 644 us.
//
// A thread's share of a row has no bound but h / 256, so the sums B of rows
// past the registers are double: the values of a chunk are added in pairs in
// the rows' type (three additions at most), the chunks' sums in double, and one
// rounding to float ends it.  (In float a row of 2^26 equal values had a mean
// off by 0.25 %.)  Rows under a chunk, at most seven values, keep float sums:
// 4 M rows of 5 bfloat16 forward 2.8 ms, with double ones 5.0, the exchange
// between lanes being two words.

// Sum of v over the block's threads, in every thread; `s` holds one value a
// wave.  Ends with all threads past their reads of `s`.
template <class B> __device__ __forceinline__ B block_sum(B v, B* s) {
    v = lane_sum<64>(v);
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
    __syncthreads();
    B t = s[0];
#pragma unroll
    for (int i = 1; i < kNormWaves; ++i) t += s[i];
    __syncthreads();
    return t;
}
// The sum of a piece's values, added in pairs (v is used up).
template <int N, class A> __device__ __forceinline__ A pair_sum(A (&v)[N]) {
#pragma unroll
    for (int d = 1; d < N; d *= 2)
#pragma unroll
        for (int j = 0; j < N; j += 2 * d) v[j] += v[j + d];
    return v[0];
}

// Calls f(first, count) for the thread's pieces of a row: whole chunks, then single elements of the rest.
template <int N, class F> __device__ __forceinline__ void for_pieces(int h, F f) {
    const int whole = h / N * N;
    for (int i = threadIdx.x * N; i < whole; i += kNormThreads * N) f(i, std::integral_constant<int, N>());
    for (int i = whole + threadIdx.x; i < h; i += kNormThreads) f(i, std::integral_constant<int, 1>());
}
template <int N, class S> __device__ __forceinline__ void piece(const S* p, int i, typename Elem<S>::acc* v) {
    if constexpr (N == 1)
        v[0] = Elem<S>::ld(p, i);
    else
        load_again<N>(p + i, v);
}

template <class B, class S, class W>
__global__ __launch_bounds__(kNormThreads) void norm_fwd_kernel(const S* __restrict__ x, const W* __restrict__ w,
                                                                const W* __restrict__ b, int64_t T, int h,
                                                                typename Elem<S>::acc eps, S* __restrict__ y,
                                                                typename Elem<S>::acc* __restrict__ mean,
                                                                typename Elem<S>::acc* __restrict__ rstd) {
    using A = typename Elem<S>::acc;
    __shared__ B s[kNormWaves];
    for (int64_t t = blockIdx.x; t < T; t += gridDim.x) {
        const S* row = x + t * h;
        B sum = 0, sq = 0;
        for_pieces<kVec<S>>(h, [&](int i, auto n) {
            constexpr int N = decltype(n)::value;
            A v[N];
            piece<N>(row, i, v);
            sum += pair_sum<N>(v);
        });
        const A mu = static_cast<A>(block_sum(sum, s) / B(h));
        for_pieces<kVec<S>>(h, [&](int i, auto n) {
            constexpr int N = decltype(n)::value;
            A v[N];
            piece<N>(row, i, v);
#pragma unroll
            for (int j = 0; j < N; ++j) v[j] = (v[j] - mu) * (v[j] - mu);
            sq += pair_sum<N>(v);
        });
        const A r = rsqrt_t(static_cast<A>(block_sum(sq, s) / B(h)) + eps);
        for_pieces<kVec<S>>(h, [&](int i, auto n) {
            constexpr int N = decltype(n)::value;
            A v[N], wv[N], bv[N];
            piece<N>(row, i, v);
            if (w) piece<N>(w, i, wv);
            if (b) piece<N>(b, i, bv);
#pragma unroll
            for (int j = 0; j < N; ++j) {
                v[j] = (v[j] - mu) * r;
                if (w) v[j] *= wv[j];
                if (b) v[j] += bv[j];
            }
            if constexpr (N == 1)
                Elem<S>::st(y + t * h, i, v[0]);
            else
                store_chunk(y + t * h + i, v);
        });
        if (threadIdx.x == 0) {
            mean[t] = mu;
            rstd[t] = r;
        }
    }
}

// The input gradient.
template <class B, class S, class W>
__global__ __launch_bounds__(kNormThreads) void norm_bwd_rows_kernel(
    const S* __restrict__ dy, const S* __restrict__ x, const W* __restrict__ w,
    const typename Elem<S>::acc* __restrict__ mean, const typename Elem<S>::acc* __restrict__ rstd,
    const S* __restrict__ dres, int64_t T, int h, S* __restrict__ dx) {
    using A = typename Elem<S>::acc;
    __shared__ B s[kNormWaves];
    for (int64_t t = blockIdx.x; t < T; t += gridDim.x) {
        const A mu = mean[t], r = rstd[t];
        const S *xr = x + t * h, *gr = dy + t * h;
        B s1 = 0, s2 = 0;
        const auto load = [&](int i, auto n, A* g, A* xh) {
            constexpr int N = decltype(n)::value;
            A wv[N];
            piece<N>(gr, i, g);
            piece<N>(xr, i, xh);
            if (w) piece<N>(w, i, wv);
#pragma unroll
            for (int j = 0; j < N; ++j) {
                xh[j] = (xh[j] - mu) * r;
                if (w) g[j] *= wv[j];
            }
        };
        for_pieces<kVec<S>>(h, [&](int i, auto n) {
            constexpr int N = decltype(n)::value;
            A g[N], xh[N];
            load(i, n, g, xh);
#pragma unroll
            for (int j = 0; j < N; ++j) xh[j] *= g[j];
            s1 += pair_sum<N>(xh);
            s2 += pair_sum<N>(g);
        });
        const A c1 = static_cast<A>(block_sum(s1, s) / B(h)), c2 = static_cast<A>(block_sum(s2, s) / B(h));
        for_pieces<kVec<S>>(h, [&](int i, auto n) {
            constexpr int N = decltype(n)::value;
            A g[N], xh[N], v[N];
            load(i, n, g, xh);
            if (dres) piece<N>(dres + t * h, i, v);
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const A d = r * (g[j] - c2 - xh[j] * c1);
                v[j] = dres ? d + v[j] : d;
            }
            if constexpr (N == 1)
                Elem<S>::st(dx + t * h, i, v[0]);
            else
                store_chunk(dx + t * h + i, v);
        });
    }
}

// Partial sums of dw and db over a slice of the rows, a chunk of columns a lane: part[slice][0 | 1][h].  The
// columns behind the last whole chunk go to the single lanes of the last block.  Of rows past the registers a lane
// takes at most some 512 (norm_slices), one float sum; of shorter rows, single elements, T / 1024 and more: 64
// at a time in float, these sums in double (16 K values of 0.1 one after the other in float are off by 1.5e-4).
// Doubles for whole chunks took 45 -> 103 us.
template <class S>
__global__ __launch_bounds__(kNormThreads) void norm_bwd_cols_kernel(
    const S* __restrict__ dy, const S* __restrict__ x, const typename Elem<S>::acc* __restrict__ mean,
    const typename Elem<S>::acc* __restrict__ rstd, int64_t T, int h, int slices,
    typename Elem<S>::acc* __restrict__ part) {
    using A = typename Elem<S>::acc;
    constexpr int N = kVec<S>;
    __shared__ A sums[kNormWaves][2 * N][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t t0 = T * blockIdx.y / slices, t1 = T * (blockIdx.y + 1) / slices;
    const int whole = h / N;                                 // chunks; then h % N columns on their own
    const int c = blockIdx.x * 64 + lane;
    A* p = part + static_cast<int64_t>(blockIdx.y) * 2 * h;
    const auto add = [&](int col, auto n) {
        constexpr int M = decltype(n)::value;
        using B = typename std::conditional<M == 1, double, A>::type;
        B dw[M] = {}, db[M] = {};
        for (int64_t t = t0 + wave; t < t1;) {
            const int64_t end = M == 1 ? min(t1, t + 64 * kNormWaves) : t1;
            A pw[M] = {}, pb[M] = {};
            for (; t < end; t += kNormWaves) {
                A g[M], v[M];
                piece<M>(dy + t * h, col, g);
                piece<M>(x + t * h, col, v);
#pragma unroll
                for (int j = 0; j < M; ++j) {
                    pw[j] += g[j] * ((v[j] - mean[t]) * rstd[t]);
                    pb[j] += g[j];
                }
            }
#pragma unroll
            for (int j = 0; j < M; ++j) {
                dw[j] += pw[j];
                db[j] += pb[j];
            }
        }
#pragma unroll
        for (int j = 0; j < M; ++j) {
            sums[wave][j][lane] = static_cast<A>(dw[j]);
            sums[wave][N + j][lane] = static_cast<A>(db[j]);
        }
    };
    const bool chunk = c < whole, single = !chunk && c - whole < h % N;
    const int col = chunk ? c * N : whole * N + (c - whole);
    if (chunk) add(col, std::integral_constant<int, N>());
    if (single) add(col, std::integral_constant<int, 1>());
    __syncthreads();
    if (wave != 0 || !(chunk || single)) return;
    for (int j = 0; j < (chunk ? N : 1); ++j) {
        A dw = sums[0][j][lane], db = sums[0][N + j][lane];
#pragma unroll
        for (int i = 1; i < kNormWaves; ++i) {
            dw += sums[i][j][lane];
            db += sums[i][N + j][lane];
        }
        p[col + j] = dw;
        p[h + col + j] = db;
    }
}
// Column blocks of norm_bwd_cols_kernel.
inline int col_blocks(int h, int n) { return (h / n + h % n + 63) / 64; }

// dw, db = the sums of the partial rows, a column a lane: 16 waves each sum every 16th, then wave 0 their sums.
constexpr int kReduceThreads = 1024;
template <class A, class W>
__global__ __launch_bounds__(kReduceThreads) void norm_bwd_reduce_kernel(const A* __restrict__ part, int parts, int h,
                                                                         W* __restrict__ dw, W* __restrict__ db) {
    constexpr int kWaves = kReduceThreads / 64;
    __shared__ A s[kWaves][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t i = static_cast<int64_t>(blockIdx.x) * 64 + lane;
    A sum = 0;
    if (i < 2 * static_cast<int64_t>(h)) {
#pragma unroll 4
        for (int k = wave; k < parts; k += kWaves) sum += part[static_cast<int64_t>(k) * 2 * h + i];
    }
    s[wave][lane] = sum;
    __syncthreads();
    if (wave != 0 || i >= 2 * static_cast<int64_t>(h)) return;
#pragma unroll
    for (int k = 1; k < kWaves; ++k) sum += s[k][lane];
    W* out = i < h ? dw : db;
    if (out) Elem<W>::st(out, i < h ? i : i - h, sum);
}

// ------------------------------------------------------------------ rows in registers

// Rows of up to 2 x 16 bytes for each of up to 1024 threads are read once and
// held in registers: TPR threads (part of a wave, or whole waves) own a row,
// each of them NV chunks of 16 bytes, TPR * 16 bytes apart.  The blocks stay
// and walk the rows; the next row's loads are in flight while this one is
// reduced, and the weight (and, in the backward, the columns' sums of dw and
// db) stay in registers from row to row.  Against a block a row that reads it
// again for each pass: 16384 x 4096 bfloat16 forward 201 -> 46 us, backward
// (with a second read of dy and x for the columns' sums) 329 -> 100 us.
//
// The shape is the smallest that holds the row, since idle lanes cost: 64 M
// bfloat16 in rows of 64 took 364 us on a wave a row, 54 on 8 lanes; in rows
// of 2560 52 us forward and 117 backward on 256 threads, 48 and 105 on 192; in
// rows of 1100 69 and 139 on 128 threads, 49 and 98 to 106 on 64 with three
// chunks.
// A row within a wave also spares the barriers, which shows where the backward
// has no residual to read: rows of 2048 76 us on 128 threads, 65 on 64 with
// four chunks.  With a residual both take 94, and of few rows the four chunks
// 2.5 us longer; rows that end inside a chunk spill, and 4096-wide ones gained
// 8 % without a residual and lost 2 to 14 % elsewhere: two chunks, then.
//
// Rows that end inside a chunk (kTail): the last chunk is the row's last 16
// bytes, so it overlaps the one before it.  Its first `dup` elements count for
// no sum; both threads store the same bits to them.

// Where a thread's chunks lie: first element, how many of its first elements
// another chunk counts, whether it has any.
template <int N, int TPR, int NV, bool kTail> struct Place {
    int off[NV], dup[NV];
    bool on[NV];
    __device__ __forceinline__ Place(int i, int h) {
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int c = (i + v * TPR) * N;
            on[v] = c < h;
            off[v] = kTail ? min(c, h - N) : c;
            dup[v] = c - off[v];
        }
    }
    __device__ __forceinline__ bool counts(int v, int j) const { return !kTail || j >= dup[v]; }
};

// Sums of K values over the TPR threads of a row, in all of them.  `s` has a
// slot a wave; a call and the next one use different slots, so one barrier a
// call is enough.
template <int K, int TPR> __device__ __forceinline__ void row_sums(float (&v)[K], float (*s)[K]) {
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] = lane_sum<(TPR < 64 ? TPR : 64)>(v[k]);
    if constexpr (TPR > 64) {
        const int wave = threadIdx.x >> 6;
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int k = 0; k < K; ++k) s[wave][k] = v[k];
        __syncthreads();
        const int w0 = wave / (TPR / 64) * (TPR / 64);
#pragma unroll
        for (int k = 0; k < K; ++k) {
            v[k] = s[w0][k];
#pragma unroll
            for (int i = 1; i < TPR / 64; ++i) v[k] += s[w0 + i][k];
        }
    }
}
// Which of the block's rows a thread works on (the same in every lane of a wave, if a wave has only one).
template <int TPR> __device__ __forceinline__ int group_of() {
    const int g = static_cast<int>(threadIdx.x) / TPR;
    if constexpr (TPR >= 64) return __builtin_amdgcn_readfirstlane(g);
    return g;
}

// Forward: blocks of 256 threads or of one row, four waves a SIMD (three: 50.5 us for 16384 x 4096, four and
// six: 47 to 48).  Backward: one block a CU of 8 to 16 waves, which keeps the partial rows of dw and db at 256
// (three blocks of 256 threads a CU: the same 96 us, and 7 us instead of 4.5 for the sum of 768 partial rows).
constexpr int fwd_threads(int tpr) { return tpr == 192 ? 384 : tpr < 256 ? 256 : tpr; }
constexpr int bwd_threads(int tpr) { return tpr == 192 ? 576 : tpr < 384 ? 512 : tpr == 384 ? 768 : tpr; }
constexpr int kFwdThreadsPerCu = 1024;

template <class S, class W, int TPR, int NV, bool kTail>
__global__ __launch_bounds__(fwd_threads(TPR)) void norm_fwd_reg_kernel(const S* __restrict__ x,
                                                                        const W* __restrict__ w,
                                                                        const W* __restrict__ b, int64_t T, int h,
                                                                        float eps, S* __restrict__ y,
                                                                        float* __restrict__ mean,
                                                                        float* __restrict__ rstd) {
    constexpr int N = kVec<S>, G = fwd_threads(TPR) / TPR;
    __shared__ float red[2][fwd_threads(TPR) / 64][1];
    const int grp = group_of<TPR>();
    const Place<N, TPR, NV, kTail> at(threadIdx.x % TPR, h);
    float wv[NV][N], bv[NV][N];
    Chunk<S> cur[NV], nxt[NV];
    const int64_t stride = static_cast<int64_t>(gridDim.x) * G;
    int64_t t = static_cast<int64_t>(blockIdx.x) * G + grp;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        cur[v].q = Q{0, 0, 0, 0};
        if (at.on[v] && t < T) cur[v].load(x + t * h + at.off[v]);
    }
#pragma unroll
    for (int v = 0; v < NV; ++v) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            wv[v][j] = 1.0f;
            bv[v][j] = 0.0f;
        }
        if (w && at.on[v]) load_again<N>(w + at.off[v], wv[v]);
        if (b && at.on[v]) load_again<N>(b + at.off[v], bv[v]);
    }
    for (int64_t base = static_cast<int64_t>(blockIdx.x) * G; base < T; base += stride, t += stride) {
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            nxt[v].q = Q{0, 0, 0, 0};
            if (at.on[v] && t + stride < T) nxt[v].load(x + (t + stride) * h + at.off[v]);
        }
        float sum[1] = {0.0f}, sq[1] = {0.0f};
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
            for (int j = 0; j < N; ++j) sum[0] += at.counts(v, j) ? cur[v].at(j) : 0.0f;
        row_sums<1, TPR>(sum, red[0]);
        const float mu = sum[0] / static_cast<float>(h);
#pragma unroll
        for (int v = 0; v < NV; ++v)
            if (at.on[v]) {
#pragma unroll
                for (int j = 0; j < N; ++j) {
                    const float d = cur[v].at(j) - mu;
                    sq[0] += at.counts(v, j) ? d * d : 0.0f;
                }
            }
        row_sums<1, TPR>(sq, red[1]);
        const float r = rsqrt_t(sq[0] / static_cast<float>(h) + eps);
        if (t < T) {
#pragma unroll
            for (int v = 0; v < NV; ++v)
                if (at.on[v]) {
                    float o[N];
#pragma unroll
                    for (int j = 0; j < N; ++j) o[j] = (cur[v].at(j) - mu) * r * wv[v][j] + bv[v][j];
                    store_chunk(y + t * h + at.off[v], o);
                }
            if (threadIdx.x % TPR == 0) {
                mean[t] = mu;
                rstd[t] = r;
            }
        }
#pragma unroll
        for (int v = 0; v < NV; ++v) cur[v] = nxt[v];
    }
}

constexpr int kNormParts = 256;      // partial sums of dw and db (blocks of the backward): one a CU
constexpr int kNormTurns = 512;      // rows a group sums in float, one after the other; past them there are more blocks

// Up to so many turns one block takes all rows and writes dw and db itself, without the second launch: 4096-wide
// bfloat16, 4 rows (two turns) 12.4 us a call and 24.0 waited for, against 15.2 and 25.1 in two blocks; 8 rows
// (four turns) 11.9 and 26.5 against 15.2 and 25.4.
constexpr int kOneBlockTurns = 2;
// Blocks of the backward.
inline int64_t bwd_blocks(int64_t T, int tpr) {
    const int groups = bwd_threads(tpr) / tpr;
    const int64_t turns = (T + groups - 1) / groups;
    if (turns <= kOneBlockTurns) return 1;
    return std::min(turns, std::max<int64_t>(kNormParts, (turns + kNormTurns - 1) / kNormTurns));
}

template <class S, int NV> struct BwdRow {
    Chunk<S> x[NV], dy[NV], res[NV];
    float mu, r;
};

template <class S, class W, int TPR, int NV, bool kTail>
__global__ __launch_bounds__(bwd_threads(TPR)) void norm_bwd_reg_kernel(
    const S* __restrict__ dy, const S* __restrict__ x, const W* __restrict__ w, const float* __restrict__ mean,
    const float* __restrict__ rstd, const S* __restrict__ dres, int64_t T, int h, S* __restrict__ dx,
    W* __restrict__ dw, W* __restrict__ db, float* __restrict__ part) {
    constexpr int N = kVec<S>, G = bwd_threads(TPR) / TPR;
    // 16 waves a block, or four chunks a thread, leave no registers for the next row (16 waves of bfloat16 spill a
    // few all the same: rows of 12288 and 16384 run at 5.0 to 5.5 TB/s).
    constexpr bool kAhead = TPR < 1024 && NV < 4;
    __shared__ float red[2][bwd_threads(TPR) / 64][2];
    const int grp = group_of<TPR>();
    const int i = threadIdx.x % TPR;
    const Place<N, TPR, NV, kTail> at(i, h);
    float wv[NV][N], aw[NV][N], ab[NV][N];
    const int64_t stride = static_cast<int64_t>(gridDim.x) * G;
    int64_t t = static_cast<int64_t>(blockIdx.x) * G + grp;
    BwdRow<S, NV> cur, nxt;
    auto load = [&](BwdRow<S, NV>& row, int64_t at_row) {
        row.mu = row.r = 0.0f;
        if (at_row < T) {
            row.mu = mean[at_row];
            row.r = rstd[at_row];
        }
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            row.x[v].q = row.dy[v].q = row.res[v].q = Q{0, 0, 0, 0};
            if (at.on[v] && at_row < T) {
                const int64_t e = at_row * h + at.off[v];
                row.dy[v].load(dy + e);
                row.x[v].load(x + e);
                if (dres) row.res[v].load(dres + e);
            }
        }
    };
    load(cur, t);
#pragma unroll
    for (int v = 0; v < NV; ++v) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            wv[v][j] = 1.0f;
            aw[v][j] = ab[v][j] = 0.0f;
        }
        if (w && at.on[v]) load_again<N>(w + at.off[v], wv[v]);
    }
    int turn = 0;
    for (int64_t base = static_cast<int64_t>(blockIdx.x) * G; base < T; base += stride, t += stride, turn ^= 1) {
        if constexpr (kAhead) load(nxt, t + stride);
        float c[2] = {0.0f, 0.0f};   // sums of g xh and of g
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            float gx = 0.0f;
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const float d = cur.dy[v].at(j), xh = (cur.x[v].at(j) - cur.mu) * cur.r;
                aw[v][j] += d * xh;
                ab[v][j] += d;
                const float g = at.counts(v, j) ? d * wv[v][j] : 0.0f;
                gx += g * xh;
                c[1] += g;
            }
            // A chunk past the row is zeros, but -mean * rstd can be infinite where no xh of the row is.
            c[0] += at.on[v] ? gx : 0.0f;
        }
        if (dx) {
            row_sums<2, TPR>(c, red[turn]);
            const float c1 = c[0] / static_cast<float>(h), c2 = c[1] / static_cast<float>(h);
            if (t < T) {
#pragma unroll
                for (int v = 0; v < NV; ++v)
                    if (at.on[v]) {
                        float o[N];
#pragma unroll
                        for (int j = 0; j < N; ++j) {
                            const float xh = (cur.x[v].at(j) - cur.mu) * cur.r;
                            o[j] = cur.r * (cur.dy[v].at(j) * wv[v][j] - c2 - xh * c1);
                            if (dres) o[j] += cur.res[v].at(j);
                        }
                        store_chunk(dx + t * h + at.off[v], o);
                    }
            }
        }
        if constexpr (kAhead)
            cur = nxt;
        else
            load(cur, t + stride);
    }
    if (!dw && !db) return;
    // The block's rows: the sums of a wave's groups, then the waves' (or groups') one after the other, then a
    // partial row each of dw and db (or the result itself, if this block had all rows).  All of it is float: 1500
    // rows of 1365 float32 are off by 1.2e-7 of themselves (rms), where a sum in double, rounded once, is off by 0.4e-7.
    if constexpr (TPR < 64) {
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
            for (int j = 0; j < N; ++j)
#pragma unroll
                for (int d = TPR; d < 64; d *= 2) {
                    aw[v][j] += __shfl_xor(aw[v][j], d, 64);
                    ab[v][j] += __shfl_xor(ab[v][j], d, 64);
                }
    }
    constexpr int kParts = TPR < 64 ? bwd_threads(TPR) / 64 : G;
    const int mine = TPR < 64 ? static_cast<int>(threadIdx.x >> 6) : grp;
    const bool has = TPR >= 64 || (threadIdx.x & 63) < TPR;
    if constexpr (kParts > 1) {
        // In pairs: half of the parts leave theirs in LDS, the other half adds it; parts that had no row are left out.
        const int64_t rows = T - static_cast<int64_t>(blockIdx.x) * G, lived = (rows * TPR + 63) / 64;
        const int live = static_cast<int>(min(TPR < 64 ? lived : rows, static_cast<int64_t>(kParts)));
        __shared__ __align__(16) float4 sums[kParts / 2][2 * NV * N / 4 * TPR];
        for (int s = 1; s < live; s *= 2) {
            __syncthreads();
            float4* slot = sums[mine / (2 * s) % (kParts / 2)];
            if (mine % (2 * s) == s && mine < live && has) {
#pragma unroll
                for (int v = 0; v < NV; ++v)
#pragma unroll
                    for (int j = 0; j < N; j += 4) {
                        const int q = (v * N + j) / 4;
                        slot[q * TPR + i] = make_float4(aw[v][j], aw[v][j + 1], aw[v][j + 2], aw[v][j + 3]);
                        slot[(NV * N / 4 + q) * TPR + i] = make_float4(ab[v][j], ab[v][j + 1], ab[v][j + 2], ab[v][j + 3]);
                    }
            }
            __syncthreads();
            if (mine % (2 * s) == 0 && mine + s < live && has) {
#pragma unroll
                for (int v = 0; v < NV; ++v)
#pragma unroll
                    for (int j = 0; j < N; j += 4) {
                        const int q = (v * N + j) / 4;
                        const float4 a = slot[q * TPR + i], b = slot[(NV * N / 4 + q) * TPR + i];
                        aw[v][j] += a.x, aw[v][j + 1] += a.y, aw[v][j + 2] += a.z, aw[v][j + 3] += a.w;
                        ab[v][j] += b.x, ab[v][j + 1] += b.y, ab[v][j + 2] += b.z, ab[v][j + 3] += b.w;
                    }
            }
        }
    }
    if (mine != 0 || !has) return;
    float* p = part + static_cast<int64_t>(blockIdx.x) * 2 * h;
#pragma unroll
    for (int v = 0; v < NV; ++v)
        if (at.on[v]) {
            if (gridDim.x == 1) {
                // (Where a chunk overlaps the one before, both threads summed the same rows: the same bits again.)
#pragma unroll
                for (int k = 0; k < N; k += kVec<W>) {
                    if (dw) store_chunk(dw + at.off[v] + k, aw[v] + k);
                    if (db) store_chunk(db + at.off[v] + k, ab[v] + k);
                }
            } else {
#pragma unroll
                for (int k = 0; k < N; k += 4) {
                    store_chunk(p + at.off[v] + k, aw[v] + k);
                    store_chunk(p + h + at.off[v] + k, ab[v] + k);
                }
            }
        }
}

constexpr int kNormMaxSlices = 256;
constexpr int kNormSliceRows = 2048;   // at most, where a lane's sums are float: 512 rows a lane
inline int norm_slices(int64_t T, int h, int dtype) {
    // About eight blocks a CU of float64's chunks.
    const int64_t want = std::max<int64_t>(1, 2048 / ((h + 127) / 128));
    const int64_t slices = std::max<int64_t>(1, std::min({want, (T + 15) / 16, int64_t(kNormMaxSlices)}));
    const bool in_double = dtype == RHP_F64 || h * static_cast<int64_t>(dtype_bytes(dtype)) < 16;
    const int64_t least = in_double ? 1 : (T + kNormSliceRows - 1) / kNormSliceRows;
    return static_cast<int>(std::max(slices, std::min<int64_t>(least, 65535)));
}

inline unsigned row_grid(int64_t T) { return static_cast<unsigned>(std::min<int64_t>(T, 1 << 20)); }

inline bool element_aligned(std::initializer_list<const void*> ps, int dt) {
    for (const void* p : ps)
        if (reinterpret_cast<uintptr_t>(p) & (dtype_bytes(dt) - 1)) return false;
    return true;
}

int check_norm(const char* what, int dtype, int w_dtype, int64_t T, int h) {
    RHP_REQUIRE(dtype == RHP_F64 || dtype == RHP_F32 || dtype == RHP_BF16,
                std::string(what) + ": unsupported dtype " + dtype_name(dtype));
    RHP_REQUIRE(w_dtype == dtype || (dtype == RHP_BF16 && w_dtype == RHP_F32),
                std::string(what) + ": weight and bias must have the rows' dtype (or float32 with bfloat16 rows)");
    RHP_REQUIRE(T >= 0, std::string(what) + ": negative row count");
    RHP_REQUIRE(h >= 1 && h <= (1 << 26), std::string(what) + ": h must be between 1 and 2^26");
    return 0;
}

// How the register kernels hold a row: threads and chunks a thread, 0 threads for rows shorter than a chunk or
// longer than 2048 chunks and for float64.  By h and the type alone (and whether the backward has a residual), so
// that a row's bits do not depend on the batch it is in.  four: whether four chunks a thread pay.
struct RowShape {
    int tpr, nv;
};
inline RowShape row_shape(int dtype, int h, bool four) {
    if (dtype == RHP_F64) return {0, 0};
    const int n = 16 / static_cast<int>(dtype_bytes(dtype));
    if (h < n || h > 2048 * n) return {0, 0};
    for (const RowShape r : {RowShape{8, 2}, {16, 2}, {32, 2}, {64, 2}, {64, 3}, {64, 4}, {128, 2}, {192, 2}, {256, 2},
                             {384, 2}, {512, 2}})
        if (r.tpr * r.nv * n >= h && (r.nv < 4 || (four && h % n == 0))) return r;
    return {1024, 2};
}
// f(threads, chunks) as integral constants for a row_shape() that has threads.
template <class F> int with_row_shape(RowShape r, F f) {
    using Two = std::integral_constant<int, 2>;
    switch (r.tpr) {
        case 8: return f(std::integral_constant<int, 8>(), Two());
        case 16: return f(std::integral_constant<int, 16>(), Two());
        case 32: return f(std::integral_constant<int, 32>(), Two());
        case 64:
            if (r.nv == 3) return f(std::integral_constant<int, 64>(), std::integral_constant<int, 3>());
            if (r.nv == 4) return f(std::integral_constant<int, 64>(), std::integral_constant<int, 4>());
            return f(std::integral_constant<int, 64>(), Two());
        case 128: return f(std::integral_constant<int, 128>(), Two());
        case 192: return f(std::integral_constant<int, 192>(), Two());
        case 256: return f(std::integral_constant<int, 256>(), Two());
        case 384: return f(std::integral_constant<int, 384>(), Two());
        case 512: return f(std::integral_constant<int, 512>(), Two());
        default: return f(std::integral_constant<int, 1024>(), Two());
    }
}

// f(a zero of the type that the any-length kernels sum in): the rows' own for short rows, else double.
template <class A, class F> int with_sums(bool few, F f) {
    if (few) return f(A(0));
    return f(0.0);
}

// f(whether rows end inside a chunk); rows of four chunks a thread do not (row_shape).
template <int NV, class F> int with_tail(bool tail, F f) {
    if constexpr (NV < 4)
        if (tail) return f(std::true_type());
    return f(std::false_type());
}

template <class S, class W>
int norm_fwd(const void* x, const void* w, const void* b, int64_t T, int h, double eps, void* y, void* mean,
             void* rstd, hipStream_t stream) {
    using A = typename Elem<S>::acc;
    const S* xp = static_cast<const S*>(x);
    const W *wp = static_cast<const W*>(w), *bp = static_cast<const W*>(b);
    S* yp = static_cast<S*>(y);
    A *mp = static_cast<A*>(mean), *rp = static_cast<A*>(rstd);
    if constexpr (sizeof(S) < 8) {
        auto launch = [&](auto tpr, auto chunks) {
            constexpr int TPR = decltype(tpr)::value, B = fwd_threads(TPR), G = B / TPR;
            constexpr int NV = std::min<int>(decltype(chunks)::value, 3);   // four are the backward's
            const int64_t most = int64_t(device_cus()) * std::max(1, (kFwdThreadsPerCu + B / 2) / B);
            const dim3 grid(static_cast<unsigned>(std::min<int64_t>((T + G - 1) / G, most)));
            const auto go = [&](auto tl) {
                hipLaunchKernelGGL((norm_fwd_reg_kernel<S, W, TPR, NV, decltype(tl)::value>), grid, dim3(B), 0, stream,
                                   xp, wp, bp, T, h, static_cast<float>(eps), yp, mp, rp);
                return check_launch("norm_fwd_reg_kernel");
            };
            return with_tail<NV>(h % kVec<S> != 0, go);
        };
        const RowShape shape = row_shape(sizeof(S) == 4 ? RHP_F32 : RHP_BF16, h, false);
        if (shape.tpr) return with_row_shape(shape, launch);
    }
    return with_sums<A>(h < kVec<S>, [&](auto b) {
        hipLaunchKernelGGL((norm_fwd_kernel<decltype(b), S, W>), dim3(row_grid(T)), dim3(kNormThreads), 0, stream, xp,
                           wp, bp, T, h, static_cast<A>(eps), yp, mp, rp);
        return check_launch("norm_fwd_kernel");
    });
}

template <class S, class W>
int norm_bwd(const void* dy, const void* x, const void* w, const void* mean, const void* rstd, const void* dres,
             int64_t T, int h, void* dx, void* dw, void* db, void* ws, hipStream_t stream) {
    using A = typename Elem<S>::acc;
    const S *dyp = static_cast<const S*>(dy), *xp = static_cast<const S*>(x), *resp = static_cast<const S*>(dres);
    const W* wp = static_cast<const W*>(w);
    const A *mp = static_cast<const A*>(mean), *rp = static_cast<const A*>(rstd);
    S* dxp = static_cast<S*>(dx);
    W *dwp = static_cast<W*>(dw), *dbp = static_cast<W*>(db);
    A* part = static_cast<A*>(ws);
    const bool sums = dw || db;
    auto reduce = [&](int parts) {
        hipLaunchKernelGGL((norm_bwd_reduce_kernel<A, W>), dim3((2 * static_cast<int64_t>(h) + 63) / 64),
                           dim3(kReduceThreads), 0, stream, part, parts, h, dwp, dbp);
        return check_launch("norm_bwd_reduce_kernel");
    };
    if (T == 0) return sums ? reduce(0) : 0;
    if constexpr (sizeof(S) < 8) {
        auto launch = [&](auto tpr, auto chunks) {
            constexpr int TPR = decltype(tpr)::value, NV = decltype(chunks)::value, B = bwd_threads(TPR);
            const int64_t nb = bwd_blocks(T, TPR);
            const auto go = [&](auto tl) {
                hipLaunchKernelGGL((norm_bwd_reg_kernel<S, W, TPR, NV, decltype(tl)::value>),
                                   dim3(static_cast<unsigned>(nb)), dim3(B), 0, stream, dyp, xp, wp, mp, rp, resp, T, h,
                                   dxp, dwp, dbp, part);
                return check_launch("norm_bwd_reg_kernel");
            };
            const int rc = with_tail<NV>(h % kVec<S> != 0, go);
            return rc || !sums || nb == 1 ? rc : reduce(static_cast<int>(nb));
        };
        const RowShape shape = row_shape(sizeof(S) == 4 ? RHP_F32 : RHP_BF16, h, !dres);
        if (shape.tpr) return with_row_shape(shape, launch);
    }
    if (dx) {
        const int rc = with_sums<A>(h < kVec<S>, [&](auto b) {
            hipLaunchKernelGGL((norm_bwd_rows_kernel<decltype(b), S, W>), dim3(row_grid(T)), dim3(kNormThreads), 0,
                               stream, dyp, xp, wp, mp, rp, resp, T, h, dxp);
            return check_launch("norm_bwd_rows_kernel");
        });
        if (rc) return rc;
    }
    if (!sums) return 0;
    const int slices = norm_slices(T, h, sizeof(S) == 8 ? RHP_F64 : sizeof(S) == 4 ? RHP_F32 : RHP_BF16);
    hipLaunchKernelGGL(norm_bwd_cols_kernel<S>, dim3(col_blocks(h, kVec<S>), slices), dim3(kNormThreads), 0, stream, dyp,
                       xp, mp, rp, T, h, slices, part);
    if (int rc = check_launch("norm_bwd_cols_kernel")) return rc;
    return reduce(slices);
}

}  // namespace
}  // namespace rhp

using namespace rhp;

extern "C" int rhp_layer_norm_fwd(const void* x, int dtype, const void* w, const void* b, int w_dtype, int64_t T,
                                  int h, double eps, void* y, void* mean, void* rstd, hipStream_t stream) {
    clear_error();
    if (int rc = check_norm("rhp_layer_norm_fwd", dtype, w_dtype, T, h)) return rc;
    RHP_REQUIRE(eps >= 0.0, "rhp_layer_norm_fwd: eps must not be negative");
    if (T == 0) return 0;
    RHP_REQUIRE(x && y && mean && rstd, "rhp_layer_norm_fwd: null pointer");
    RHP_REQUIRE(x != y, "rhp_layer_norm_fwd: y must not be x");
    RHP_REQUIRE(element_aligned({x, y}, dtype) && element_aligned({w, b}, w_dtype) &&
                    element_aligned({mean, rstd}, dtype == RHP_F64 ? RHP_F64 : RHP_F32),
                "rhp_layer_norm_fwd: a tensor is not aligned to its elements");
    const auto run = [&](auto f) { return f(x, w, b, T, h, eps, y, mean, rstd, stream); };
    if (dtype == RHP_F64) return run(norm_fwd<double, double>);
    if (dtype == RHP_F32) return run(norm_fwd<float, float>);
    return w_dtype == RHP_F32 ? run(norm_fwd<bf16, float>) : run(norm_fwd<bf16, bf16>);
}

extern "C" size_t rhp_layer_norm_bwd_workspace_bytes(int64_t T, int h, int dtype) {
    if (T < 0 || h <= 0) return 0;
    int64_t parts = 0;   // with or without a residual's gradient
    for (const bool four : {false, true}) {
        const int tpr = row_shape(dtype, h, four).tpr;
        parts = std::max<int64_t>(parts, tpr ? bwd_blocks(T, tpr) : norm_slices(T, h, dtype));
    }
    return static_cast<size_t>(parts) * 2 * h * (dtype == RHP_F64 ? 8 : 4);
}

extern "C" int rhp_layer_norm_bwd(const void* dy, const void* x, int dtype, const void* w, int w_dtype,
                                  const void* mean, const void* rstd, const void* dres, int64_t T, int h, void* dx,
                                  void* dw, void* db, void* workspace, size_t workspace_bytes, hipStream_t stream) {
    clear_error();
    if (int rc = check_norm("rhp_layer_norm_bwd", dtype, w_dtype, T, h)) return rc;
    RHP_REQUIRE(T == 0 || (dy && x && mean && rstd), "rhp_layer_norm_bwd: null pointer");
    RHP_REQUIRE(T == 0 || !dx || (dx != dy && dx != x && dx != dres), "rhp_layer_norm_bwd: dx must not be an input");
    RHP_REQUIRE(dx || !dres, "rhp_layer_norm_bwd: the residual's gradient goes into dx, which is null");
    RHP_REQUIRE(element_aligned({dy, x, dres, dx}, dtype) && element_aligned({w, dw, db}, w_dtype) &&
                    element_aligned({mean, rstd}, dtype == RHP_F64 ? RHP_F64 : RHP_F32),
                "rhp_layer_norm_bwd: a tensor is not aligned to its elements");
    RHP_REQUIRE((!dw && !db) || (aligned16(workspace) && workspace &&
                                 workspace_bytes >= rhp_layer_norm_bwd_workspace_bytes(T, h, dtype)),
                "rhp_layer_norm_bwd: workspace smaller than rhp_layer_norm_bwd_workspace_bytes(), null or unaligned");
    const auto run = [&](auto f) { return f(dy, x, w, mean, rstd, dres, T, h, dx, dw, db, workspace, stream); };
    if (dtype == RHP_F64) return run(norm_bwd<double, double>);
    if (dtype == RHP_F32) return run(norm_bwd<float, float>);
    return w_dtype == RHP_F32 ? run(norm_bwd<bf16, float>) : run(norm_bwd<bf16, bf16>);
}
