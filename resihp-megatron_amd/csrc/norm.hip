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
// Sums and statistics are float (double for double rows); a bfloat16 result
// is rounded once, when it is stored.  Nothing uses atomics: every sum has an
// order fixed by the sizes, so results are reproducible bit for bit.

#include <algorithm>
#include <initializer_list>

#include "rhp_common.h"

namespace rhp {
namespace {

constexpr int kNormThreads = 256;
constexpr int kNormWaves = kNormThreads / 64;

__device__ __forceinline__ float rsqrt_t(float x) { return 1.0f / __builtin_sqrtf(x); }
__device__ __forceinline__ double rsqrt_t(double x) { return 1.0 / __builtin_sqrt(x); }

template <class A> __device__ __forceinline__ A wave_sum(A v) {
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) v += __shfl_xor(v, d, 64);
    return v;
}

// Sum of v over the block's threads, in every thread; `s` holds one value a
// wave.  Ends with all threads past their reads of `s`.
template <class A> __device__ __forceinline__ A block_sum(A v, A* s) {
    v = wave_sum(v);
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
    __syncthreads();
    A t = s[0];
#pragma unroll
    for (int i = 1; i < kNormWaves; ++i) t += s[i];
    __syncthreads();
    return t;
}

// One block a row, any h: the row is read three times, the last two from the caches.
template <class S, class W>
__global__ __launch_bounds__(kNormThreads) void norm_fwd_kernel(const S* __restrict__ x, const W* __restrict__ w,
                                                                const W* __restrict__ b, int64_t T, int h,
                                                                typename Elem<S>::acc eps, S* __restrict__ y,
                                                                typename Elem<S>::acc* __restrict__ mean,
                                                                typename Elem<S>::acc* __restrict__ rstd) {
    using A = typename Elem<S>::acc;
    __shared__ A s[kNormWaves];
    for (int64_t t = blockIdx.x; t < T; t += gridDim.x) {
        const S* row = x + t * h;
        A sum = 0;
        for (int i = threadIdx.x; i < h; i += kNormThreads) sum += Elem<S>::ld(row, i);
        const A mu = block_sum(sum, s) / A(h);
        A sq = 0;
        for (int i = threadIdx.x; i < h; i += kNormThreads) {
            const A d = Elem<S>::ld(row, i) - mu;
            sq += d * d;
        }
        const A r = rsqrt_t(block_sum(sq, s) / A(h) + eps);
        for (int i = threadIdx.x; i < h; i += kNormThreads) {
            A v = (Elem<S>::ld(row, i) - mu) * r;
            if (w) v *= static_cast<A>(Elem<W>::ld(w, i));
            if (b) v += static_cast<A>(Elem<W>::ld(b, i));
            Elem<S>::st(y + t * h, i, v);
        }
        if (threadIdx.x == 0) {
            mean[t] = mu;
            rstd[t] = r;
        }
    }
}

// The input gradient, one block a row, any h.
template <class S, class W>
__global__ __launch_bounds__(kNormThreads) void norm_bwd_rows_kernel(
    const S* __restrict__ dy, const S* __restrict__ x, const W* __restrict__ w,
    const typename Elem<S>::acc* __restrict__ mean, const typename Elem<S>::acc* __restrict__ rstd,
    const S* __restrict__ dres, int64_t T, int h, S* __restrict__ dx) {
    using A = typename Elem<S>::acc;
    __shared__ A s[kNormWaves];
    for (int64_t t = blockIdx.x; t < T; t += gridDim.x) {
        const A mu = mean[t], r = rstd[t];
        const S *xr = x + t * h, *gr = dy + t * h;
        A c1 = 0, c2 = 0;
        for (int i = threadIdx.x; i < h; i += kNormThreads) {
            const A g = Elem<S>::ld(gr, i) * (w ? static_cast<A>(Elem<W>::ld(w, i)) : A(1));
            c1 += g * ((Elem<S>::ld(xr, i) - mu) * r);
            c2 += g;
        }
        c1 = block_sum(c1, s) / A(h);
        c2 = block_sum(c2, s) / A(h);
        for (int i = threadIdx.x; i < h; i += kNormThreads) {
            const A g = Elem<S>::ld(gr, i) * (w ? static_cast<A>(Elem<W>::ld(w, i)) : A(1));
            const A xh = (Elem<S>::ld(xr, i) - mu) * r;
            A v = r * (g - c2 - xh * c1);
            if (dres) v += Elem<S>::ld(dres + t * h, i);
            Elem<S>::st(dx + t * h, i, v);
        }
    }
}

// Partial sums of dw and db over a slice of the rows: part[slice][0 | 1][h].
template <class S>
__global__ __launch_bounds__(kNormThreads) void norm_bwd_cols_kernel(
    const S* __restrict__ dy, const S* __restrict__ x, const typename Elem<S>::acc* __restrict__ mean,
    const typename Elem<S>::acc* __restrict__ rstd, int64_t T, int h, int slices,
    typename Elem<S>::acc* __restrict__ part) {
    using A = typename Elem<S>::acc;
    __shared__ A sw[kNormWaves][64], sb[kNormWaves][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int col = blockIdx.x * 64 + lane;
    const int64_t t0 = T * blockIdx.y / slices, t1 = T * (blockIdx.y + 1) / slices;
    A dw = 0, db = 0;
    if (col < h)
        for (int64_t t = t0 + wave; t < t1; t += kNormWaves) {
            const A g = Elem<S>::ld(dy, t * h + col);
            dw += g * ((Elem<S>::ld(x, t * h + col) - mean[t]) * rstd[t]);
            db += g;
        }
    sw[wave][lane] = dw;
    sb[wave][lane] = db;
    __syncthreads();
    if (wave == 0 && col < h) {
#pragma unroll
        for (int i = 1; i < kNormWaves; ++i) {
            dw += sw[i][lane];
            db += sb[i][lane];
        }
        A* p = part + static_cast<int64_t>(blockIdx.y) * 2 * h;
        p[col] = dw;
        p[h + col] = db;
    }
}

// dw, db = the sum of the slices' partial sums.
template <class A, class W>
__global__ __launch_bounds__(kNormThreads) void norm_bwd_reduce_kernel(const A* __restrict__ part, int slices, int h,
                                                                       W* __restrict__ dw, W* __restrict__ db) {
    const int i = blockIdx.x * kNormThreads + threadIdx.x;
    if (i >= 2 * h) return;
    A sum = 0;
    for (int s = 0; s < slices; ++s) sum += part[static_cast<int64_t>(s) * 2 * h + i];
    W* out = i < h ? dw : db;
    if (out) Elem<W>::st(out, i < h ? i : i - h, sum);
}

constexpr int kNormMaxSlices = 256;
inline int norm_slices(int64_t T, int h) {
    const int64_t cols = (h + 63) / 64;
    const int64_t want = std::max<int64_t>(1, 2048 / cols);            // about eight blocks a CU
    return static_cast<int>(std::max<int64_t>(1, std::min({want, (T + 15) / 16, int64_t(kNormMaxSlices)})));
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
    RHP_REQUIRE(h >= 1 && h <= (1 << 28), std::string(what) + ": h must be between 1 and 2^28");
    return 0;
}

template <class S, class W>
int norm_fwd(const void* x, const void* w, const void* b, int64_t T, int h, double eps, void* y, void* mean,
             void* rstd, hipStream_t stream) {
    using A = typename Elem<S>::acc;
    hipLaunchKernelGGL((norm_fwd_kernel<S, W>), dim3(row_grid(T)), dim3(kNormThreads), 0, stream,
                       static_cast<const S*>(x), static_cast<const W*>(w), static_cast<const W*>(b), T, h,
                       static_cast<A>(eps), static_cast<S*>(y), static_cast<A*>(mean), static_cast<A*>(rstd));
    return check_launch("norm_fwd_kernel");
}

template <class S, class W>
int norm_bwd(const void* dy, const void* x, const void* w, const void* mean, const void* rstd, const void* dres,
             int64_t T, int h, void* dx, void* dw, void* db, void* ws, hipStream_t stream) {
    using A = typename Elem<S>::acc;
    const S *dyp = static_cast<const S*>(dy), *xp = static_cast<const S*>(x);
    const A *mp = static_cast<const A*>(mean), *rp = static_cast<const A*>(rstd);
    if (dx && T > 0) {
        hipLaunchKernelGGL((norm_bwd_rows_kernel<S, W>), dim3(row_grid(T)), dim3(kNormThreads), 0, stream, dyp, xp,
                           static_cast<const W*>(w), mp, rp, static_cast<const S*>(dres), T, h, static_cast<S*>(dx));
        if (int rc = check_launch("norm_bwd_rows_kernel")) return rc;
    }
    if (dw || db) {
        const int slices = norm_slices(T, h);
        A* part = static_cast<A*>(ws);
        hipLaunchKernelGGL(norm_bwd_cols_kernel<S>, dim3((h + 63) / 64, slices), dim3(kNormThreads), 0, stream, dyp,
                           xp, mp, rp, T, h, slices, part);
        if (int rc = check_launch("norm_bwd_cols_kernel")) return rc;
        hipLaunchKernelGGL((norm_bwd_reduce_kernel<A, W>), dim3((2 * h + kNormThreads - 1) / kNormThreads),
                           dim3(kNormThreads), 0, stream, part, slices, h, static_cast<W*>(dw), static_cast<W*>(db));
        if (int rc = check_launch("norm_bwd_reduce_kernel")) return rc;
    }
    return 0;
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
    RHP_REQUIRE(element_aligned({x, y}, dtype) && element_aligned({w, b}, w_dtype) &&
                    element_aligned({mean, rstd}, dtype == RHP_F64 ? RHP_F64 : RHP_F32),
                "rhp_layer_norm_fwd: a tensor is not aligned to its elements");
    if (dtype == RHP_F64) return norm_fwd<double, double>(x, w, b, T, h, eps, y, mean, rstd, stream);
    if (dtype == RHP_F32) return norm_fwd<float, float>(x, w, b, T, h, eps, y, mean, rstd, stream);
    if (w_dtype == RHP_F32) return norm_fwd<bf16, float>(x, w, b, T, h, eps, y, mean, rstd, stream);
    return norm_fwd<bf16, bf16>(x, w, b, T, h, eps, y, mean, rstd, stream);
}

extern "C" size_t rhp_layer_norm_bwd_workspace_bytes(int64_t T, int h, int dtype) {
    if (T < 0 || h <= 0) return 0;
    return static_cast<size_t>(norm_slices(T, h)) * 2 * h * (dtype == RHP_F64 ? 8 : 4);
}

extern "C" int rhp_layer_norm_bwd(const void* dy, const void* x, int dtype, const void* w, int w_dtype,
                                  const void* mean, const void* rstd, const void* dres, int64_t T, int h, void* dx,
                                  void* dw, void* db, void* workspace, size_t workspace_bytes, hipStream_t stream) {
    clear_error();
    if (int rc = check_norm("rhp_layer_norm_bwd", dtype, w_dtype, T, h)) return rc;
    RHP_REQUIRE(T == 0 || (dy && x && mean && rstd), "rhp_layer_norm_bwd: null pointer");
    RHP_REQUIRE(dx || !dres, "rhp_layer_norm_bwd: the residual's gradient goes into dx, which is null");
    RHP_REQUIRE(element_aligned({dy, x, dres, dx}, dtype) && element_aligned({w, dw, db}, w_dtype) &&
                    element_aligned({mean, rstd}, dtype == RHP_F64 ? RHP_F64 : RHP_F32),
                "rhp_layer_norm_bwd: a tensor is not aligned to its elements");
    RHP_REQUIRE((!dw && !db) || (aligned16(workspace) && workspace &&
                                 workspace_bytes >= rhp_layer_norm_bwd_workspace_bytes(T, h, dtype)),
                "rhp_layer_norm_bwd: workspace smaller than rhp_layer_norm_bwd_workspace_bytes(), null or unaligned");
    if (dtype == RHP_F64) return norm_bwd<double, double>(dy, x, w, mean, rstd, dres, T, h, dx, dw, db, workspace, stream);
    if (dtype == RHP_F32) return norm_bwd<float, float>(dy, x, w, mean, rstd, dres, T, h, dx, dw, db, workspace, stream);
    if (w_dtype == RHP_F32) return norm_bwd<bf16, float>(dy, x, w, mean, rstd, dres, T, h, dx, dw, db, workspace, stream);
    return norm_bwd<bf16, bf16>(dy, x, w, mean, rstd, dres, T, h, dx, dw, db, workspace, stream);
}
