// AdamW over many tensors in one launch for gfx950, with the moments in 32
// bits or in 8, and the norm of all gradients that clips them.
//
// The reference has Adam only (resihp/runtime/optim.py:15-62: moments in the
// parameter's type, decay added to the gradient); this is the optimizer of
// large models beside it: decoupled decay, float32 moments and, if wanted,
// float32 masters for bfloat16 weights, or moments of one byte.
//
//   g = gradient * *grad_scale          (0 without a gradient, 1 without a scale)
//   m = b1 m + (1 - b1) g               v = b2 v + ((1 - b2) g) g
//   p = (1 - lr wd) p - (lr / bc1) * (m / (sqrt(v) / sqrt(bc2) + eps))
//   bc1 = 1 - b1^step, bc2 = 1 - b2^step
//
// in float (double for double weights), the moments one operation at a time
// (no fused multiply-adds: what a moment rounds to in 8 bits is then the same
// wherever these lines are evaluated in float); the weight is rounded once,
// when it is stored.
//
// Moments in 8 bits.  128 neighbouring elements share the exponent E of the
// largest of them (one byte a moment).  A code is the float's exponent and its
// top three mantissa bits, counted from the lowest binade the block keeps:
// sign and 7 bits over 16 binades for m, 8 bits over 32 binades for v (its
// square root spans as many as m); code 0 is zero.  The scale is a power of
// two, so a code's value is a float with four significant bits and no
// multiplication comes in.  Rounding is stochastic: up with the probability of
// the part cut off.  Nearest rounding would hold v still: b2 = 0.999 moves it
// by 1/1000 a step, and a code's step is 1/16 to 1/8.  What is too small for
// the block becomes 0 for m and the smallest code for v: a v of 0 under an m
// that is not would divide by eps.  A block with a value that is not finite
// (or past 1.875 * 2^127) stores E = 255 and reads as NaN.
// The random bits are a hash of (seed, step, the tensor's key, index).
//
// The step is bound by HBM: with float32 masters and moments 28 bytes a
// bfloat16 weight (0.57 G of them: 16.0 GB in 2.65 to 2.9 ms, 5.5 to 6.0 TB/s,
// with where the buffers lie), with 8-bit moments 10 (1.41 G: 14.1 GB in
// 2.55 to 2.7 ms, 5.2 to 5.5 TB/s).  There the codes' arithmetic fills nine
// tenths of the VALU's time beside the accesses: 55 operations an element
// (3.36 ms before the hardware's root and reciprocal, the exponent by lane
// exchange and the once-a-block checks; without any of it the same accesses
// take 2.56 ms).  Large blocks or several groups a thread for float32 moments
// were slower (two groups a thread 3.1 ms); two for 8-bit ones a little faster
// (2.69 -> 2.6).  Non-temporal or ordinary accesses, 128 to 512 threads a
// block: the same within what the buffers' places change.  Double weights take
// 56 bytes each: 0.27 G of them 3.39 ms, 4.4 TB/s; float ones 1.27 ms, 5.9.
#pragma clang fp contract(off)

#include <algorithm>
#include <cmath>
#include <cstring>
#include <exception>
#include <type_traits>
#include <utility>
#include <vector>

#include "rhp_common.h"

namespace rhp {
namespace {

constexpr int kThreads = 256;
constexpr int kGroups8 = 2, kElems8 = 8 * kGroups8, kElems32 = 4;   // elements a thread steps
constexpr int kBlock8 = kThreads * kElems8, kBlock32 = kThreads * kElems32;
constexpr int kScaleBlock = 128;       // elements that share an exponent
constexpr int kMaxGrads = 448;         // tensors a launch takes (their gradients' pointers are kernel arguments)
constexpr uint32_t kMaxBlocks = 1 << 20;   // blocks a launch takes: HIP has no launch of 2^32 threads

// ------------------------------------------------------------------ the plan

// A plan is an image of plain bytes, made on the host and copied to the
// device: a header, one record a tensor, and the tensor of every block.
constexpr uint32_t kPlanMagic = 0x57444152;
struct PlanHeader {
    uint32_t magic, count, blocks, state8;
    uint32_t f64, pad[3];
};
struct PlanTensor {
    void* p;
    float* master;
    void* m;
    void* v;
    uint8_t* scales;
    int64_t n;
    uint32_t key, block0;
    uint32_t dtype, decay;
};
static_assert(sizeof(PlanHeader) == 32 && sizeof(PlanTensor) == 64, "plan layout");

inline int64_t blocks_of(int64_t n, bool state8) {
    const int64_t k = state8 ? kBlock8 : kBlock32;
    return (n + k - 1) / k;
}
inline size_t plan_bytes(uint64_t count, uint64_t blocks) {
    return sizeof(PlanHeader) + count * sizeof(PlanTensor) + blocks * 4;
}

// ------------------------------------------------------------------ element access

// Tensors need only their element's alignment: gfx950 takes vector accesses
// at any address, and the aligned ones cost the same.
typedef uint32_t U2 __attribute__((ext_vector_type(2)));
typedef uint32_t U4 __attribute__((ext_vector_type(4)));
typedef U2 U2a __attribute__((aligned(1)));
typedef U4 U4a __attribute__((aligned(2)));
typedef U2 U2b __attribute__((aligned(2)));

// The plan's and the gradients' addresses come out of memory, so the compiler
// would take them for generic ones (flat accesses); they are global.
#define RHP_GLOBAL __attribute__((address_space(1)))
template <class V> __device__ __forceinline__ V load_at(const void* p) {
    return __builtin_nontemporal_load((const RHP_GLOBAL V*)(reinterpret_cast<uintptr_t>(p)));
}
template <class V, class T> __device__ __forceinline__ void store_at(void* p, T v) {
    __builtin_nontemporal_store(v, (RHP_GLOBAL V*)(reinterpret_cast<uintptr_t>(p)));
}

template <class S> struct Bits;
template <> struct Bits<double> {
    __device__ __forceinline__ static double ld(const void* p) { return load_at<double>(p); }
    __device__ __forceinline__ static void st(void* p, double v) { store_at<double>(p, v); }
};
template <> struct Bits<float> {
    __device__ __forceinline__ static float ld(const void* p) { return load_at<float>(p); }
    __device__ __forceinline__ static void st(void* p, float v) { store_at<float>(p, v); }
};
template <> struct Bits<bf16> {
    __device__ __forceinline__ static float ld(const void* p) { return bf16_to_f32(load_at<uint16_t>(p)); }
    __device__ __forceinline__ static void st(void* p, float v) { store_at<uint16_t>(p, f32_to_bf16(v)); }
};

// N elements from p + e on; those at n and past it read as 0 and are not stored.
template <int N, class S, class A> __device__ __forceinline__ void load_n(const S* p, int64_t e, int64_t n, A* v) {
    if (e + N <= n) {
        constexpr int kWords = N * static_cast<int>(sizeof(S)) / 4;
        uint32_t w[kWords];
        const char* q = reinterpret_cast<const char*>(p + e);
#pragma unroll
        for (int i = 0; i < kWords; i += 4) {
            if constexpr (kWords >= 4) {
                const U4 t = load_at<U4a>(q + 4 * i);
                w[i] = t[0]; w[i + 1] = t[1]; w[i + 2] = t[2]; w[i + 3] = t[3];
            } else {
                const U2 t = load_at<U2b>(q);
                w[0] = t[0]; w[1] = t[1];
            }
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if constexpr (sizeof(S) == 2)
                v[i] = i & 1 ? __uint_as_float(w[i / 2] & 0xffff0000u) : __uint_as_float(w[i / 2] << 16);
            else if constexpr (sizeof(S) == 4)
                v[i] = __uint_as_float(w[i]);
            else
                v[i] = __hiloint2double(static_cast<int>(w[2 * i + 1]), static_cast<int>(w[2 * i]));
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = e + i < n ? static_cast<A>(Bits<S>::ld(p + e + i)) : A(0);
    }
}

template <int N, class S, class A> __device__ __forceinline__ void store_n(S* p, int64_t e, int64_t n, const A* v) {
    if (e + N <= n) {
        constexpr int kWords = N * static_cast<int>(sizeof(S)) / 4;
        uint32_t w[kWords];
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if constexpr (sizeof(S) == 2) {
                if (i & 1) w[i / 2] = pack_bf16x2(v[i - 1], v[i]);
            } else if constexpr (sizeof(S) == 4) {
                w[i] = __float_as_uint(v[i]);
            } else {
                w[2 * i] = static_cast<uint32_t>(__double2loint(v[i]));
                w[2 * i + 1] = static_cast<uint32_t>(__double2hiint(v[i]));
            }
        }
        char* q = reinterpret_cast<char*>(p + e);
#pragma unroll
        for (int i = 0; i < kWords; i += 4) {
            if constexpr (kWords >= 4) {
                const U4 t = {w[i], w[i + 1], w[i + 2], w[i + 3]};
                store_at<U4a>(q + 4 * i, t);
            } else {
                const U2 t = {w[0], w[1]};
                store_at<U2b>(q, t);
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (e + i < n) Bits<S>::st(p + e + i, v[i]);
    }
}

// ------------------------------------------------------------------ moments in 8 bits

// A 32-bit hash: lowbias32 as C. Wellons published it (hash prospector), shifts and constants.
__host__ __device__ __forceinline__ uint32_t mix(uint32_t x) {
    x = (x ^ (x >> 16)) * 0x7FEB352Du;
    x = (x ^ (x >> 15)) * 0x846CA68Bu;
    return x ^ (x >> 16);
}
// Element e of the group of eight whose hash is x: one multiplication, the first half of that hash.
__device__ __forceinline__ uint32_t random_of(uint32_t x, uint32_t e) {
    x += e * 0x9E3779B9u;
    x = (x ^ (x >> 16)) * 0x7FEB352Du;
    return x ^ (x >> 15);
}

// Maximum over the 16 lanes of a DPP row, in all of them: neighbours, pairs, mirrored eights and sixteens.
__device__ __forceinline__ uint32_t max16(uint32_t v) {
    const auto of = [&](auto ctrl) {
        return static_cast<uint32_t>(
            __builtin_amdgcn_update_dpp(0, static_cast<int>(v), decltype(ctrl)::value, 0xf, 0xf, true));
    };
    v = max(v, of(std::integral_constant<int, 0xB1>()));    // quad_perm [1,0,3,2]
    v = max(v, of(std::integral_constant<int, 0x4E>()));    // quad_perm [2,3,0,1]
    v = max(v, of(std::integral_constant<int, 0x141>()));   // row_half_mirror
    return max(v, of(std::integral_constant<int, 0x140>()));   // row_mirror
}
// The exponent of a block whose largest magnitude has the bits `top`, such
// that a magnitude rounded up still has that exponent.
__device__ __forceinline__ uint32_t exponent_of(uint32_t top) { return min((top + 0xFFFFFu) >> 23, 255u); }
__device__ __forceinline__ int base_of(uint32_t e, int binades) {
    return max(static_cast<int>(e) - (binades - 1), 0) * 8;
}
// The values of byte k of a word of codes; base = base_of(the block's exponent), whose 255 is the caller's to see.
__device__ __forceinline__ float decode_m(uint32_t w, int k, int base) {
    const uint32_t c = (w >> (8 * k)) & 127, sign = (w << (24 - 8 * k)) & 0x80000000u;
    return c ? __uint_as_float(((c + static_cast<uint32_t>(base)) << 20) | sign) : 0.0f;
}
__device__ __forceinline__ float decode_v(uint32_t w, int k, int base) {
    const uint32_t c = (w >> (8 * k)) & 255;
    return c ? __uint_as_float((c + static_cast<uint32_t>(base)) << 20) : 0.0f;
}
// bits: of the moment; r: the 16 random bits.  Without the low four bits of the moment, which no carry leaves,
// the random bits and the code lie in half-words.
__device__ __forceinline__ uint32_t encode_m(uint32_t bits, int base, uint32_t r) {   // without the sign
    return static_cast<uint32_t>(max(static_cast<int>((((bits >> 4) & 0x7FFFFFFu) + r) >> 16) - base, 0));
}
__device__ __forceinline__ uint32_t encode_v(uint32_t bits, int base, uint32_t r) {
    // At least 1 for what is not 0: the middle of (code, 1, bits), bits being 0 only for 0 and never under a code.
    const int c = static_cast<int>(((bits >> 4) + r) >> 16) - base, b = static_cast<int>(bits);
    return static_cast<uint32_t>(max(min(max(c, 1), b), min(c, 1)));
}
// Four bytes from the low (kByte 0) or high (3) bytes of four words.
template <int kByte> __device__ __forceinline__ uint32_t pack_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    constexpr uint32_t kPair = (uint32_t(kByte) + 4) << 8 | uint32_t(kByte);   // that byte of the 2nd and of the 1st
    const uint32_t lo = __builtin_amdgcn_perm(b, a, 0x0C0C0000u | kPair);
    const uint32_t hi = __builtin_amdgcn_perm(d, c, kPair << 16 | 0x00000C0Cu);
    return lo | hi;
}

// Eight codes at p + e (those at n and past it read as 0 and are not stored).
__device__ __forceinline__ U2 load_codes(const uint8_t* p, int64_t e, int64_t n) {
    if (e + 8 <= n) return load_at<U2a>(p + e);
    U2 q = {0, 0};
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (e + i < n) q[i / 4] |= static_cast<uint32_t>(load_at<uint8_t>(p + e + i)) << (8 * (i & 3));
    return q;
}
__device__ __forceinline__ void store_codes(uint8_t* p, int64_t e, int64_t n, U2 q) {
    if (e + 8 <= n) {
        store_at<U2a>(p + e, q);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (e + i < n) store_at<uint8_t>(p + e + i, static_cast<uint8_t>(q[i / 4] >> (8 * (i & 3))));
    }
}

// The exponents of the block that element e lies in (two bytes; a plain store: its neighbours come from
// other waves).
__device__ __forceinline__ void load_scales(const uint8_t* p, int64_t e, uint32_t* em, uint32_t* ev) {
    typedef uint16_t H __attribute__((aligned(1)));
    const uint32_t h = *(const RHP_GLOBAL H*)(reinterpret_cast<uintptr_t>(p + e / kScaleBlock * 2));
    *em = h & 255;
    *ev = h >> 8;
}
__device__ __forceinline__ void store_scales(uint8_t* p, int64_t e, uint32_t em, uint32_t ev) {
    typedef uint16_t H __attribute__((aligned(1)));
    *(RHP_GLOBAL H*)(reinterpret_cast<uintptr_t>(p + e / kScaleBlock * 2)) = static_cast<uint16_t>(em | ev << 8);
}

// Eight elements' values from their codes; every one of a block that is not finite is NaN.
__device__ __forceinline__ void decode_group(U2 qm, U2 qv, uint32_t em, uint32_t ev, float* m, float* v) {
    const int bm = base_of(em, 16), bv = base_of(ev, 32);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        m[i] = decode_m(qm[i / 4], i & 3, bm);
        v[i] = decode_v(qv[i / 4], i & 3, bv);
    }
    if (em == 255 || ev == 255) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (em == 255) m[i] = __builtin_nanf("");
            if (ev == 255) v[i] = __builtin_nanf("");
        }
    }
}

// Encodes eight elements a lane, 16 lanes a block of 128, with the random bits random(i), and stores them with
// the block's exponents.  Every lane of the wave takes part; a lane past the tensor's end brings zeros.
template <class Random>
__device__ __forceinline__ void encode_group(const float* m, const float* v, Random random, int64_t e0, int64_t n,
                                             uint8_t* qm, uint8_t* qv, uint8_t* scales) {
    uint32_t tm = 0, tv = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        tm = max(tm, __float_as_uint(m[i]) & 0x7FFFFFFFu);
        tv = max(tv, __float_as_uint(v[i]));   // a v with a sign is a NaN (of -0 the callers make 0)
    }
    const uint32_t em = exponent_of(max16(tm)), ev = exponent_of(max16(tv) & 0x7FFFFFFFu);
    const int bm = base_of(em, 16), bv = base_of(ev, 32);
    uint32_t cm[8], cv[8], bits[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t r = random(i);
        bits[i] = __float_as_uint(m[i]);
        cm[i] = encode_m(bits[i], bm, r & 0xFFFFu);
        cv[i] = encode_v(__float_as_uint(v[i]), bv, r >> 16);
    }
    U2 pm, pv;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const uint32_t* c = cm + 4 * k;
        const uint32_t* b = bits + 4 * k;
        // The signs are the top bits of the moments' top bytes.
        pm[k] = pack_bytes<0>(c[0], c[1], c[2], c[3]) | (pack_bytes<3>(b[0], b[1], b[2], b[3]) & 0x80808080u);
        c = cv + 4 * k;
        pv[k] = pack_bytes<0>(c[0], c[1], c[2], c[3]);
    }
    if (em == 255) pm = U2{0, 0};
    if (ev == 255) pv = U2{0, 0};
    if (e0 < n) {
        store_codes(qm, e0, n, pm);
        store_codes(qv, e0, n, pv);
        if ((threadIdx.x & 15) == 0) store_scales(scales, e0, em, ev);
    }
}

// ------------------------------------------------------------------ the step

template <class A> struct Scalars {
    A b1, c1, b2, c2, ibc2s, eps, a, keep;   // c = 1 - b, ibc2s = 1 / sqrt(bc2), a = lr / bc1, keep = 1 - lr wd
};
// A gradient's address and, in the top bits, its dtype code.
struct Grads {
    uint64_t g[kMaxGrads];
};
constexpr int kDtypeShift = 60;

// sqrt(v) and m / d.  In float by the hardware's square root and reciprocal (each within one unit in the last
// place; the update is rounded once more into a weight some hundred times its size).  They may take subnormals
// for zero: a subnormal v has a root under 1.1e-19, and times ibc2s, which is 1000 at the first step of b2 =
// 1 - 1e-6, it is less than half a unit of d beside eps >= 2e-12 ibc2s.  With a smaller eps (kTinyEps) the
// correctly rounded forms run.  Over 4 M
// elements of any size the update is off by 1.02 u (rms; u = 2^-24 of itself) and 4.3 at most, with the correctly
// rounded forms by 0.98 and 3.7.
template <bool kTinyEps> __device__ __forceinline__ float sqrt_of(float x) {
    return kTinyEps ? __builtin_sqrtf(x) : __builtin_amdgcn_sqrtf(x);
}
template <bool kTinyEps> __device__ __forceinline__ double sqrt_of(double x) { return __builtin_sqrt(x); }
template <bool kTinyEps> __device__ __forceinline__ float quotient(float m, float d) {
    return kTinyEps ? m / d : m * __builtin_amdgcn_rcpf(d);
}
template <bool kTinyEps> __device__ __forceinline__ double quotient(double m, double d) { return m / d; }
constexpr double kLeastFastEps = 2e-12;   // times ibc2s
__device__ __forceinline__ float fma_of(float a, float b, float c) { return __builtin_fmaf(a, b, c); }
__device__ __forceinline__ double fma_of(double a, double b, double c) { return a * b + c; }

template <int N, bool kTinyEps, class A, class G>
__device__ __forceinline__ void update(const Scalars<A>& s, A keep, const G* grad_scale, A* p, A* g, A* m, A* v) {
    if (grad_scale) {
        const A gs = static_cast<A>(*grad_scale);
#pragma unroll
        for (int i = 0; i < N; ++i) g[i] *= gs;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
        m[i] = m[i] * s.b1 + g[i] * s.c1;
        v[i] = v[i] * s.b2 + (g[i] * s.c2) * g[i];
        const A d = fma_of(sqrt_of<kTinyEps>(v[i]), s.ibc2s, s.eps);
        p[i] = fma_of(-s.a, quotient<kTinyEps>(m[i], d), p[i] * keep);
    }
}

template <int N, class A> __device__ __forceinline__ void load_grad(uint64_t g, int64_t e, int64_t n, A* v) {
    if (g == 0) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = A(0);
        return;
    }
    const uint64_t at = g & ((uint64_t(1) << kDtypeShift) - 1);
    if constexpr (std::is_same<A, double>::value) {
        load_n<N>(reinterpret_cast<const double*>(at), e, n, v);
    } else {
        if ((g >> kDtypeShift) == RHP_BF16)
            load_n<N>(reinterpret_cast<const bf16*>(at), e, n, v);
        else
            load_n<N>(reinterpret_cast<const float*>(at), e, n, v);
    }
}

// The weight: a master's value where there is one, else the parameter's.
template <int N, class A> __device__ __forceinline__ void load_weight(const PlanTensor& t, int64_t e, A* p) {
    if constexpr (std::is_same<A, double>::value) {
        load_n<N>(static_cast<const double*>(t.p), e, t.n, p);
    } else {
        if (t.master)
            load_n<N>(static_cast<const float*>(t.master), e, t.n, p);
        else if (t.dtype == RHP_BF16)
            load_n<N>(static_cast<const bf16*>(t.p), e, t.n, p);
        else
            load_n<N>(static_cast<const float*>(t.p), e, t.n, p);
    }
}
template <int N, class A> __device__ __forceinline__ void store_weight(const PlanTensor& t, int64_t e, const A* p) {
    if constexpr (std::is_same<A, double>::value) {
        store_n<N>(static_cast<double*>(t.p), e, t.n, p);
    } else {
        if (t.master) store_n<N>(t.master, e, t.n, p);
        if (t.dtype == RHP_BF16)
            store_n<N>(static_cast<bf16*>(t.p), e, t.n, p);
        else
            store_n<N>(static_cast<float*>(t.p), e, t.n, p);
    }
}

// G: the type of *grad_scale, double only for double weights.
template <class A, bool kState8, bool kTinyEps, class G>
__global__ __launch_bounds__(kThreads) void adamw_kernel(const PlanTensor* __restrict__ tensors,
                                                         const uint32_t* __restrict__ of_block, Grads grads,
                                                         uint32_t t0, uint32_t b0, Scalars<A> s,
                                                         const G* __restrict__ grad_scale, uint32_t salt) {
    const uint32_t b = b0 + blockIdx.x;
    const uint32_t ti = of_block[b];
    const PlanTensor t = tensors[ti];
    const uint64_t g = grads.g[ti - t0];
    const A keep = t.decay ? s.keep : A(1);
    const int64_t base = static_cast<int64_t>(b - t.block0) * (kState8 ? kBlock8 : kBlock32);
    if constexpr (kState8) {
        // Groups of eight neighbouring elements, a wave's groups one behind the other: 1024 elements a wave.
        float p[kGroups8][8], gv[kGroups8][8], m[8], v[8];
        U2 qm[kGroups8], qv[kGroups8];
        uint32_t em[kGroups8], ev[kGroups8];
        const int64_t e0 = base + (threadIdx.x >> 6) * (64 * kElems8) + (threadIdx.x & 63) * 8;
        uint8_t *tm = static_cast<uint8_t*>(t.m), *tv = static_cast<uint8_t*>(t.v);
#pragma unroll
        for (int u = 0; u < kGroups8; ++u) {
            const int64_t e = e0 + u * 512;
            qm[u] = load_codes(tm, e, t.n);
            qv[u] = load_codes(tv, e, t.n);
            em[u] = ev[u] = 0;
            if (e < t.n) load_scales(t.scales, e, &em[u], &ev[u]);
            load_weight<8>(t, e, p[u]);
            load_grad<8>(g, e, t.n, gv[u]);
        }
        const uint32_t key = mix(t.key ^ salt);
#pragma unroll
        for (int u = 0; u < kGroups8; ++u) {
            const int64_t e = e0 + u * 512;
            decode_group(qm[u], qv[u], em[u], ev[u], m, v);
            update<8, kTinyEps>(s, keep, grad_scale, p[u], gv[u], m, v);
            store_weight<8>(t, e, p[u]);
            if (e + 8 > t.n) {
                // Elements past the end read as zeros and, but in a block that is not finite, stay zeros.
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (e + i >= t.n) m[i] = v[i] = 0.0f;
            }
            const uint32_t hash = mix(key + static_cast<uint32_t>(e >> 3));
            encode_group(m, v, [&](int i) { return random_of(hash, i); }, e, t.n, tm, tv, t.scales);
        }
    } else {
        const int64_t e0 = base + threadIdx.x * kElems32;
        A p[kElems32], gv[kElems32], m[kElems32], v[kElems32];
        load_n<kElems32>(static_cast<const A*>(t.m), e0, t.n, m);
        load_n<kElems32>(static_cast<const A*>(t.v), e0, t.n, v);
        load_weight<kElems32>(t, e0, p);
        load_grad<kElems32>(g, e0, t.n, gv);
        update<kElems32, kTinyEps>(s, keep, grad_scale, p, gv, m, v);
        store_weight<kElems32>(t, e0, p);
        store_n<kElems32>(static_cast<A*>(t.m), e0, t.n, m);
        store_n<kElems32>(static_cast<A*>(t.v), e0, t.n, v);
    }
}

// The values of codes (bfloat16 holds each exactly), or the codes nearest to given moments (a state's change of
// width).  Bound by HBM: the values of 1.41 G elements (6 bytes each) in 1.39 ms, 6.1 TB/s.
__global__ __launch_bounds__(kThreads) void moments_decode_kernel(const uint8_t* __restrict__ qm,
                                                                  const uint8_t* __restrict__ qv,
                                                                  const uint8_t* __restrict__ scales, int64_t n,
                                                                  bf16* __restrict__ m, bf16* __restrict__ v) {
    const int64_t e0 = (static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x) * 8;
    if (e0 >= n) return;
    float a[8], b[8];
    const U2 wm = load_codes(qm, e0, n), wv = load_codes(qv, e0, n);
    uint32_t em, ev;
    load_scales(scales, e0, &em, &ev);
    decode_group(wm, wv, em, ev, a, b);
    store_n<8>(m, e0, n, a);
    store_n<8>(v, e0, n, b);
}
__global__ __launch_bounds__(kThreads) void moments_encode_kernel(const float* __restrict__ m,
                                                                  const float* __restrict__ v, int64_t n,
                                                                  uint8_t* __restrict__ qm, uint8_t* __restrict__ qv,
                                                                  uint8_t* __restrict__ scales) {
    const int64_t e0 = (static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x) * 8;
    float a[8], b[8];
    load_n<8>(m, e0, n, a);
    load_n<8>(v, e0, n, b);
    // A caller's v, which a step's own cannot be: -0 is 0, and what has no root makes its block NaN as a NaN does.
#pragma unroll
    for (int i = 0; i < 8; ++i) b[i] = b[i] < 0.0f ? __builtin_nanf("") : __builtin_fabsf(b[i]);
    encode_group(a, b, [](int) { return 0x80008000u; }, e0, n, qm, qv, scales);
}

// ------------------------------------------------------------------ the gradients' norm

constexpr int kNormMax = 192;          // tensors a launch
constexpr int kNormBlocks = 2048;      // partial sums a launch
constexpr int kNormChunk = 4096;       // elements

struct NormTensors {
    uint64_t g[kNormMax];              // address and dtype code
    int64_t n[kNormMax];
    uint32_t chunk0[kNormMax + 1];
    int count;
};

template <class S> __device__ __forceinline__ double sum_squares(const S* p, int64_t e0, int64_t e1) {
    constexpr int N = 16 / static_cast<int>(sizeof(S));
    double sum = 0;
    for (int64_t e = e0 + threadIdx.x * N; e < e1; e += kThreads * N) {
        typename Elem<S>::acc v[N];
        load_n<N>(p, e, e1, v);
#pragma unroll
        for (int i = 0; i < N; ++i) sum = __builtin_fma(static_cast<double>(v[i]), static_cast<double>(v[i]), sum);
    }
    return sum;
}

__device__ __forceinline__ double block_sum(double v, double* s) {
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) v += __shfl_xor(v, d, 64);
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
    __syncthreads();
    v = s[0];
    for (int i = 1; i < kThreads / 64; ++i) v += s[i];
    return v;
}

// Partial sums of squares, in double: a bfloat16's square leaves float's range
// and the sum of 10^9 of them its precision.  Block b takes the b-th part of
// the chunks, so its sum does not depend on what runs beside it.  Bound by
// HBM: 1.41 G bfloat16 (2.8 GB) in 0.42 ms, 6.7 TB/s.
__global__ __launch_bounds__(kThreads) void grad_norm_kernel(NormTensors ts, double* __restrict__ part) {
    __shared__ double s[kThreads / 64];
    const uint32_t chunks = ts.chunk0[ts.count];
    uint32_t c = static_cast<uint32_t>(static_cast<uint64_t>(chunks) * blockIdx.x / gridDim.x);
    const uint32_t c1 = static_cast<uint32_t>(static_cast<uint64_t>(chunks) * (blockIdx.x + 1) / gridDim.x);
    double sum = 0;
    int t = 0;
    while (c < c1) {
        while (ts.chunk0[t + 1] <= c) ++t;
        const uint32_t end = min(c1, ts.chunk0[t + 1]);
        const uint64_t g = ts.g[t], at = g & ((uint64_t(1) << kDtypeShift) - 1);
        const int64_t e0 = static_cast<int64_t>(c - ts.chunk0[t]) * kNormChunk;
        const int64_t e1 = min(ts.n[t], static_cast<int64_t>(end - ts.chunk0[t]) * kNormChunk);
        const int dt = static_cast<int>(g >> kDtypeShift);
        if (dt == RHP_BF16)
            sum += sum_squares(reinterpret_cast<const bf16*>(at), e0, e1);
        else if (dt == RHP_F32)
            sum += sum_squares(reinterpret_cast<const float*>(at), e0, e1);
        else
            sum += sum_squares(reinterpret_cast<const double*>(at), e0, e1);
        c = end;
    }
    sum = block_sum(sum, s);
    if (threadIdx.x == 0) part[blockIdx.x] = sum;
}

// One block: the launch and 2048 loads, 4 us.  In a launch of its own, so that no counter has to be zero before a
// call and none is shared between two.  out = [norm, min(1, max_norm / (norm + 1e-6))]; a norm that is NaN makes
// the coefficient NaN.
template <class O>
__global__ __launch_bounds__(kThreads) void grad_norm_finish_kernel(const double* __restrict__ part, int n,
                                                                    double max_norm, O* __restrict__ out) {
    __shared__ double s[kThreads / 64];
    double sum = 0;
    for (int i = threadIdx.x; i < n; i += kThreads) sum += part[i];
    sum = block_sum(sum, s);
    if (threadIdx.x == 0) {
        const double norm = __builtin_sqrt(sum);
        const double c = max_norm / (norm + 1e-6);
        out[0] = static_cast<O>(norm);
        out[1] = static_cast<O>(c >= 1.0 ? 1.0 : c);
    }
}

inline bool float_dtype(int dt) { return dt == RHP_F64 || dt == RHP_F32 || dt == RHP_BF16; }
inline bool element_aligned(const void* p, int dt) {
    return (reinterpret_cast<uintptr_t>(p) & (dtype_bytes(dt) - 1)) == 0;
}
inline uint64_t tag(const void* p, int dt) {
    return reinterpret_cast<uint64_t>(p) | static_cast<uint64_t>(dt) << kDtypeShift;
}

template <class A, bool kState8, bool kTinyEps, class G>
int launch_step(const uint8_t* host, const uint8_t* dev, const void* const* grads, const int* g_dtypes,
                const Scalars<A>& s, const G* grad_scale, uint32_t salt, hipStream_t stream) {
    const PlanHeader& head = *reinterpret_cast<const PlanHeader*>(host);
    const PlanTensor* ts = reinterpret_cast<const PlanTensor*>(host + sizeof(PlanHeader));
    const PlanTensor* tensors = reinterpret_cast<const PlanTensor*>(dev + sizeof(PlanHeader));
    const uint32_t* of_block = reinterpret_cast<const uint32_t*>(tensors + head.count);
    for (uint32_t t0 = 0; t0 < head.count; t0 += kMaxGrads) {
        const uint32_t t1 = std::min(head.count, t0 + kMaxGrads);
        const uint32_t b0 = ts[t0].block0, b1 = t1 < head.count ? ts[t1].block0 : head.blocks;
        if (b1 == b0) continue;
        Grads g{};
        for (uint32_t t = t0; t < t1; ++t)
            if (grads && grads[t]) g.g[t - t0] = tag(grads[t], g_dtypes[t]);
        for (uint32_t b = b0; b < b1; b += kMaxBlocks) {
            hipLaunchKernelGGL((adamw_kernel<A, kState8, kTinyEps, G>), dim3(std::min(b1 - b, kMaxBlocks)),
                               dim3(kThreads), 0, stream, tensors, of_block, g, t0, b, s, grad_scale, salt);
            if (int rc = check_launch("adamw_kernel")) return rc;
        }
    }
    return 0;
}

}  // namespace
}  // namespace rhp

using namespace rhp;

extern "C" size_t rhp_adamw_plan_bytes(int count, const int64_t* numel, int state_bits) {
    if (count < 0 || (count > 0 && !numel) || (state_bits != 32 && state_bits != 8)) return 0;
    uint64_t blocks = 0;
    for (int i = 0; i < count; ++i) {
        if (numel[i] < 0 || numel[i] > (int64_t(1) << 34)) return 0;
        blocks += static_cast<uint64_t>(blocks_of(numel[i], state_bits == 8));
    }
    return plan_bytes(static_cast<uint64_t>(count), blocks);
}

extern "C" int rhp_adamw_plan(int count, void* const* params, const int* dtypes, void* const* masters,
                              void* const* exp_avg, void* const* exp_avg_sq, void* const* scales,
                              const int64_t* numel, const uint32_t* keys, const int* decay, int state_bits,
                              void* image, size_t image_bytes) {
    clear_error();
    RHP_REQUIRE(count >= 0, "rhp_adamw_plan: count must be >= 0");
    RHP_REQUIRE(state_bits == 32 || state_bits == 8, "rhp_adamw_plan: the moments have 32 or 8 bits");
    RHP_REQUIRE(image && (reinterpret_cast<uintptr_t>(image) & 7) == 0, "rhp_adamw_plan: null or unaligned image");
    RHP_REQUIRE(count == 0 || (params && dtypes && exp_avg && exp_avg_sq && numel &&
                               (state_bits == 32 || (scales && keys))),
                "rhp_adamw_plan: null array");
    uint64_t blocks = 0;
    bool any64 = false, other = false;
    // What a step writes: two tensors on the same memory would race.
    std::vector<std::pair<uintptr_t, uintptr_t>> written;
    try {
        written.reserve(5 * static_cast<size_t>(count));
    } catch (const std::exception&) {
        return fail("rhp_adamw_plan: out of host memory");
    }
    const auto writes = [&](const void* p, uint64_t bytes) {
        if (p && bytes) written.emplace_back(reinterpret_cast<uintptr_t>(p), reinterpret_cast<uintptr_t>(p) + bytes);
    };
    for (int i = 0; i < count; ++i) {
        RHP_REQUIRE(numel[i] >= 0 && numel[i] <= (int64_t(1) << 34), "rhp_adamw_plan: element count out of range");
        RHP_REQUIRE(float_dtype(dtypes[i]), std::string("rhp_adamw_plan: unsupported dtype ") + dtype_name(dtypes[i]));
        (dtypes[i] == RHP_F64 ? any64 : other) = true;
        RHP_REQUIRE(!masters || !masters[i] || dtypes[i] == RHP_BF16,
                    "rhp_adamw_plan: masters are for bfloat16 weights");
        blocks += static_cast<uint64_t>(blocks_of(numel[i], state_bits == 8));
        if (numel[i] == 0) continue;
        RHP_REQUIRE(params[i] && exp_avg[i] && exp_avg_sq[i] && (state_bits == 32 || scales[i]),
                    "rhp_adamw_plan: null tensor");
        const int st = dtypes[i] == RHP_F64 ? RHP_F64 : RHP_F32;
        RHP_REQUIRE(element_aligned(params[i], dtypes[i]) &&
                        (state_bits == 8 || (element_aligned(exp_avg[i], st) && element_aligned(exp_avg_sq[i], st))) &&
                        (!masters || element_aligned(masters[i], RHP_F32)),
                    "rhp_adamw_plan: a tensor is not aligned to its elements");
        const uint64_t n = static_cast<uint64_t>(numel[i]);
        const uint64_t moment = n * (state_bits == 8 ? 1 : dtype_bytes(st));
        writes(params[i], n * dtype_bytes(dtypes[i]));
        if (masters) writes(masters[i], n * 4);
        writes(exp_avg[i], moment);
        writes(exp_avg_sq[i], moment);
        if (state_bits == 8) writes(scales[i], (n + kScaleBlock - 1) / kScaleBlock * 2);
    }
    std::sort(written.begin(), written.end());
    for (size_t i = 1; i < written.size(); ++i)
        RHP_REQUIRE(written[i].first >= written[i - 1].second, "rhp_adamw_plan: two tensors share memory");
    RHP_REQUIRE(!(any64 && other), "rhp_adamw_plan: float64 weights need a plan of their own");
    RHP_REQUIRE(!(any64 && state_bits == 8), "rhp_adamw_plan: float64 weights have float64 moments, not 8 bits");
    RHP_REQUIRE(blocks < (uint64_t(1) << 31), "rhp_adamw_plan: too many elements in one plan");
    RHP_REQUIRE(image_bytes >= plan_bytes(static_cast<uint64_t>(count), blocks),
                "rhp_adamw_plan: image smaller than rhp_adamw_plan_bytes()");
    const PlanHeader head{kPlanMagic, static_cast<uint32_t>(count), static_cast<uint32_t>(blocks), state_bits == 8,
                          any64, {}};
    uint8_t* out = static_cast<uint8_t*>(image);
    std::memcpy(out, &head, sizeof head);
    PlanTensor* ts = reinterpret_cast<PlanTensor*>(out + sizeof head);
    uint32_t* of_block = reinterpret_cast<uint32_t*>(ts + count);
    uint32_t b = 0;
    for (int i = 0; i < count; ++i) {
        const PlanTensor t{params[i], masters ? static_cast<float*>(masters[i]) : nullptr, exp_avg[i], exp_avg_sq[i],
                           state_bits == 8 ? static_cast<uint8_t*>(scales[i]) : nullptr, numel[i], keys ? keys[i] : 0u,
                           b, static_cast<uint32_t>(dtypes[i]), static_cast<uint32_t>(!decay || decay[i])};
        std::memcpy(&ts[i], &t, sizeof t);
        for (int64_t k = blocks_of(numel[i], state_bits == 8); k > 0; --k) of_block[b++] = static_cast<uint32_t>(i);
    }
    return 0;
}

// grad_scale64: *grad_scale in double, for float64 weights; one of the two is null.
static int adamw_step(const void* image, const void* dev_image, size_t image_bytes, const void* const* grads,
                      const int* g_dtypes, double lr, double beta1, double beta2, double eps, double weight_decay,
                      int64_t step, const float* grad_scale, const double* grad_scale64, uint64_t seed,
                      hipStream_t stream) {
    RHP_REQUIRE(image && image_bytes >= sizeof(PlanHeader) && (reinterpret_cast<uintptr_t>(image) & 7) == 0,
                "rhp_adamw_step: null, unaligned or short image");
    const uint8_t* host = static_cast<const uint8_t*>(image);
    const PlanHeader& head = *reinterpret_cast<const PlanHeader*>(host);
    RHP_REQUIRE(head.magic == kPlanMagic && image_bytes >= plan_bytes(head.count, head.blocks),
                "rhp_adamw_step: not an image of rhp_adamw_plan");
    RHP_REQUIRE(step >= 1, "rhp_adamw_step: step counts from 1");
    RHP_REQUIRE(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0, "rhp_adamw_step: betas must be in [0, 1)");
    RHP_REQUIRE(lr >= 0.0 && eps >= 0.0 && weight_decay >= 0.0,
                "rhp_adamw_step: lr, eps and weight_decay must not be negative");
    RHP_REQUIRE(!grad_scale64 || head.f64, "rhp_adamw_step64: the plan's weights are not float64");
    if (head.blocks == 0) return 0;
    RHP_REQUIRE(dev_image && aligned16(dev_image), "rhp_adamw_step: null or unaligned device image");
    RHP_REQUIRE(!grads || g_dtypes, "rhp_adamw_step: gradients without their dtypes");
    for (uint32_t i = 0; grads && i < head.count; ++i) {
        if (!grads[i]) continue;
        const int dt = g_dtypes[i];
        RHP_REQUIRE(head.f64 ? dt == RHP_F64 : dt == RHP_F32 || dt == RHP_BF16,
                    std::string("rhp_adamw_step: unsupported gradient dtype ") + dtype_name(dt));
        RHP_REQUIRE(element_aligned(grads[i], dt), "rhp_adamw_step: a gradient is not aligned to its elements");
    }
    const double bc1 = 1.0 - std::pow(beta1, static_cast<double>(step));
    const double ibc2s = 1.0 / std::sqrt(1.0 - std::pow(beta2, static_cast<double>(step)));
    const Scalars<double> d{beta1, 1.0 - beta1, beta2, 1.0 - beta2, ibc2s, eps, lr / bc1, 1.0 - lr * weight_decay};
    const uint64_t count = static_cast<uint64_t>(step);
    const uint32_t salt = mix(mix(mix(static_cast<uint32_t>(count) ^ static_cast<uint32_t>(count >> 32)) ^
                                  static_cast<uint32_t>(seed >> 32)) ^
                              static_cast<uint32_t>(seed));
    const uint8_t* dev = static_cast<const uint8_t*>(dev_image);
    if (grad_scale64)
        return launch_step<double, false, false, double>(host, dev, grads, g_dtypes, d, grad_scale64, salt, stream);
    const auto go = [&](auto launch, const auto& scalars) {
        return launch(host, dev, grads, g_dtypes, scalars, grad_scale, salt, stream);
    };
    if (head.f64) return go(launch_step<double, false, false, float>, d);
    const Scalars<float> f{static_cast<float>(d.b1), static_cast<float>(d.c1), static_cast<float>(d.b2),
                           static_cast<float>(d.c2), static_cast<float>(d.ibc2s), static_cast<float>(d.eps),
                           static_cast<float>(d.a), static_cast<float>(d.keep)};
    if (eps < kLeastFastEps * ibc2s)
        return head.state8 ? go(launch_step<float, true, true, float>, f) : go(launch_step<float, false, true, float>, f);
    return head.state8 ? go(launch_step<float, true, false, float>, f) : go(launch_step<float, false, false, float>, f);
}

extern "C" int rhp_adamw_step(const void* image, const void* dev_image, size_t image_bytes, const void* const* grads,
                              const int* g_dtypes, double lr, double beta1, double beta2, double eps,
                              double weight_decay, int64_t step, const float* grad_scale, uint64_t seed,
                              hipStream_t stream) {
    clear_error();
    return adamw_step(image, dev_image, image_bytes, grads, g_dtypes, lr, beta1, beta2, eps, weight_decay, step,
                      grad_scale, nullptr, seed, stream);
}

extern "C" int rhp_adamw_step64(const void* image, const void* dev_image, size_t image_bytes, const void* const* grads,
                                const int* g_dtypes, double lr, double beta1, double beta2, double eps,
                                double weight_decay, int64_t step, const double* grad_scale, hipStream_t stream) {
    clear_error();
    RHP_REQUIRE(grad_scale, "rhp_adamw_step64: null grad_scale");
    return adamw_step(image, dev_image, image_bytes, grads, g_dtypes, lr, beta1, beta2, eps, weight_decay, step,
                      nullptr, grad_scale, 0, stream);
}

static int check_codes(const char* what, int64_t n, const void* const* ptrs, int count) {
    RHP_REQUIRE(n >= 0 && n <= (int64_t(1) << 34), std::string(what) + ": element count out of range");
    for (int i = 0; i < count; ++i) RHP_REQUIRE(n == 0 || ptrs[i], std::string(what) + ": null pointer");
    return 0;
}

extern "C" int rhp_moments_decode(const uint8_t* q_m, const uint8_t* q_v, const uint8_t* scales, int64_t n, void* m,
                                  void* v, hipStream_t stream) {
    clear_error();
    const void* ptrs[] = {q_m, q_v, scales, m, v};
    if (int rc = check_codes("rhp_moments_decode", n, ptrs, 5)) return rc;
    if (n == 0) return 0;
    RHP_REQUIRE(element_aligned(m, RHP_BF16) && element_aligned(v, RHP_BF16), "rhp_moments_decode: unaligned output");
    hipLaunchKernelGGL(moments_decode_kernel, dim3(static_cast<unsigned>((n + kThreads * 8 - 1) / (kThreads * 8))),
                       dim3(kThreads), 0, stream, q_m, q_v, scales, n, static_cast<bf16*>(m), static_cast<bf16*>(v));
    return check_launch("moments_decode_kernel");
}

extern "C" int rhp_moments_encode(const float* m, const float* v, int64_t n, uint8_t* q_m, uint8_t* q_v,
                                  uint8_t* scales, hipStream_t stream) {
    clear_error();
    const void* ptrs[] = {m, v, q_m, q_v, scales};
    if (int rc = check_codes("rhp_moments_encode", n, ptrs, 5)) return rc;
    if (n == 0) return 0;
    RHP_REQUIRE(element_aligned(m, RHP_F32) && element_aligned(v, RHP_F32), "rhp_moments_encode: unaligned input");
    hipLaunchKernelGGL(moments_encode_kernel, dim3(static_cast<unsigned>((n + kThreads * 8 - 1) / (kThreads * 8))),
                       dim3(kThreads), 0, stream, m, v, n, q_m, q_v, scales);
    return check_launch("moments_encode_kernel");
}

extern "C" size_t rhp_grad_norm_workspace_bytes(int count) {
    if (count < 0) return 0;
    return static_cast<size_t>(std::max(1, (count + kNormMax - 1) / kNormMax)) * kNormBlocks * sizeof(double);
}

template <class O>
static int grad_norm(int count, const void* const* grads, const int* dtypes, const int64_t* numel, double max_norm,
                     O* out, void* workspace, size_t workspace_bytes, hipStream_t stream) {
    RHP_REQUIRE(count >= 0, "rhp_grad_norm: count must be >= 0");
    RHP_REQUIRE(count == 0 || (grads && dtypes && numel), "rhp_grad_norm: null array");
    RHP_REQUIRE(max_norm > 0.0, "rhp_grad_norm: max_norm must be positive");
    RHP_REQUIRE(out && (reinterpret_cast<uintptr_t>(out) & (sizeof(O) - 1)) == 0, "rhp_grad_norm: null or unaligned output");
    RHP_REQUIRE(workspace && aligned16(workspace) && workspace_bytes >= rhp_grad_norm_workspace_bytes(count),
                "rhp_grad_norm: workspace smaller than rhp_grad_norm_workspace_bytes(), null or unaligned");
    for (int i = 0; i < count; ++i) {
        RHP_REQUIRE(numel[i] >= 0 && numel[i] <= (int64_t(1) << 34), "rhp_grad_norm: element count out of range");
        RHP_REQUIRE(float_dtype(dtypes[i]), std::string("rhp_grad_norm: unsupported dtype ") + dtype_name(dtypes[i]));
        RHP_REQUIRE(element_aligned(grads[i], dtypes[i]), "rhp_grad_norm: a gradient is not aligned to its elements");
    }
    double* part = static_cast<double*>(workspace);
    int parts = 0;
    for (int t0 = 0; t0 < count; t0 += kNormMax) {
        NormTensors ts{};
        ts.count = std::min(kNormMax, count - t0);
        uint64_t chunks = 0;
        for (int i = 0; i < ts.count; ++i) {
            ts.g[i] = tag(grads[t0 + i], dtypes[t0 + i]);
            ts.n[i] = grads[t0 + i] ? numel[t0 + i] : 0;
            ts.chunk0[i] = static_cast<uint32_t>(chunks);
            chunks += static_cast<uint64_t>((ts.n[i] + kNormChunk - 1) / kNormChunk);
        }
        ts.chunk0[ts.count] = static_cast<uint32_t>(chunks);
        if (chunks == 0) continue;
        const int nb = static_cast<int>(std::min<uint64_t>(chunks, kNormBlocks));
        hipLaunchKernelGGL(grad_norm_kernel, dim3(nb), dim3(kThreads), 0, stream, ts, part + parts);
        if (int rc = check_launch("grad_norm_kernel")) return rc;
        parts += nb;
    }
    hipLaunchKernelGGL(grad_norm_finish_kernel<O>, dim3(1), dim3(kThreads), 0, stream, part, parts, max_norm, out);
    return check_launch("grad_norm_finish_kernel");
}

extern "C" int rhp_grad_norm(int count, const void* const* grads, const int* dtypes, const int64_t* numel,
                             double max_norm, float* out, void* workspace, size_t workspace_bytes,
                             hipStream_t stream) {
    clear_error();
    return grad_norm(count, grads, dtypes, numel, max_norm, out, workspace, workspace_bytes, stream);
}

extern "C" int rhp_grad_norm64(int count, const void* const* grads, const int* dtypes, const int64_t* numel,
                               double max_norm, double* out, void* workspace, size_t workspace_bytes,
                               hipStream_t stream) {
    clear_error();
    return grad_norm(count, grads, dtypes, numel, max_norm, out, workspace, workspace_bytes, stream);
}
