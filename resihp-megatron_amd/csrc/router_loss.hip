// The router's losses for gfx950: the balance loss with the per-expert counts
// and the z loss, forward and backward.
//
// They stand beside the aux-loss-free bias of resihp/runtime/moe.py:64-66 (the
// reference's way to balance) on the logits of route() (moe.py:75-79).
//
// Of the tokens t of sequence s that count (n_s of them, S' sequences with any, N
// in all), with c_se the pairs of the sequence that chose expert e:
//   p_t     = softmax_e(u_te)    u = logits (softmax scores), log sigmoid(logits)
//                                (sigmoid scores divided by their sum)
//   balance = 1/S' sum_s E / (k n_s^2) sum_e c_se sum_{t in s} p_te
//   z       = 1/N sum_t lse_t^2  lse_t = log sum_e exp(logits_te)
// and with g_b, g_z the gradients of the two:
//   dlogits_te = g_b E / (k n_s^2 S') p_te (c_se - sum_j c_sj p_tj) u'_te
//                + g_z 2 lse_t / N exp(logits_te - lse_t)
//                u' = 1 or sigmoid(-logits)
// (the counts carry no gradient).  A row of logits that are all -inf has no
// probabilities: it adds nothing to the sums and its gradient is zero.
//
// Softmaxes are taken about the row's largest value, in the logits' type; sums
// over tokens are that type within a block and double across blocks, in an
// order that the sizes alone decide.  Bound by latency: the largest batches (32768 x
// 128 float32, 17 MB each way) take microseconds at the memory's rate, so the
// design is about few launches (two forward, one backward) and short chains: a
// row on few lanes with several experts each, whose sums take lane exchanges
// within sixteen lanes (DPP), and a partial row of sums a block, 256 blocks.
// Measured (forward + finish, backward): 16384 tokens of 64 experts, sigmoid scores
// 11 + 7, 12 us; 32768 of 128 8 + 9, 18; 64 tokens 3 + 5, 4 (float64, forward and backward of
// the first two: 25, 21 and 29, 32).  With a row on 64 lanes and 1024 partial rows: 30 + 16,
// 35 and 33 + 22, 50 of the first two.  Many sequences: see router_loss_finish_kernel.

#include <algorithm>
#include <type_traits>

#include "rhp_common.h"

namespace rhp {
namespace {

constexpr int kLossThreads = 1024;   // forward: many tokens a block, so that there are few partial rows
constexpr int kLossBwdThreads = 256;
constexpr int kLossBlocks = 256;     // partial rows: about a block a CU
constexpr int kLossMaxE = 1024;
constexpr int kFinishThreads = 1024;

// exp(x) to about an ulp: the hardware's 2^x on x log2(e), whose rounding error goes in as a correction.
__device__ __forceinline__ float exp_loss(float x) {
    const float t = x * 0x1.715476p+0f;
    float lo = __builtin_fmaf(x, 0x1.715476p+0f, -t);
    lo = __builtin_fmaf(x, 0x1.4ae0cp-26f, lo);
    const float r = __builtin_amdgcn_exp2f(t);
    return r > 0.0f && r < __builtin_inff() ? __builtin_fmaf(r, lo * 0x1.62e43p-1f, r) : r;
}
__device__ __forceinline__ double exp_loss(double x) { return exp(x); }
__device__ __forceinline__ float log_loss(float x) { return logf(x); }
__device__ __forceinline__ double log_loss(double x) { return log(x); }
__device__ __forceinline__ float log1p_loss(float x) { return log1pf(x); }
__device__ __forceinline__ double log1p_loss(double x) { return log1p(x); }

// Sums and maxima over LPT neighbouring lanes, in all of them.
template <int kCtrl> __device__ __forceinline__ float lane_of(float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), kCtrl, 0xf, 0xf, true));
}
template <int LPT, class A, class F> __device__ __forceinline__ A over_lanes(A v, F f) {
    if constexpr (std::is_same<A, float>::value) {
        v = f(v, lane_of<0xB1>(v));                               // quad_perm [1,0,3,2]
        v = f(v, lane_of<0x4E>(v));                               // quad_perm [2,3,0,1]
        v = f(v, lane_of<0x141>(v));                              // row_half_mirror: the other four of eight
        if constexpr (LPT > 8) v = f(v, lane_of<0x140>(v));       // row_mirror: the other eight of sixteen
        if constexpr (LPT > 16) v = f(v, __shfl_xor(v, 16, 64));
        if constexpr (LPT > 32) v = f(v, __shfl_xor(v, 32, 64));
    } else {
#pragma unroll
        for (int d = LPT / 2; d >= 1; d >>= 1) v = f(v, __shfl_xor(v, d, 64));
    }
    return v;
}
template <int LPT, class A> __device__ __forceinline__ A row_sum(A v) {
    return over_lanes<LPT>(v, [](A a, A b) { return a + b; });
}
template <int LPT, class A> __device__ __forceinline__ A row_max(A v) {
    return over_lanes<LPT>(v, [](A a, A b) { return b > a || b != b ? b : a; });   // a NaN stays
}

struct LossArgs {
    const void* logits;       // [T, E]
    const int32_t* topi;      // [T, k]
    const uint8_t* mask;      // [T]: tokens that count, or null (all)
    const int32_t* seqs;      // [S + 1] token offsets, or null (one sequence of all tokens)
    int64_t T;
    int E, k, S, score;
    int chunk;                // tokens a block of the forward
    int blocks;               // of the forward
    bool vec;                 // rows can be read in 16 bytes
};

// Token offsets of sequence s, kept within the tokens.
__device__ __forceinline__ int64_t seq_begin(const LossArgs& a, int s) {
    return a.seqs ? min(max(static_cast<int64_t>(a.seqs[s]), int64_t(0)), a.T) : (s ? a.T : 0);
}
// The first sequence that ends past token t0 (S if none): every thread counts some, the block sums.
__device__ __forceinline__ int first_seq(const LossArgs& a, int64_t t0, int* s_cnt) {
    if (!a.seqs) return a.T <= t0;
    int n = 0;
    for (int i = threadIdx.x; i < a.S; i += blockDim.x) n += seq_begin(a, i + 1) <= t0;
    n = over_lanes<64>(n, [](int x, int y) { return x + y; });
    if ((threadIdx.x & 63) == 0) s_cnt[threadIdx.x >> 6] = n;
    __syncthreads();
    n = 0;
    for (int w = 0; w < static_cast<int>(blockDim.x >> 6); ++w) n += s_cnt[w];
    return n;
}

// A token's row: lane i of LPT lanes holds experts NE i .. + NE - 1.
template <class A, int LPT, int NE> struct LossRow {
    static constexpr int V = NE < 16 / static_cast<int>(sizeof(A)) ? NE : 16 / static_cast<int>(sizeof(A));   // a load's
    typedef A Vec __attribute__((ext_vector_type(V)));
    A x[NE];
    __device__ __forceinline__ void load(const A* logits, int64_t t, int E, int lane, bool live, bool vec) {
        const A* p = logits + t * E + lane * NE;
#pragma unroll
        for (int j = 0; j < NE; ++j) x[j] = -__builtin_huge_val();
        if (!live) return;
        if (vec) {
#pragma unroll
            for (int j = 0; j < NE; j += V)
                if (lane * NE + j < E) {
                    const Vec v = *reinterpret_cast<const Vec*>(p + j);
#pragma unroll
                    for (int i = 0; i < V; ++i) x[j + i] = v[i];
                }
        } else {
#pragma unroll
            for (int j = 0; j < NE; ++j)
                if (lane * NE + j < E) x[j] = p[j];
        }
    }
    static __device__ __forceinline__ void store(A* out, int64_t t, int E, int lane, const A (&d)[NE], bool vec) {
        A* p = out + t * E + lane * NE;
        if (vec) {
#pragma unroll
            for (int j = 0; j < NE; j += V)
                if (lane * NE + j < E) {
                    Vec v;
#pragma unroll
                    for (int i = 0; i < V; ++i) v[i] = d[j + i];
                    *reinterpret_cast<Vec*>(p + j) = v;
                }
        } else {
#pragma unroll
            for (int j = 0; j < NE; ++j)
                if (lane * NE + j < E) p[j] = d[j];
        }
    }
    // exp(v - max) of values v into p, their sum and the largest.
    static __device__ __forceinline__ A softmax(const A (&v)[NE], A (&p)[NE], A* top) {
        A m = v[0];
#pragma unroll
        for (int j = 1; j < NE; ++j) m = v[j] > m || v[j] != v[j] ? v[j] : m;
        m = row_max<LPT>(m);
        *top = m;
        A sum = 0;
#pragma unroll
        for (int j = 0; j < NE; ++j) {
            p[j] = m == -__builtin_huge_val() ? A(0) : exp_loss(v[j] - m);
            sum += p[j];
        }
        return row_sum<LPT>(sum);
    }
    // Probabilities into p (zeros for a row without any), and the log of the sum of exp(logits) (zero there).
    __device__ __forceinline__ void scores(int score, A (&p)[NE], A* lse) const {
        A m;
        A sum = softmax(x, p, &m);
        *lse = m == -__builtin_huge_val() ? A(0) : m + log_loss(sum);
        if (score == RHP_SCORE_SIGMOID) {
            A u[NE];
#pragma unroll
            for (int j = 0; j < NE; ++j) {
                const A t = x[j] < 0 ? x[j] : -x[j];   // -|x|
                u[j] = x[j] == -__builtin_huge_val() ? x[j] : (x[j] < 0 ? x[j] : A(0)) - log1p_loss(exp_loss(t));
            }
            sum = softmax(u, p, &m);
        }
        const A inv = sum > 0 || sum != sum ? A(1) / sum : A(0);
#pragma unroll
        for (int j = 0; j < NE; ++j) p[j] *= inv;
    }
};

// Forward, a block a chunk of tokens: the sums of p and the counts by expert, of
// lse^2 and the tokens that count, for every sequence that the chunk touches, at
// partial row block + sequence (distinct: along the pairs that occur either of
// the two grows).  part: [blocks + S][E + 1] (the last lse^2), npart: the same
// in int32 (the last the tokens).
template <class A, int LPT, int NE>
__global__ __launch_bounds__(kLossThreads) void router_loss_fwd_kernel(LossArgs a, A* __restrict__ part,
                                                                       int32_t* __restrict__ npart) {
    constexpr int G = kLossThreads / LPT, kWaves = kLossThreads / 64;   // tokens side by side
    constexpr int kE = LPT * NE;
    __shared__ A s_p[kWaves][kE], s_z[kWaves];
    __shared__ int32_t s_n[kE + 1];
    __shared__ int s_cnt[kWaves];
    const A* logits = static_cast<const A*>(a.logits);
    const int lane = threadIdx.x % LPT, grp = threadIdx.x / LPT, wave = threadIdx.x >> 6;
    const int64_t t0 = static_cast<int64_t>(blockIdx.x) * a.chunk, t1 = min(a.T, t0 + a.chunk);
    int s = first_seq(a, t0, s_cnt);
    int64_t at = max(t0, s < a.S ? seq_begin(a, s) : a.T);
    for (; s < a.S && at < t1; ++s) {
        const int64_t first = seq_begin(a, s), begin = max(at, first), end = min(t1, seq_begin(a, s + 1));
        if (first >= t1) break;
        if (begin >= end) continue;
        at = end;
        for (int i = threadIdx.x; i <= kE; i += kLossThreads) s_n[i] = 0;
        __syncthreads();
        for (int64_t i = begin * a.k + threadIdx.x; i < end * a.k; i += kLossThreads) {
            const int e = a.topi[i];
            if (e >= 0 && e < a.E && (!a.mask || a.mask[i / a.k])) atomicAdd(&s_n[e], 1);
        }
        A acc[NE] = {}, z = 0;
        int n = 0;
        LossRow<A, LPT, NE> row;
        for (int64_t t = begin + grp; t < begin + (end - begin + G - 1) / G * G; t += G) {
            const bool live = t < end && (!a.mask || a.mask[t]);
            row.load(logits, t, a.E, lane, live, a.vec);
            A p[NE], lse;
            row.scores(a.score, p, &lse);
            if (live) {
#pragma unroll
                for (int j = 0; j < NE; ++j) acc[j] += p[j];
                z += lse * lse;
                ++n;
            }
        }
        // The wave's tokens, then the waves'.
#pragma unroll
        for (int d = LPT; d < 64; d <<= 1) {
#pragma unroll
            for (int j = 0; j < NE; ++j) acc[j] += __shfl_xor(acc[j], d, 64);
            z += __shfl_xor(z, d, 64);
            n += __shfl_xor(n, d, 64);
        }
        if ((threadIdx.x & 63) < LPT) {
#pragma unroll
            for (int j = 0; j < NE; ++j) s_p[wave][lane * NE + j] = acc[j];
        }
        if ((threadIdx.x & 63) == 0) {
            s_z[wave] = z;
            if (n) atomicAdd(&s_n[kE], n);
        }
        __syncthreads();
        const int64_t out = (static_cast<int64_t>(blockIdx.x) + s) * (a.E + 1);
        for (int e = threadIdx.x; e <= a.E; e += kLossThreads) {
            A sum = 0;
#pragma unroll
            for (int w = 0; w < kWaves; ++w) sum += e < a.E ? s_p[w][e] : s_z[w];
            part[out + e] = sum;
            npart[out + e] = s_n[e < a.E ? e : kE];
        }
        __syncthreads();
    }
}

// The partial rows' sums: counts [S, E], the tokens of each sequence, and the
// losses.  One block: a wave a sequence and 64 experts, or, where those are
// few, several waves that share its partial rows.  The rows come from other
// XCDs' caches, some 2 us a load that waits for the one before, so 16 rows
// are on their way at a time (one after the other, four at a time: 21 us of 256 rows).
// A turn takes 16 sequences of up to 64 experts, some 2.7 us, whatever the number of tokens: 32768
// tokens of 128 experts in 64 sequences 35 us of both launches, in 256 97, in 1024 355, in 16384 5470.
template <class A>
__global__ __launch_bounds__(kFinishThreads) void router_loss_finish_kernel(LossArgs a, const A* __restrict__ part,
                                                                            const int32_t* __restrict__ npart,
                                                                            A* __restrict__ balance_out,
                                                                            A* __restrict__ z_out,
                                                                            int32_t* __restrict__ counts,
                                                                            int32_t* __restrict__ tokens) {
    constexpr int kWaves = kFinishThreads / 64, kBatch = 16;
    __shared__ double s_p[kWaves][64], s_z[kWaves], s_b[kWaves];
    __shared__ int s_c[kWaves][64], s_n[kWaves], s_full[kWaves], s_total[kWaves];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int per = (a.E + 63) / 64, width = a.E + 1;
    const int64_t tasks = static_cast<int64_t>(a.S) * per;
    const int share = static_cast<int>(max(int64_t(1), min(int64_t(kWaves), kWaves / tasks)));
    const int teams = kWaves / share, team = wave / share, member = wave % share;
    double balance = 0.0, z = 0.0;
    int full = 0, total = 0;
    const int64_t turns = (tasks + teams - 1) / teams;
    for (int64_t turn = 0; turn < turns; ++turn) {
        const int64_t task = turn * teams + team;
        const bool has = team < teams && task < tasks;
        const int s = has ? static_cast<int>(task / per) : 0, chunk = has ? static_cast<int>(task % per) : 0;
        const int e = chunk * 64 + lane;
        double p = 0.0, zs = 0.0;
        int c = 0, n = 0;
        if (has) {
            const int64_t b = seq_begin(a, s), end = seq_begin(a, s + 1);
            const int r0 = b < end ? static_cast<int>(static_cast<uint32_t>(b) / static_cast<uint32_t>(a.chunk)) + s : 0;
            const int r1 = b < end ? static_cast<int>(static_cast<uint32_t>(end - 1) / static_cast<uint32_t>(a.chunk)) + s + 1 : 0;
            for (int r = r0 + member * 64 + lane; r < r1; r += share * 64) {
                n += npart[static_cast<int64_t>(r) * width + a.E];
                zs += static_cast<double>(part[static_cast<int64_t>(r) * width + a.E]);
            }
            for (int r = r0 + member; r < r1; r += kBatch * share) {
                A pv[kBatch];
                int cv[kBatch];
#pragma unroll
                for (int i = 0; i < kBatch; ++i) {
                    const int at = r + i * share;
                    pv[i] = 0;
                    cv[i] = 0;
                    if (at < r1 && e < a.E) {
                        pv[i] = part[static_cast<int64_t>(at) * width + e];
                        cv[i] = npart[static_cast<int64_t>(at) * width + e];
                    }
                }
#pragma unroll
                for (int i = 0; i < kBatch; ++i) {
                    p += static_cast<double>(pv[i]);
                    c += cv[i];
                }
            }
            n = over_lanes<64>(n, [](int x, int y) { return x + y; });
            zs = row_sum<64>(zs);
        }
        if (share > 1) {
            s_p[wave][lane] = p;
            s_c[wave][lane] = c;
            if (lane == 0) {
                s_n[wave] = n;
                s_z[wave] = zs;
            }
            __syncthreads();
            if (member == 0)
                for (int m = 1; m < share; ++m) {
                    p += s_p[wave + m][lane];
                    c += s_c[wave + m][lane];
                    n += s_n[wave + m];
                    zs += s_z[wave + m];
                }
            __syncthreads();
        }
        if (!has || member != 0) continue;
        if (e < a.E) counts[static_cast<int64_t>(s) * a.E + e] = c;
        if (n > 0) balance += static_cast<double>(c) * p / (static_cast<double>(n) * n);
        if (chunk == 0) {
            z += zs;
            full += n > 0;
            total += n;
            if (lane == 0) tokens[s] = n;
        }
    }
    balance = row_sum<64>(balance);
    if (lane == 0) {
        s_b[wave] = balance;
        s_z[wave] = z;
        s_full[wave] = full;
        s_total[wave] = total;
    }
    __syncthreads();
    if (threadIdx.x != 0) return;
    for (int w = 1; w < kWaves; ++w) {
        balance += s_b[w];
        z += s_z[w];
        full += s_full[w];
        total += s_total[w];
    }
    *balance_out = static_cast<A>(full ? balance * a.E / (static_cast<double>(a.k) * full) : 0.0);
    *z_out = static_cast<A>(total ? z / static_cast<double>(total) : 0.0);
    tokens[a.S] = full;
    tokens[a.S + 1] = total;
}

// Backward, a block some tokens: the rows again, with the counts of their sequence in registers.
template <class A, int LPT, int NE>
__global__ __launch_bounds__(kLossBwdThreads) void router_loss_bwd_kernel(LossArgs a, int chunk,
                                                                          const A* __restrict__ d_balance,
                                                                          const A* __restrict__ d_z,
                                                                          const int32_t* __restrict__ counts,
                                                                          const int32_t* __restrict__ tokens,
                                                                          A* __restrict__ dlogits) {
    constexpr int G = kLossBwdThreads / LPT;
    __shared__ int s_cnt[kLossBwdThreads / 64];
    const A* logits = static_cast<const A*>(a.logits);
    const int lane = threadIdx.x % LPT, grp = threadIdx.x / LPT;
    const int64_t t0 = static_cast<int64_t>(blockIdx.x) * chunk, t1 = min(a.T, t0 + chunk);
    const A gb = d_balance ? *d_balance : A(0);
    const int full = tokens[a.S], total = tokens[a.S + 1];
    const A gz = d_z && total ? *d_z * A(2) / static_cast<A>(total) : A(0);
    int s = first_seq(a, t0, s_cnt);
    int64_t at = t0;
    // Runs of a sequence, and what lies before, between and behind the sequences (s = S): zeros.
    while (at < t1) {
        const int64_t begin = s < a.S ? seq_begin(a, s) : a.T;
        const int64_t end = at < begin ? min(t1, begin) : s < a.S ? min(t1, seq_begin(a, s + 1)) : t1;
        const bool inside = at >= begin && s < a.S;
        if (inside && end <= at) {
            ++s;
            continue;
        }
        A c[NE], scale = 0;
        if (inside) {
            const A n = static_cast<A>(tokens[s]);
            if (n > 0) scale = gb * (static_cast<A>(a.E) / (static_cast<A>(a.k) * n)) / (n * static_cast<A>(full));
#pragma unroll
            for (int j = 0; j < NE; ++j) {
                const int e = lane * NE + j;
                c[j] = e < a.E ? static_cast<A>(counts[static_cast<int64_t>(s) * a.E + e]) : A(0);
            }
        }
        LossRow<A, LPT, NE> row;
        for (int64_t t = at + grp; t < at + (end - at + G - 1) / G * G; t += G) {
            const bool live = inside && t < end && (!a.mask || a.mask[t]);
            A d[NE] = {};
            if (inside) {
                row.load(logits, t, a.E, lane, live, a.vec);
                A p[NE], lse, mean = 0;
                row.scores(a.score, p, &lse);
#pragma unroll
                for (int j = 0; j < NE; ++j) mean += c[j] * p[j];
                mean = row_sum<LPT>(mean);
#pragma unroll
                for (int j = 0; j < NE; ++j) {
                    const A x = row.x[j];
                    A v = scale * p[j] * (c[j] - mean);
                    if (a.score == RHP_SCORE_SIGMOID) v /= A(1) + exp_loss(x);
                    const A q = x == -__builtin_huge_val() ? A(0) : exp_loss(x - lse);
                    d[j] = live ? v + gz * lse * q : A(0);
                }
            }
            if (t < end) LossRow<A, LPT, NE>::store(dlogits, t, a.E, lane, d, a.vec);
        }
        at = end;
    }
}

// f(lanes a token, experts a lane): 8 or 16 lanes up to 128 experts, so that a row's sums stay within sixteen lanes.
template <class F> int with_loss_shape(int E, F f) {
    using std::integral_constant;
    if (E <= 8) return f(integral_constant<int, 8>(), integral_constant<int, 1>());
    if (E <= 16) return f(integral_constant<int, 16>(), integral_constant<int, 1>());
    if (E <= 32) return f(integral_constant<int, 16>(), integral_constant<int, 2>());
    if (E <= 64) return f(integral_constant<int, 16>(), integral_constant<int, 4>());
    if (E <= 128) return f(integral_constant<int, 16>(), integral_constant<int, 8>());
    if (E <= 256) return f(integral_constant<int, 32>(), integral_constant<int, 8>());
    return f(integral_constant<int, 64>(), integral_constant<int, 16>());
}

int loss_chunk(int64_t T) {
    const int64_t c = (T + kLossBlocks - 1) / kLossBlocks;
    return static_cast<int>(std::max<int64_t>(64, (c + 63) / 64 * 64));
}

int loss_args(const char* what, const void* logits, int dtype, const int32_t* topi, const uint8_t* mask,
              const int32_t* seqs, int64_t T, int E, int k, int S, int score, LossArgs* a) {
    const std::string f(what);
    RHP_REQUIRE(dtype == RHP_F32 || dtype == RHP_F64, f + ": logits must be float32 or float64");
    RHP_REQUIRE(T >= 0 && T < (int64_t(1) << 31) && E >= 1 && E <= kLossMaxE && k >= 1 && k <= kMaxTopK,
                f + ": need T >= 0, 1 <= E <= 1024 and 1 <= k <= 16");
    RHP_REQUIRE(score == RHP_SCORE_SOFTMAX || score == RHP_SCORE_SIGMOID, f + ": unknown score function");
    RHP_REQUIRE(S >= 1 && S <= (1 << 20) && (seqs || S == 1), f + ": 1 to 2^20 sequences, one without offsets");
    RHP_REQUIRE(T == 0 || (logits && topi), f + ": null pointer");
    RHP_REQUIRE(reinterpret_cast<uintptr_t>(logits) % dtype_bytes(dtype) == 0, f + ": unaligned logits");
    const int chunk = loss_chunk(T);
    // 16 bytes at a time where every row starts at a multiple of what a lane loads at once.
    const bool vec = E % 4 == 0 && aligned16(logits);
    *a = LossArgs{logits, topi, mask, seqs, T, E, k, S, score, chunk, static_cast<int>((T + chunk - 1) / chunk), vec};
    return 0;
}

template <class A>
int loss_fwd(const LossArgs& a, void* balance, void* z, int32_t* counts, int32_t* tokens, void* ws, hipStream_t stream) {
    A* part = static_cast<A*>(ws);
    int32_t* npart = reinterpret_cast<int32_t*>(part + (static_cast<int64_t>(a.blocks) + a.S) * (a.E + 1));
    if (a.blocks) {
        const int rc = with_loss_shape(a.E, [&](auto lanes, auto ne) {
            hipLaunchKernelGGL((router_loss_fwd_kernel<A, decltype(lanes)::value, decltype(ne)::value>), dim3(a.blocks),
                               dim3(kLossThreads), 0, stream, a, part, npart);
            return check_launch("router_loss_fwd_kernel");
        });
        if (rc) return rc;
    }
    hipLaunchKernelGGL(router_loss_finish_kernel<A>, dim3(1), dim3(kFinishThreads), 0, stream, a, part, npart,
                       static_cast<A*>(balance), static_cast<A*>(z), counts, tokens);
    return check_launch("router_loss_finish_kernel");
}

template <class A>
int loss_bwd(const LossArgs& a, const void* d_balance, const void* d_z, const int32_t* counts, const int32_t* tokens,
             void* dlogits, hipStream_t stream) {
    return with_loss_shape(a.E, [&](auto lanes, auto ne) {
        // A turn or more of the block's tokens, some eight blocks a CU.
        constexpr int G = kLossBwdThreads / decltype(lanes)::value;
        const int chunk = static_cast<int>(std::max<int64_t>(1, (a.T + 2048 * G - 1) / (2048 * G))) * G;
        hipLaunchKernelGGL((router_loss_bwd_kernel<A, decltype(lanes)::value, decltype(ne)::value>),
                           dim3(static_cast<unsigned>((a.T + chunk - 1) / chunk)), dim3(kLossBwdThreads), 0, stream, a,
                           chunk, static_cast<const A*>(d_balance),
                           static_cast<const A*>(d_z), counts, tokens, static_cast<A*>(dlogits));
        return check_launch("router_loss_bwd_kernel");
    });
}

}  // namespace
}  // namespace rhp

using namespace rhp;

extern "C" size_t rhp_router_loss_workspace_bytes(int64_t T, int E, int S, int dtype) {
    if (T < 0 || E < 1 || S < 1) return 0;
    const int chunk = loss_chunk(T);
    return static_cast<size_t>((T + chunk - 1) / chunk + S) * (E + 1) * (dtype_bytes(dtype) + 4);
}

extern "C" int rhp_router_loss(const void* logits, int dtype, const int32_t* topi, const uint8_t* mask,
                               const int32_t* seq_offsets, int64_t T, int E, int k, int S, int score, void* balance,
                               void* z, int32_t* counts, int32_t* tokens, void* workspace, size_t workspace_bytes,
                               hipStream_t stream) {
    clear_error();
    LossArgs a;
    if (int rc = loss_args("rhp_router_loss", logits, dtype, topi, mask, seq_offsets, T, E, k, S, score, &a)) return rc;
    RHP_REQUIRE(balance && z && counts && tokens, "rhp_router_loss: null pointer");
    RHP_REQUIRE(workspace && aligned16(workspace) &&
                    workspace_bytes >= rhp_router_loss_workspace_bytes(T, E, S, dtype),
                "rhp_router_loss: workspace smaller than rhp_router_loss_workspace_bytes(), null or unaligned");
    return dtype == RHP_F64 ? loss_fwd<double>(a, balance, z, counts, tokens, workspace, stream)
                            : loss_fwd<float>(a, balance, z, counts, tokens, workspace, stream);
}

extern "C" int rhp_router_loss_bwd(const void* d_balance, const void* d_z, const void* logits, int dtype,
                                   const int32_t* topi, const uint8_t* mask, const int32_t* seq_offsets, int64_t T,
                                   int E, int k, int S, int score, const int32_t* counts, const int32_t* tokens,
                                   void* dlogits, hipStream_t stream) {
    clear_error();
    LossArgs a;
    if (int rc = loss_args("rhp_router_loss_bwd", logits, dtype, topi, mask, seq_offsets, T, E, k, S, score, &a)) return rc;
    if (T == 0) return 0;
    RHP_REQUIRE(counts && tokens && dlogits && dlogits != logits, "rhp_router_loss_bwd: null pointer, or dlogits is logits");
    a.vec = a.vec && aligned16(dlogits);
    return dtype == RHP_F64 ? loss_bwd<double>(a, d_balance, d_z, counts, tokens, dlogits, stream)
                            : loss_bwd<float>(a, d_balance, d_z, counts, tokens, dlogits, stream);
}
