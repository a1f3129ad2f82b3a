// swarm_policyloss.hip — log-probabilities and the clipped policy loss with a KL term, from logits
// (include/swarmseq.h: swarm_log_probs, swarm_policy_loss_*).
//
// Per row of K logits z with the taken action a, m = max z, x_k = z_k - m, e_k = exp x_k, s = sum e_k,
// t = sum e_k x_k:
//   log p_k = x_k - log s,  p_k = e_k / s,  l = log p_a,  H = log s - t / s
//   dz_k = c [ g (1[k = a] - p_k) + entropy_coef p_k (log p_k + H) ],   c = incoming gradient / denominator,
//   g = d pg / d l + kl_coef (1 - exp(ref - l)).
// x is held above -138, where e is 0 in float32: a logit of -inf adds nothing to either sum and has no gradient. A
// NaN or an infinite maximum would be lost there, so such a row's s is set to NaN.
//
// Memory bound. A row is read once and held in registers by as many threads as it needs; maximum, then both sums,
// are reduced over them. Since the denominator does not depend on the logits, the gradient for an incoming gradient
// of 1 follows at once, from the same registers: reading the logits once and writing their gradient is all the
// traffic there is. The backward call keeps that gradient if the incoming one is 1, and otherwise forms it again
// (scaling a rounded gradient would round it twice). Rows that no workgroup holds are read twice. In float32, rows of
// 8193 to 32768 logits leave 172 bytes a thread to scratch memory, which four waves a SIMD cost.
//
// Measured (a 4 GiB copy reaches 4.8 TB/s of reads and writes together on this card):
// A tenth of the rows is masked in each loss.
//   loss, 4096 x 50001, bf16: 214 to 225 us, 3.5 TB/s. Some 115 us of that is arithmetic (two exponentials
//     an element), and of rows of 100 KB a CU's registers and LDS hold two: too few for one row's loads to hide the
//     other's arithmetic altogether. Rows read twice took 290 us, three rows a CU of 256 threads each 247 us.
//   loss, 100000 x 1000, bf16: 96 us, 4.0 TB/s;  20000 x 5000, bf16: 96 us, 4.0;  10000 x 15000, bf16: 128 us, 4.4;
//     10000 x 12000, float32: 210 us, 4.3 TB/s
//   the backward call that forms the gradient again (any incoming one but 1), after its forward call: 4096 x 50001, bf16
//     183 us after 225, float32 384 after 468; 100000 x 1000, bf16 75 after 96; float16, whose forward call forms none,
//     4096 x 50001 163 after 156, 2048 x 6 3.7 after 4.9
//   loss, 2048 x 6, float32: 6.6 + 3.2 us, launches and the last sum
//   log-probabilities, 8192 x 32768, bf16: 99 us, 5.4 TB/s;  81920 x 18, float32: 3.8 us
#include <type_traits>

#include "swarm_seq.h"

using namespace swarm_seq;

namespace {

constexpr int kMaxBlocks = 2048;      // SWARM_POLICY_LOSS_PARTIALS = kSums for each
constexpr int kSums = 6;              // pg, kl, H, outside, pg + kl_coef kl - entropy_coef H, active rows
constexpr int kFinish = 256;          // threads of the last sums
constexpr float kBound = 20.0f;       // bound of the log-ratios
constexpr float kInactive = -1.0f;    // s of a row that takes no part (s >= 1 elsewhere: e = 1 at the maximum)
// Up to this many workgroups, each counts the active rows itself, which spares a launch of 2 us and more. It pays while
// the rows are few, of any length (loss_rows_kernel, us, against a count of its own: 2048 x 6 6.5 / 5.7, 240 x 5000 bf16
// 9.5 / 8.2), and not for many short ones (16384 x 6 13.6 / 5.8, 65536 x 6 36.9 / 6.5).
constexpr unsigned kCountHere = 256;

__device__ __forceinline__ float exponent(float z, float m) { return fmaxf(z - m, -138.0f); }

// e of an exponent, of T's logits: good to 3 + |x| / 20 units of 2^-24 in float32, else to 2 + |x|. (float32 with and
// without the remainder: loss of 5000 x 30000 269 against 264 us, 20000 x 5000 187 against 182. For 16 bits, whose logits'
// own steps are far larger, it would cost 103 against 94 us at 100000 x 1000.)
template <typename T>
__device__ __forceinline__ float exp_of(float x) {
    const float h = x * kLog2e;
    return kExact<T> ? exp_from(h, __builtin_fmaf(h, -kLn2, x)) : __builtin_amdgcn_exp2f(h);
}

// clamp that keeps a NaN
__device__ __forceinline__ float clamp_nan(float x, float lo, float hi) { return x < lo ? lo : (x > hi ? hi : x); }

// Reductions over a row's GROUP threads, in every one.
template <int GROUP>
__device__ __forceinline__ float group_max(float v, float* red) {
    v = lanes_reduce<(GROUP < 64 ? GROUP : 64)>(v, Maximum{});
    if constexpr (GROUP > 64) {
        __syncthreads();
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
        __syncthreads();
        v = red[0];
#pragma unroll
        for (int k = 1; k < GROUP / 64; ++k) v = Maximum{}(v, red[k]);
    }
    return v;
}

template <int GROUP>
__device__ __forceinline__ void group_sums(float& s, float& t, float* red) {
    s = lanes_reduce<(GROUP < 64 ? GROUP : 64)>(s, Add{});
    t = lanes_reduce<(GROUP < 64 ? GROUP : 64)>(t, Add{});
    if constexpr (GROUP > 64) {
        constexpr int W = GROUP / 64;
        __syncthreads();
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s, red[W + (threadIdx.x >> 6)] = t;
        __syncthreads();
        s = t = 0.0f;
#pragma unroll
        for (int k = 0; k < W; ++k) s += red[k], t += red[W + k];
    }
}

// A row of at most N logits, in one lane.
template <typename E, int N>
struct Single {
    using T = E;
    static constexpr int kGroup = 1, kThreads = 256;
    float z[N];
    static size_t lds_bytes(int64_t) { return 0; }

    __device__ __forceinline__ void load(const T* p, int, int64_t K) {
#pragma unroll
        for (int k = 0; k < N; ++k) z[k] = (float)p[k < (int)K ? k : (int)K - 1];
#pragma unroll
        for (int k = 0; k < N; ++k) z[k] = k < (int)K ? z[k] : -INFINITY;
    }
    // f of all values, a few at a time
    template <typename F>
    __device__ __forceinline__ void each(int, F&& f) const {
        f(z);
    }
    // out[k] = f(z_k)
    template <typename F>
    __device__ __forceinline__ void write(T* out, int, int64_t K, F&& f) const {
#pragma unroll
        for (int k = 0; k < N; ++k)
            if (k < (int)K) out[k] = (T)f(z[k]);
    }
    // the thread that stores an element
    static __device__ __forceinline__ int owner(int64_t) { return 0; }
};

// Pack i of a thread of a long row: its first column, and how many of its elements belong to the pack before (the
// last pack is moved left to end with the row).
template <int V>
__device__ __forceinline__ void place(int64_t pack, int64_t K, int64_t& start, int& skip) {
    const int64_t want = pack * V;
    start = want < K - V ? want : K - V;
    skip = want - start < V ? (int)(want - start) : V;
}

// Stores f of a pack's own elements.
template <typename T, int V, typename F>
__device__ __forceinline__ void write_pack(T* out, const Pack<T>& x, int skip, F&& f) {
    float v[V];
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = f(x.get(j));
    Pack<T> w;
    w.set(v);
    if (skip == 0) {
        w.store(out);
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j)
            if (j >= skip) out[j] = (T)w.get(j);
    }
}

// A longer row: EPT logits of each of GROUP threads in registers, in packs of 16 bytes at any alignment, and up to
// EXTRA more packs of each in LDS, where only their own thread reads them.
template <typename E, int GROUP, int EPT, int EXTRA = 0>
struct Wide {
    using T = E;
    static constexpr int kGroup = GROUP, kThreads = GROUP <= 64 ? 256 : GROUP;
    static constexpr int V = 16 / sizeof(T), NP = EPT / V;
    static constexpr int64_t kMost = (int64_t)GROUP * V * (NP + EXTRA);
    Pack<T> x[NP];
    int used;      // packs of a thread that any thread needs

    static size_t lds_bytes(int64_t K) {
        const int64_t packs = (K + GROUP * V - 1) / (GROUP * V);
        return EXTRA > 0 && packs > NP ? (size_t)(packs - NP) * GROUP * 16 : 0;
    }
    static __device__ __forceinline__ Pack<T>* extra(int i, int lane) {
        extern __shared__ __align__(16) uint32_t row_lds[];
        return reinterpret_cast<Pack<T>*>(row_lds) + (i - NP) * GROUP + lane;
    }

    // Pack i's first column, in 32 bits: one register an address, next to the row's uniform base.
    static __device__ __forceinline__ uint32_t column(int i, int lane, int64_t K) {
        const uint32_t want = (uint32_t)(i * GROUP + lane) * V, last = (uint32_t)K - V;
        return want < last ? want : last;
    }
    // What a thread leaves out of its last pack: only packs of the last turn can reach behind the row.
    __device__ __forceinline__ int skipped(int lane, int64_t K) const {
        const uint32_t want = (uint32_t)((used - 1) * GROUP + lane) * V, start = column(used - 1, lane, K);
        return want - start < (uint32_t)V ? (int)(want - start) : V;
    }

    __device__ __forceinline__ Pack<T> fetch(const T* p, int i, int lane, int64_t K, int skip) const {
        Pack<T> x;
        x.load(p + column(i, lane, K));
        if (i == used - 1) {
            float v[V];
#pragma unroll
            for (int j = 0; j < V; ++j) v[j] = j < skip ? -INFINITY : x.get(j);
            x.set(v);
        }
        return x;
    }

    __device__ __forceinline__ void load(const T* p, int lane, int64_t K) {
        used = (int)((K + GROUP * V - 1) / (GROUP * V));
        const int skip = skipped(lane, K);
#pragma unroll
        for (int i = 0; i < NP; ++i)
            if (i < used) x[i] = fetch(p, i, lane, K, skip);
        if constexpr (EXTRA > 0) {
            Pack<T> y[EXTRA];
#pragma unroll
            for (int i = NP; i < NP + EXTRA; ++i)
                if (i < used) y[i - NP] = fetch(p, i, lane, K, skip);
#pragma unroll
            for (int i = NP; i < NP + EXTRA; ++i)
                if (i < used) *extra(i, lane) = y[i - NP];
        }
    }
    template <typename F>
    __device__ __forceinline__ void each(int lane, F&& f) const {
#pragma unroll
        for (int i = 0; i < NP + EXTRA; ++i) {
            if (i >= used) continue;
            float v[V];
            const Pack<T> y = i < NP ? x[i < NP ? i : 0] : *extra(i, lane);
#pragma unroll
            for (int j = 0; j < V; ++j) v[j] = y.get(j);
            f(v);
        }
    }
    template <typename F>
    __device__ __forceinline__ void write(T* out, int lane, int64_t K, F&& f) const {
        const int skip = skipped(lane, K);
#pragma unroll
        for (int i = 0; i < NP + EXTRA; ++i) {
            if (i >= used) continue;
            const Pack<T> y = i < NP ? x[i < NP ? i : 0] : *extra(i, lane);
            T* to = out + column(i, lane, K);
            if (i < used - 1) write_pack<T, V>(to, y, 0, f);
            else if (skip < V) write_pack<T, V>(to, y, skip, f);
        }
    }
    static __device__ __forceinline__ int owner(int64_t a) { return (int)(a / V % GROUP); }
};

// A row that is not held: read for every use.
template <typename E, int GROUP>
struct Streamed {
    using T = E;
    static constexpr int kGroup = GROUP, kThreads = GROUP <= 64 ? 256 : GROUP;
    static constexpr int V = 16 / sizeof(T);
    const T* row;
    int64_t K;
    int lane;
    static size_t lds_bytes(int64_t) { return 0; }

    __device__ __forceinline__ void load(const T* p, int l, int64_t k) { row = p, lane = l, K = k; }
    template <typename F>
    __device__ __forceinline__ void each(int, F&& f) const {
#pragma unroll 2
        for (int64_t pack = lane; pack * V < K; pack += kGroup) {
            int64_t start;
            int skip;
            place<V>(pack, K, start, skip);
            Pack<T> x;
            x.load(row + start);
            float v[V];
#pragma unroll
            for (int j = 0; j < V; ++j) v[j] = j >= skip ? x.get(j) : -INFINITY;
            f(v);
        }
    }
    template <typename F>
    __device__ __forceinline__ void write(T* out, int, int64_t, F&& f) const {
#pragma unroll 2
        for (int64_t pack = lane; pack * V < K; pack += kGroup) {
            int64_t start;
            int skip;
            place<V>(pack, K, start, skip);
            Pack<T> x;
            x.load(row + start);
            write_pack<T, V>(out + start, x, skip, f);
        }
    }
    static __device__ __forceinline__ int owner(int64_t a) { return (int)(a / V % GROUP); }
};

// The row that a thread begins with; uniform where a workgroup has one row.
template <typename R>
__device__ __forceinline__ int64_t first_row() {
    constexpr int kRows = R::kThreads / R::kGroup;
    return (int64_t)blockIdx.x * kRows + (kRows == 1 ? 0 : threadIdx.x / R::kGroup);
}

struct Stats {
    float m, s, log_s, H;
};

struct Sums {
    float m, s, t;
};

__device__ __forceinline__ Stats stats_from(const Sums& a) {
    const float s = fabsf(a.m) < INFINITY ? a.s : NAN, log_s = logf(s);
    return {a.m, s, log_s, log_s - a.t * __builtin_amdgcn_rcpf(s)};
}

// Maximum, then both sums. The longest rows, and all that are not held, gather them in one pass, while their later
// packs are still on the way: a running maximum rescales the sums when it grows. (4096 x 50001, bf16: 214 us against
// 224; with 256 threads a row the two passes are even or ahead by up to 2 %.)
constexpr int kOnePass = 512;

template <typename R>
__device__ __forceinline__ Sums sums_of(const R& r, int lane, float* red) {
    float m = -INFINITY, s = 0.0f, t = 0.0f;
    auto largest = [](const auto& v, float m) {
#pragma unroll
        for (unsigned j = 0; j < sizeof(v) / sizeof(float); ++j) m = Maximum{}(m, v[j]);
        return m;
    };
    auto add = [&](const auto& v) {
#pragma unroll
        for (unsigned j = 0; j < sizeof(v) / sizeof(float); ++j) {
            const float x = exponent(v[j], m), e = exp_of<typename R::T>(x);
            s += e;
            t += e * x;
        }
    };
    if constexpr (R::kGroup < kOnePass) {
        r.each(lane, [&](const auto& v) { m = largest(v, m); });
        m = group_max<R::kGroup>(m, red);
        r.each(lane, add);
    } else {
        auto rescale = [&](float to) {
            const float x = exponent(m, to), e = exp_of<typename R::T>(x);
            t = e * (t + x * s);
            s *= e;
            m = to;
        };
        r.each(lane, [&](const auto& v) {
            const float to = largest(v, m);
            if (!(to <= m)) rescale(to);
            add(v);
        });
        rescale(group_max<R::kGroup>(m, red));
    }
    group_sums<R::kGroup>(s, t, red);
    return {m, s, t};
}

template <typename R>
__device__ __forceinline__ Stats stats_of(const R& r, int lane, float* red) {
    return stats_from(sums_of(r, lane, red));
}

// log p of a logit
__device__ __forceinline__ float log_prob(const Stats& st, float z) { return (z - st.m) - st.log_s; }

// A row's action and its logit.
struct Taken {
    int64_t a;
    float z;
    bool in;
};

template <typename T>
__device__ __forceinline__ Taken taken_of(const int64_t* actions, int64_t m, const T* row, int64_t K) {
    Taken t;
    t.a = actions[m];
    t.in = t.a >= 0 && t.a < K;
    t.z = (float)row[t.in ? t.a : 0];
    return t;
}

// Four waves a SIMD: what a row in LDS beside registers, or a long one read in one pass, needs to keep loads in flight.
template <typename R>
__global__ __launch_bounds__(R::kThreads, R::kThreads >= 512 ? 4 : 0) void log_probs_kernel(
    int64_t M, int64_t K, const typename R::T* __restrict__ logits, int64_t ld, const int64_t* __restrict__ actions,
    float* __restrict__ logp, float* __restrict__ ent, int32_t* __restrict__ bad) {
    constexpr int kRows = R::kThreads / R::kGroup;
    __shared__ float red[2 * R::kThreads / 64];
    const int lane = R::kThreads == R::kGroup ? threadIdx.x : threadIdx.x % R::kGroup;
    for (int64_t m = first_row<R>(); m < M; m += (int64_t)gridDim.x * kRows) {
        R r;
        r.load(logits + m * ld, lane, K);
        const Taken a = taken_of(actions, m, logits + m * ld, K);
        const Stats st = stats_of(r, lane, red);
        if (lane == 0) {
            logp[m] = a.in ? log_prob(st, a.z) : NAN;
            ent[m] = st.H;
            if (!a.in && bad) atomicOr(bad, 1);
        }
    }
}

// Few long rows: each is read by several workgroups, whose maxima and sums are joined by a second kernel.
constexpr int kJoin = 64;

template <typename T>
__global__ __launch_bounds__(512) void log_probs_part_kernel(int64_t K, const T* __restrict__ logits, int64_t ld,
                                                             int64_t part, int64_t parts, float* __restrict__ work) {
    using R = Streamed<T, 512>;
    __shared__ float red[2 * 512 / 64];
    const int64_t m = blockIdx.x / parts, p = blockIdx.x - m * parts;
    const int64_t from = p * part, size = K - from < part ? K - from : part;
    R r;
    r.load(logits + m * ld + from, threadIdx.x, size);
    const Sums a = sums_of(r, threadIdx.x, red);
    if (threadIdx.x == 0) {
        float* w = work + (m * parts + p) * 3;
        w[0] = a.m, w[1] = a.s, w[2] = a.t;
    }
}

template <typename T>
__global__ __launch_bounds__(kJoin) void log_probs_join_kernel(int64_t K, const T* __restrict__ logits, int64_t ld,
                                                               int64_t parts, const float* __restrict__ work,
                                                               const int64_t* __restrict__ actions,
                                                               float* __restrict__ logp, float* __restrict__ ent,
                                                               int32_t* __restrict__ bad) {
    const int64_t m = blockIdx.x;
    const float* w = work + m * parts * 3;
    const Taken a = taken_of(actions, m, logits + m * ld, K);
    float top = -INFINITY, s = 0.0f, t = 0.0f;
    for (int64_t p = threadIdx.x; p < parts; p += kJoin) top = Maximum{}(top, w[3 * p]);
    top = group_max<kJoin>(top, nullptr);
    for (int64_t p = threadIdx.x; p < parts; p += kJoin) {
        const float x = exponent(w[3 * p], top), e = exp_of<T>(x);
        s += e * w[3 * p + 1];
        t += e * (w[3 * p + 2] + x * w[3 * p + 1]);
    }
    group_sums<kJoin>(s, t, nullptr);
    const Stats st = stats_from({top, s, t});
    if (threadIdx.x == 0) {
        logp[m] = a.in ? log_prob(st, a.z) : NAN;
        ent[m] = st.H;
        if (!a.in && bad) atomicOr(bad, 1);
    }
}

struct LossArgs {
    const int64_t* actions;
    const float* old_lp;
    const float* ref_lp;
    const float* adv;
    const uint8_t* mask;
    const float* denom;
    float lo, hi, kl_coef, ent_coef;
};

// active rows, by the whole workgroup, in every thread
template <int THREADS>
__device__ __forceinline__ float count_active(const uint8_t* mask, int64_t M, float* red) {
    int n = 0;
    for (int64_t m = threadIdx.x; m < M; m += THREADS) n += mask[m] ? 1 : 0;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) n += __shfl_xor(n, o);
    int* r = reinterpret_cast<int*>(red);
    if ((threadIdx.x & 63) == 0) r[threadIdx.x >> 6] = n;
    __syncthreads();
    n = 0;
    for (int k = 0; k < THREADS / 64; ++k) n += r[k];
    __syncthreads();
    return (float)n;
}

__device__ __forceinline__ float at_least_one(float n) { return n > 1.0f ? n : 1.0f; }

__global__ __launch_bounds__(1024) void loss_count_kernel(int64_t M, const uint8_t* __restrict__ mask,
                                                          float* __restrict__ used_denom) {
    int64_t n = 0;
    const int64_t packs = M / 16;
    for (int64_t k = threadIdx.x; k < packs; k += 1024) {
        uint32_t w[4];
        __builtin_memcpy(w, mask + 16 * k, 16);
#pragma unroll
        for (int j = 0; j < 4; ++j)      // the top bit of every byte that is not 0
            n += __builtin_popcount((((w[j] & 0x7f7f7f7fu) + 0x7f7f7f7fu) | w[j]) & 0x80808080u);
    }
    for (int64_t m = packs * 16 + threadIdx.x; m < M; m += 1024) n += mask[m] ? 1 : 0;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) n += __shfl_xor(n, o);
    __shared__ int64_t counts[1024 / 64];
    if ((threadIdx.x & 63) == 0) counts[threadIdx.x >> 6] = n;
    __syncthreads();
    if (threadIdx.x != 0) return;
    for (int k = 1; k < 1024 / 64; ++k) n += counts[k];
    *used_denom = at_least_one((float)n);
}

// A row's operands, fetched one row ahead.
struct RowIn {
    bool active;
    float old_lp, ref_lp, adv;
};

__device__ __forceinline__ RowIn row_in(const LossArgs& p, int64_t m, int64_t M) {
    const int64_t k = m < M ? m : M - 1;
    return {!p.mask || p.mask[k], p.old_lp[k], p.ref_lp ? p.ref_lp[k] : 0.0f, p.adv[k]};
}

// What a row adds to the sums, and the gradient g of its terms in l.
struct RowTerms {
    float pg, kl, outside, g;
};

// exp d - d - 1. Its parts cancel where d is small, as it is while a policy stays near its reference: d^2 / 2 (1 + d / 3
// (1 + d / 4 (...))) there, of which 1e-10 is left out at |d| = 1 / 2.
__device__ __forceinline__ float kl_of(float d, float exp_less_1) {
    if (!(fabsf(d) < 0.5f)) return exp_less_1 - d;
    float series = 1.0f;
#pragma unroll
    for (int k = 10; k > 2; --k) series = 1.0f + d * (1.0f / k) * series;
    return 0.5f * d * d * series;
}

__device__ __forceinline__ RowTerms terms_of(const LossArgs& p, const RowIn& in, float l) {
    RowTerms o;
    const float x = l - in.old_lp, A = in.adv;
    const float r = expf(clamp_nan(x, -kBound, kBound));
    const float u = r * A, v = clamp_nan(r, p.lo, p.hi) * A;
    const bool far = x < -kBound || x > kBound;
    // u + v: NaN where either is. At a tie both sides of the minimum carry the gradient of u.
    o.pg = u <= v ? -u : (u > v ? -v : u + v);
    o.g = u <= v ? (far ? 0.0f : -u) : (u > v ? 0.0f : u + v);
    o.outside = r < p.lo || r > p.hi ? 1.0f : 0.0f;
    o.kl = 0.0f;
    if (p.ref_lp) {
        const float y = in.ref_lp - l, d = clamp_nan(y, -kBound, kBound), e = expm1f(d);
        o.kl = kl_of(d, e);
        if (!(y < -kBound || y > kBound)) o.g -= p.kl_coef * e;
    }
    return o;
}

// p_k c (entropy_coef (log p_k + H) - g) = e_k (c1 x_k + c0): a row's gradient but for its action
template <typename T>
struct RowGrad {
    float m, c1, c0;
    __device__ __forceinline__ RowGrad(float m, float s, float log_s, float H, float g, float c, float ent_coef) : m(m) {
        const float share = __builtin_amdgcn_rcpf(s), ce = c * ent_coef;
        c1 = ce * share;
        c0 = (ce * (H - log_s) - c * g) * share;
    }
    __device__ __forceinline__ float operator()(float z) const {
        const float x = exponent(z, m);
        return exp_of<T>(x) * (c1 * x + c0);
    }
};

// A row's gradient. The action's element is stored once more, with its own term, by the thread that stored it.
template <typename R>
__device__ __forceinline__ void write_grad(const R& r, typename R::T* out, int lane, int64_t K, const Taken& a,
                                           float more, const RowGrad<typename R::T>& f) {
    r.write(out, lane, K, f);
    if (a.in && lane == R::owner(a.a)) out[a.a] = (typename R::T)(f(a.z) + more);
}

template <typename R>
__device__ __forceinline__ void zero_row(typename R::T* out, int lane, int64_t K) {
    constexpr int V = 16 / sizeof(typename R::T);
    Pack<typename R::T> none;
    none.clear();
    const int64_t packs = K / V;
    for (int64_t k = lane; k < packs; k += R::kGroup) none.store(out + k * V);
    for (int64_t k = packs * V + lane; k < K; k += R::kGroup) out[k] = (typename R::T)0.0f;
}

template <typename R>
__global__ __launch_bounds__(R::kThreads, 4) void loss_rows_kernel(
    int64_t M, int64_t K, const typename R::T* __restrict__ logits, int64_t ld, LossArgs p,
    const float* __restrict__ counted, float* __restrict__ row_stats, float* __restrict__ partials,
    typename R::T* __restrict__ dz, int32_t* __restrict__ bad) {
    constexpr int kRows = R::kThreads / R::kGroup, W = R::kThreads / 64;
    __shared__ float red[2 * W];
    __shared__ float out[W][kSums];
    const int lane = R::kThreads == R::kGroup ? threadIdx.x : threadIdx.x % R::kGroup;
    float c = 0.0f;
    if (dz) {
        const float d = p.denom ? *p.denom
                        : counted ? *counted
                        : p.mask ? at_least_one(count_active<R::kThreads>(p.mask, M, red)) : (float)M;
        c = 1.0f / d;
    }
    float sums[kSums] = {};
    RowIn next = row_in(p, first_row<R>(), M);
    for (int64_t m = first_row<R>(); m < M; m += (int64_t)gridDim.x * kRows) {
        const RowIn in = next;
        next = row_in(p, m + (int64_t)gridDim.x * kRows, M);
        if (!in.active) {
            if (lane == 0) {
                row_stats[4 * m] = row_stats[4 * m + 2] = row_stats[4 * m + 3] = 0.0f;
                row_stats[4 * m + 1] = kInactive;
            }
            if (dz) zero_row<R>(dz + m * K, lane, K);
            continue;
        }
        R r;
        r.load(logits + m * ld, lane, K);
        const Taken a = taken_of(p.actions, m, logits + m * ld, K);
        const Stats st = stats_of(r, lane, red);
        const RowTerms t = terms_of(p, in, a.in ? log_prob(st, a.z) : NAN);
        if (lane == 0) {
            if (!a.in && bad) atomicOr(bad, 1);
            sums[0] += t.pg;
            sums[1] += t.kl;
            sums[2] += st.H;
            sums[3] += t.outside;
            sums[4] += t.pg + p.kl_coef * t.kl - p.ent_coef * st.H;
            sums[5] += 1.0f;
            row_stats[4 * m] = st.m;
            row_stats[4 * m + 1] = st.s;
            row_stats[4 * m + 2] = st.H;
            row_stats[4 * m + 3] = t.g;
        }
        if (dz) write_grad(r, dz + m * K, lane, K, a, c * t.g, RowGrad<typename R::T>(st.m, st.s, st.log_s, st.H, t.g, c, p.ent_coef));
    }
#pragma unroll
    for (int k = 0; k < kSums; ++k) {
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) sums[k] += __shfl_xor(sums[k], o);
        if ((threadIdx.x & 63) == 0) out[threadIdx.x >> 6][k] = sums[k];
    }
    __syncthreads();
    if (threadIdx.x < kSums) {
        float v = 0.0f;
        for (int w = 0; w < W; ++w) v += out[w][threadIdx.x];
        partials[blockIdx.x * kSums + threadIdx.x] = v;
    }
}

__global__ __launch_bounds__(kFinish) void loss_finish_kernel(int blocks, int64_t M, int has_mask,
                                                          const float* __restrict__ partials,
                                                          const float* __restrict__ denom, float* __restrict__ loss,
                                                          float* __restrict__ terms, float* __restrict__ used_denom) {
    __shared__ double red[kFinish / 64][kSums];
    double s[kSums] = {};
    for (int b = threadIdx.x; b < blocks; b += kFinish)
        for (int k = 0; k < kSums; ++k) s[k] += (double)partials[b * kSums + k];
    for (int k = 0; k < kSums; ++k) {
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) s[k] += __shfl_xor(s[k], o);
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6][k] = s[k];
    }
    __syncthreads();
    if (threadIdx.x != 0) return;
    for (int k = 0; k < kSums; ++k)
        for (int w = 1; w < kFinish / 64; ++w) s[k] += red[w][k];
    const float n = has_mask ? (float)s[5] : (float)M;
    const float d = denom ? *denom : at_least_one(n);
    *loss = (float)(s[4] / (double)d);
    for (int k = 0; k < 4; ++k) terms[k] = (float)(s[k] / (double)d);
    *used_denom = d;
}

template <typename R>
__global__ __launch_bounds__(R::kThreads) void loss_bwd_kernel(
    int64_t M, int64_t K, const typename R::T* __restrict__ logits, int64_t ld, const int64_t* __restrict__ actions,
    float ent_coef, const float* __restrict__ row_stats, const float* __restrict__ used_denom,
    const float* __restrict__ grad, int have, typename R::T* __restrict__ dz) {
    constexpr int kRows = R::kThreads / R::kGroup;
    const float g = *grad;
    if (have && g == 1.0f) return;
    const float c = g / *used_denom;
    const int lane = R::kThreads == R::kGroup ? threadIdx.x : threadIdx.x % R::kGroup;
    for (int64_t m = first_row<R>(); m < M; m += (int64_t)gridDim.x * kRows) {
        const float mx = row_stats[4 * m], s = row_stats[4 * m + 1], H = row_stats[4 * m + 2];
        const float gl = row_stats[4 * m + 3];
        if (s == kInactive) {
            zero_row<R>(dz + m * K, lane, K);
            continue;
        }
        R r;
        r.load(logits + m * ld, lane, K);
        write_grad(r, dz + m * K, lane, K, taken_of(actions, m, logits + m * ld, K), c * gl,
                   RowGrad<typename R::T>(mx, s, logf(s), H, gl, c, ent_coef));
    }
}

// Threads that hold a row of K logits, up to kNarrow of them. Few threads with many loads each leave no barrier and
// little of the last turn unused. 16-bit rows, a thread's 32 / 48 / 64 elements chosen so that few of them are empty,
// against 32 always (loss, us): 66 logits of 10^6 rows 110 / 145, 300 of 200000 63 / 73, 600 of 150000 90 / 108,
// 1200 of 80000 93 / 111; above 2048 a wave and two against four waves: 2500 of 40000 109 / 183, 7000 of 15000 102 / 109.
// For float32 64 elements do not fit the registers, and the same steps gained nothing.
constexpr int64_t kNarrow = 8192;

template <typename T, typename F>
void with_narrow_layout(int64_t K, F&& fn) {
    if (K <= 8) return fn(Single<T, 8>{});
    if (K <= 64) return fn(Wide<T, 4, 16>{});
    if constexpr (sizeof(T) == 2) {
        if (K <= 128) return fn(Wide<T, 4, 32>{});
        if (K <= 256) return fn(Wide<T, 8, 32>{});
        if (K <= 384) return fn(Wide<T, 8, 48>{});
        if (K <= 512) return fn(Wide<T, 16, 32>{});
        if (K <= 768) return fn(Wide<T, 16, 48>{});
        if (K <= 1024) return fn(Wide<T, 32, 32>{});
        if (K <= 1536) return fn(Wide<T, 32, 48>{});
        if (K <= 2048) return fn(Wide<T, 64, 32>{});
        if (K <= 4096) return fn(Wide<T, 64, 64>{});
        fn(Wide<T, 128, 64>{});
    } else {
        if (K <= 256) return fn(Wide<T, 8, 32>{});
        if (K <= 512) return fn(Wide<T, 16, 32>{});
        if (K <= 1024) return fn(Wide<T, 32, 32>{});
        if (K <= 2048) return fn(Wide<T, 64, 32>{});
        fn(Wide<T, 256, 32>{});
    }
}

template <typename T, typename F>
void with_layout(int64_t K, F&& fn) {
    if (K <= kNarrow) return with_narrow_layout<T>(K, fn);
    if constexpr (sizeof(T) == 2) {
        if (K <= 16384) return fn(Wide<T, 256, 64>{});
        if (K <= Wide<T, 256, 64, 8>::kMost) return fn(Wide<T, 256, 64, 8>{});
        if (K <= Wide<T, 512, 64, 8>::kMost) return fn(Wide<T, 512, 64, 8>{});
    } else {
        if (K <= Wide<T, 256, 32, 8>::kMost) return fn(Wide<T, 256, 32, 8>{});
        if (K <= Wide<T, 512, 32, 8>::kMost) return fn(Wide<T, 512, 32, 8>{});
    }
    fn(Streamed<T, 512>{});
}

// For one use of a row, the backward call's: nothing has to be held.
template <typename T, typename F>
void with_pass(int64_t K, F&& fn) {
    if (K <= 8) fn(Single<T, 8>{});
    else if (K <= 64) fn(Streamed<T, 4>{});
    else if (K <= 512) fn(Streamed<T, 16>{});
    else if (K <= 2048) fn(Streamed<T, 64>{});
    else fn(Streamed<T, 256>{});
}

// How log_probs splits rows: long ones, when there are fewer than two for each CU, into parts of at least 8192
// logits (a workgroup's 512 threads with two packs of 16 bits or four of 32 each). 100 x 150000, bf16: 11.6 + 3.8 us.
struct Parts {
    int64_t part, parts;
};

Parts parts_of(int64_t M, int64_t K) {
    constexpr int64_t kLeast = 8192, kFull = 512;
    if (M < 1 || M >= kFull || K < 2 * kLeast) return {K, 1};
    int64_t parts = (kFull + M - 1) / M;
    if (parts > K / kLeast) parts = K / kLeast;
    const int64_t part = ((K + parts - 1) / parts + 7) / 8 * 8;
    return {part, (K + part - 1) / part};
}

template <typename R>
unsigned grid_of(int64_t M, int64_t most) {
    const int64_t rows = R::kThreads / R::kGroup, b = (M + rows - 1) / rows;
    return (unsigned)(b < most ? b : most);
}

}  // namespace

extern "C" {

int64_t swarm_log_probs_workspace(int64_t M, int64_t K) {
    if (M < 0 || K < 1 || !sane(M, K)) return SWARM_ERR_ARG;
    const Parts p = parts_of(M, K);
    return p.parts > 1 ? M * p.parts * 3 : 0;
}

int32_t swarm_log_probs(int32_t dtype, int64_t M, int64_t K, const void* logits, int64_t row_stride,
                        const int64_t* actions, float* log_probs, float* entropy, float* work, int32_t* bad_actions,
                        void* stream) {
    if (!known_type(dtype) || M < 0 || K < 1 || !sane(M, K)) return SWARM_ERR_ARG;
    if (M == 0) return SWARM_OK;
    if (!logits || !actions || !log_probs || !entropy || row_stride < 0) return SWARM_ERR_ARG;
    if (parts_of(M, K).parts > 1 && !work) return SWARM_ERR_ARG;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    with_type(dtype, [&](auto e) {
        using E = decltype(e);
        auto run = [&](auto layout) {
            using R = decltype(layout);
            log_probs_kernel<R><<<grid_of<R>(M, 1 << 20), R::kThreads, 0, st>>>(
                M, K, static_cast<const E*>(logits), row_stride, actions, log_probs, entropy, bad_actions);
        };
        const Parts p = parts_of(M, K);
        if (p.parts > 1) {
            const E* z = static_cast<const E*>(logits);
            log_probs_part_kernel<E><<<(unsigned)(M * p.parts), 512, 0, st>>>(K, z, row_stride, p.part, p.parts, work);
            log_probs_join_kernel<E><<<(unsigned)M, kJoin, 0, st>>>(K, z, row_stride, p.parts, work, actions, log_probs,
                                                                  entropy, bad_actions);
        } else if (K > kNarrow) {      // nothing uses the row a second time: no need to hold it
            run(Streamed<E, 512>{});
        } else {
            with_narrow_layout<E>(K, run);
        }
    });
    return swarm::record_hip_status();
}

int32_t swarm_policy_loss_forward(int32_t dtype, int64_t M, int64_t K, const void* logits, int64_t row_stride,
                                  const int64_t* actions, const float* old_log_probs, const float* ref_log_probs,
                                  const float* advantages, const uint8_t* mask_u8, const float* denom, float clip_lo,
                                  float clip_hi, float kl_coef, float entropy_coef, float* loss, float* terms,
                                  float* used_denom, float* row_stats, void* d_logits, float* partials,
                                  int32_t* bad_actions, void* stream) {
    if (!known_type(dtype) || M < 0 || K < 1 || !sane(M, K) || !loss || !terms || !used_denom || !partials ||
        !(clip_lo <= clip_hi))
        return SWARM_ERR_ARG;
    if (M > 0 && (!logits || !actions || !old_log_probs || !advantages || !row_stats || row_stride < 0))
        return SWARM_ERR_ARG;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    unsigned blocks = 0;
    if (M > 0) {
        const LossArgs p{actions, old_log_probs, ref_log_probs, advantages, mask_u8, denom, clip_lo, clip_hi, kl_coef,
                         entropy_coef};
        with_type(dtype, [&](auto e) {
            using E = decltype(e);
            with_layout<E>(K, [&](auto layout) {
                using R = decltype(layout);
                blocks = grid_of<R>(M, kMaxBlocks);
                const bool count = d_logits && mask_u8 && !denom && blocks > kCountHere;
                if (count) loss_count_kernel<<<1, 1024, 0, st>>>(M, mask_u8, used_denom);
                loss_rows_kernel<R><<<blocks, R::kThreads, R::lds_bytes(K), st>>>(M, K, static_cast<const E*>(logits), row_stride, p,
                                                                  count ? used_denom : nullptr, row_stats, partials,
                                                                  static_cast<E*>(d_logits), bad_actions);
            });
        });
    }
    loss_finish_kernel<<<1, kFinish, 0, st>>>((int)blocks, M, mask_u8 != nullptr, partials, denom, loss, terms, used_denom);
    return swarm::record_hip_status();
}

int32_t swarm_policy_loss_backward(int32_t dtype, int64_t M, int64_t K, const void* logits, int64_t row_stride,
                                   const int64_t* actions, float entropy_coef, const float* row_stats,
                                   const float* used_denom, const float* grad, int32_t have_unit, void* d_logits,
                                   void* stream) {
    if (!known_type(dtype) || M < 0 || K < 1 || !sane(M, K)) return SWARM_ERR_ARG;
    if (M == 0) return SWARM_OK;
    if (!logits || !actions || !row_stats || !used_denom || !grad || !d_logits || row_stride < 0) return SWARM_ERR_ARG;
    with_type(dtype, [&](auto e) {
        using E = decltype(e);
        with_pass<E>(K, [&](auto layout) {
            using R = decltype(layout);
            loss_bwd_kernel<R><<<grid_of<R>(M, kMaxBlocks), R::kThreads, 0, static_cast<hipStream_t>(stream)>>>(
                M, K, static_cast<const E*>(logits), row_stride, actions, entropy_coef, row_stats, used_denom, grad,
                have_unit, static_cast<E*>(d_logits));
        });
    });
    return swarm::record_hip_status();
}

}  // extern "C"
