// swarm_policyloss.hip — log-probabilities and the clipped policy loss with a KL term, from logits
// (include/swarmseq.h: swarm_log_probs, swarm_policy_loss_*).
//
// Per row of K logits z with the taken action a, m = max z, s = sum exp(z - m), t = sum exp(z - m) (z - m):
//   L = m + log s,  l = z_a - L,  H = log s - t / s,  p_k = exp(z_k - L)
//   dz_k = (1 / denom) [ g (1[k = a] - p_k) + entropy_coef p_k (log p_k + H) ],
//   g = d pg / d l + kl_coef (1 - exp(ref - l)).
// m, s and t are gathered in one pass: a running maximum rescales the two sums when it grows. A logit of -inf
// adds nothing to either sum and has no gradient.
#include "swarm_seq.h"

using namespace swarm_seq;

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kMaxBlocks = 2048;      // SWARM_POLICY_LOSS_PARTIALS = 6 sums for each
constexpr int kSums = 6;              // pg, kl, H, outside, pg + kl_coef kl - entropy_coef H, active rows
constexpr float kBound = 20.0f;       // bound of the log-ratios

struct Stats {
    float m, s, t;
};

__device__ __forceinline__ float exp_of(float x) { return __builtin_amdgcn_exp2f(x * kLog2e); }

__device__ __forceinline__ void add_logit(Stats& a, float z) {
    if (z > a.m) {
        const float d = a.m - z;
        if (a.m != -INFINITY) {
            const float e = exp_of(d);
            a.t = e * (a.t + d * a.s);
            a.s *= e;
        }
        a.m = z;
    }
    if (z != -INFINITY) {
        const float d = z - a.m, e = exp_of(d);
        a.s += e;
        a.t += e > 0.0f ? e * d : e;   // e * d: 0 * -inf for a logit far below; a NaN stays
    }
}

__device__ __forceinline__ Stats merge(const Stats& a, const Stats& b) {
    if (b.m == -INFINITY && b.s == 0.0f) return a;
    if (a.m == -INFINITY && a.s == 0.0f) return b;
    Stats r;
    r.m = fmaxf(a.m, b.m);
    const float da = a.m - r.m, db = b.m - r.m, ea = exp_of(da), eb = exp_of(db);
    r.s = ea * a.s + eb * b.s;
    r.t = (ea > 0.0f || ea != ea ? ea * (a.t + da * a.s) : 0.0f) + (eb > 0.0f || eb != eb ? eb * (b.t + db * b.s) : 0.0f);
    return r;
}

template <typename T>
__device__ Stats row_stats_of(const T* __restrict__ z, int64_t K, Stats* red) {
    Stats a{-INFINITY, 0.0f, 0.0f};
    for (int64_t k = threadIdx.x; k < K; k += kThreads) add_logit(a, (float)z[k]);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        Stats b{__shfl_xor(a.m, o), __shfl_xor(a.s, o), __shfl_xor(a.t, o)};
        a = merge(a, b);
    }
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = a;
    __syncthreads();
    a = red[0];
    for (int k = 1; k < kWaves; ++k) a = merge(a, red[k]);
    return a;
}

// clamp that keeps a NaN
__device__ __forceinline__ float clamp_nan(float x, float lo, float hi) { return x < lo ? lo : (x > hi ? hi : x); }

template <typename T>
__global__ __launch_bounds__(kThreads) void log_probs_kernel(int64_t M, int64_t K, const T* __restrict__ logits, int64_t ld,
                                                             const int64_t* __restrict__ actions,
                                                             float* __restrict__ logp, float* __restrict__ ent,
                                                             int32_t* __restrict__ bad) {
    __shared__ Stats red[kWaves];
    for (int64_t m = blockIdx.x; m < M; m += gridDim.x) {
        const T* z = logits + m * ld;
        const Stats a = row_stats_of(z, K, red);
        if (threadIdx.x == 0) {
            const int64_t k = actions[m];
            const bool in = k >= 0 && k < K;
            const float ls = logf(a.s);
            logp[m] = in ? ((float)z[k] - a.m) - ls : NAN;
            ent[m] = ls - a.t / a.s;
            if (!in && bad) atomicOr(bad, 1);
        }
    }
}

struct LossArgs {
    const int64_t* actions;
    const float* old_lp;
    const float* ref_lp;
    const float* adv;
    const uint8_t* mask;
    float lo, hi, kl_coef, ent_coef;
};

template <typename T>
__global__ __launch_bounds__(kThreads) void loss_rows_kernel(int64_t M, int64_t K, const T* __restrict__ logits, int64_t ld,
                                                             LossArgs p, float* __restrict__ row_stats,
                                                             float* __restrict__ partials, int32_t* __restrict__ bad) {
    __shared__ Stats red[kWaves];
    float sums[kSums] = {};
    for (int64_t m = blockIdx.x; m < M; m += gridDim.x) {
        if (p.mask && !p.mask[m]) {
            if (threadIdx.x < 4) row_stats[4 * m + threadIdx.x] = 0.0f;
            continue;
        }
        const T* z = logits + m * ld;
        const Stats a = row_stats_of(z, K, red);
        if (threadIdx.x != 0) continue;
        const int64_t k = p.actions[m];
        const bool in = k >= 0 && k < K;
        if (!in && bad) atomicOr(bad, 1);
        const float ls = logf(a.s);
        const float l = in ? ((float)z[k] - a.m) - ls : NAN;
        const float H = ls - a.t / a.s;
        const float x = l - p.old_lp[m], A = p.adv[m];
        const float r = expf(clamp_nan(x, -kBound, kBound));
        const float u = r * A, v = clamp_nan(r, p.lo, p.hi) * A;
        const float pg = u <= v ? -u : (u > v ? -v : u + v);
        float g = (u <= v && x >= -kBound && x <= kBound) ? -u : (u > v ? 0.0f : u + v);
        if (u <= v && !(x >= -kBound && x <= kBound)) g = 0.0f;
        float kl = 0.0f;
        if (p.ref_lp) {
            const float y = p.ref_lp[m] - l, d = clamp_nan(y, -kBound, kBound), e = expf(d);
            kl = e - d - 1.0f;
            if (y >= -kBound && y <= kBound) g += p.kl_coef * (1.0f - e);
        }
        sums[0] += pg;
        sums[1] += kl;
        sums[2] += H;
        sums[3] += (r < p.lo || r > p.hi) ? 1.0f : 0.0f;
        sums[4] += pg + p.kl_coef * kl - p.ent_coef * H;
        sums[5] += 1.0f;
        row_stats[4 * m] = a.m + ls;
        row_stats[4 * m + 1] = H;
        row_stats[4 * m + 2] = g;
        row_stats[4 * m + 3] = 1.0f;
    }
    if (threadIdx.x == 0)
        for (int k = 0; k < kSums; ++k) partials[blockIdx.x * kSums + k] = sums[k];
}

__global__ __launch_bounds__(kThreads) void loss_finish_kernel(int blocks, int64_t M, int has_mask,
                                                               const float* __restrict__ partials,
                                                               const float* __restrict__ denom,
                                                               float* __restrict__ loss, float* __restrict__ terms,
                                                               float* __restrict__ used_denom) {
    __shared__ double red[kWaves][kSums];
    double s[kSums] = {};
    for (int b = threadIdx.x; b < blocks; b += kThreads)
        for (int k = 0; k < kSums; ++k) s[k] += (double)partials[b * kSums + k];
    for (int k = 0; k < kSums; ++k) {
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) s[k] += __shfl_xor(s[k], o);
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6][k] = s[k];
    }
    __syncthreads();
    if (threadIdx.x != 0) return;
    for (int k = 0; k < kSums; ++k)
        for (int w = 1; w < kWaves; ++w) s[k] += red[w][k];
    const double n = has_mask ? s[5] : (double)M;
    const double d = denom ? (double)*denom : (n > 1.0 ? n : 1.0);
    *loss = (float)(s[4] / d);
    for (int k = 0; k < 4; ++k) terms[k] = (float)(s[k] / d);
    *used_denom = (float)d;
}

template <typename T>
__global__ __launch_bounds__(kThreads) void loss_bwd_kernel(int64_t M, int64_t K, const T* __restrict__ logits, int64_t ld,
                                                            const int64_t* __restrict__ actions, float ent_coef,
                                                            const float* __restrict__ row_stats,
                                                            const float* __restrict__ used_denom,
                                                            const float* __restrict__ grad, T* __restrict__ dz) {
    const float scale = *grad / *used_denom;
    for (int64_t m = blockIdx.x; m < M; m += gridDim.x) {
        const float L = row_stats[4 * m], H = row_stats[4 * m + 1], g = row_stats[4 * m + 2];
        const bool active = row_stats[4 * m + 3] != 0.0f;
        const int64_t a = actions[m];
        for (int64_t k = threadIdx.x; k < K; k += kThreads) {
            float d = 0.0f;
            if (active) {
                const float lp = (float)logits[m * ld + k] - L, q = exp_of(lp);
                d = g * ((k == a ? 1.0f : 0.0f) - q) + (q == 0.0f ? 0.0f : ent_coef * q * (lp + H));
                d *= scale;
            }
            dz[m * K + k] = (T)d;
        }
    }
}

unsigned blocks_of(int64_t M) { return (unsigned)(M < kMaxBlocks ? M : kMaxBlocks); }

}  // namespace

extern "C" {

int32_t swarm_log_probs(int32_t dtype, int64_t M, int64_t K, const void* logits, int64_t row_stride,
                        const int64_t* actions, float* log_probs, float* entropy, int32_t* bad_actions, void* stream) {
    if (!known_type(dtype) || M < 0 || K < 1 || !sane(M, K)) return SWARM_ERR_ARG;
    if (M == 0) return SWARM_OK;
    if (!logits || !actions || !log_probs || !entropy || row_stride < 0) return SWARM_ERR_ARG;
    with_type(dtype, [&](auto e) {
        using E = decltype(e);
        log_probs_kernel<E><<<(unsigned)(M < 65536 ? M : 65536), kThreads, 0, static_cast<hipStream_t>(stream)>>>(
            M, K, static_cast<const E*>(logits), row_stride, actions, log_probs, entropy, bad_actions);
    });
    return swarm::record_hip_status();
}

int32_t swarm_policy_loss_forward(int32_t dtype, int64_t M, int64_t K, const void* logits, int64_t row_stride,
                                  const int64_t* actions, const float* old_log_probs, const float* ref_log_probs,
                                  const float* advantages, const uint8_t* mask_u8, const float* denom, float clip_lo,
                                  float clip_hi, float kl_coef, float entropy_coef, float* loss, float* terms,
                                  float* used_denom, float* row_stats, float* partials, int32_t* bad_actions,
                                  void* stream) {
    if (!known_type(dtype) || M < 0 || K < 1 || !sane(M, K) || !loss || !terms || !used_denom || !partials ||
        !(clip_lo <= clip_hi))
        return SWARM_ERR_ARG;
    if (M > 0 && (!logits || !actions || !old_log_probs || !advantages || !row_stats || row_stride < 0))
        return SWARM_ERR_ARG;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    const unsigned blocks = blocks_of(M);
    if (M > 0) {
        const LossArgs p{actions, old_log_probs, ref_log_probs, advantages, mask_u8, clip_lo, clip_hi, kl_coef,
                         entropy_coef};
        with_type(dtype, [&](auto e) {
            using E = decltype(e);
            loss_rows_kernel<E><<<blocks, kThreads, 0, st>>>(M, K, static_cast<const E*>(logits), row_stride, p,
                                                            row_stats, partials, bad_actions);
        });
    }
    loss_finish_kernel<<<1, kThreads, 0, st>>>((int)blocks, M, mask_u8 != nullptr, partials, denom, loss, terms,
                                              used_denom);
    return swarm::record_hip_status();
}

int32_t swarm_policy_loss_backward(int32_t dtype, int64_t M, int64_t K, const void* logits, int64_t row_stride,
                                   const int64_t* actions, float entropy_coef, const float* row_stats,
                                   const float* used_denom, const float* grad, void* d_logits, void* stream) {
    if (!known_type(dtype) || M < 0 || K < 1 || !sane(M, K)) return SWARM_ERR_ARG;
    if (M == 0) return SWARM_OK;
    if (!logits || !actions || !row_stats || !used_denom || !grad || !d_logits || row_stride < 0) return SWARM_ERR_ARG;
    with_type(dtype, [&](auto e) {
        using E = decltype(e);
        loss_bwd_kernel<E><<<(unsigned)(M < 65536 ? M : 65536), kThreads, 0, static_cast<hipStream_t>(stream)>>>(
            M, K, static_cast<const E*>(logits), row_stride, actions, entropy_coef, row_stats, used_denom, grad,
            static_cast<E*>(d_logits));
    });
    return swarm::record_hip_status();
}

}  // extern "C"
