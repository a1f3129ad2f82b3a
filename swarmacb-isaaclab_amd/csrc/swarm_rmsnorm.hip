// swarm_rmsnorm.hip — root-mean-square norm of a residual sum (include/swarmseq.h: swarm_residual_norm_*).
//
//   s = x + r,  rstd = (mean(s^2) + eps)^-1/2,  n = s rstd,  y = n w
//   d_x = d_r = rstd (w dy - n mean(w dy n)) + d_stream,   d_w = sum over rows of dy n
//
// Memory bound: a row is read once, held in registers by as many threads as it needs (part of a wave or a wave up to
// 2048 elements, else a workgroup), and written once. Packs of 16 bytes at any alignment; the last pack of a row is moved left to
// end with it, so no load crosses the row: the elements it shares with the pack before are left out of the sums and
// not stored. The backward pass keeps every thread's columns over all rows of its workgroup and adds the weight
// gradient there; the workgroups' sums are added in a fixed order by a second kernel.
//
// Measured (a 4 GiB copy reaches 4.8 TB/s of reads and writes together on this card):
//   16384 x 4096, bf16: forward 83 us, 6.5 TB/s; backward 139 us, 4.8 TB/s, and 5 us for the weight gradient's last sum
//   5001 x 1001, float16: 9 us, then 16 + 7 us;  200000 x 512, bf16: 143 and 164 us, 5.7 and 6.2 TB/s
//   16384 x 4096, float16: 80 us, then 139 + 5 us
//   4096 x 16384, float32, where the backward pass spills 80 bytes a thread (16 bits: 36 to 44): 250 and 278 us, 4.3 and
//     4.8 TB/s
//   20000 x 20000, bf16, read twice: 1.5 and 2.9 ms, 2.2 and 1.4 TB/s by what one reading would move
#include <type_traits>

#include "swarm_seq.h"

using namespace swarm_seq;

namespace {

constexpr int64_t kResident = 256 * 1024;   // threads of the backward pass, at most: four waves on each SIMD
constexpr int kFinish = 1024;               // threads of the weight gradient's last sum, 32 to a column
constexpr int kFinishCols = 32;

// One row's layout: GROUP threads (part of a wave, a wave, or the whole workgroup), EPT elements of each.
template <typename T, int GROUP, int EPT>
struct Row {
    static constexpr int V = 16 / sizeof(T);
    static constexpr int NP = EPT / V;
    static constexpr int kThreads = GROUP <= 64 ? 256 : GROUP;
    static constexpr int kRows = kThreads / GROUP;     // rows of a workgroup at a time
    static constexpr int kWaves = kThreads / 64;

    // pack i of a thread: its first column, and how many of its elements belong to the pack before
    static __device__ __forceinline__ void place(int i, int lane, int64_t D, int64_t& start, int& skip) {
        const int64_t want = (int64_t)(i * GROUP + lane) * V;
        start = want < D - V ? want : D - V;
        skip = want - start < V ? (int)(want - start) : V;
    }
};

// Stores the elements of a pack that are its own.
template <typename T, int N>
__device__ __forceinline__ void store_own(T* p, const Pack<T, N>& v, int skip) {
    if (skip == 0) {
        v.store(p);
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j)
            if (j >= skip) p[j] = (T)v.get(j);
    }
}

// the sum of v over a row's threads, in every one
template <int GROUP>
__device__ __forceinline__ float row_sum(float v, float* red) {
    v = lanes_reduce<(GROUP < 64 ? GROUP : 64)>(v, Add{});
    if constexpr (GROUP > 64) {
        __syncthreads();
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
        __syncthreads();
        v = 0.0f;
#pragma unroll
        for (int k = 0; k < GROUP / 64; ++k) v += red[k];
    }
    return v;
}

template <typename T, int GROUP, int EPT>
__global__ __launch_bounds__((Row<T, GROUP, EPT>::kThreads)) void norm_fwd_kernel(
    int64_t rows, int64_t D, const T* __restrict__ x, int64_t xr, const T* __restrict__ res, int64_t rr,
    const T* __restrict__ w, float eps, T* __restrict__ y, T* __restrict__ out, float* __restrict__ rstd) {
    using R = Row<T, GROUP, EPT>;
    __shared__ float red[R::kWaves];
    const int lane = threadIdx.x % GROUP;
    const int64_t row = (int64_t)blockIdx.x * R::kRows + threadIdx.x / GROUP;
    if (row >= rows) return;      // whole rows: with GROUP > 64 a workgroup has one
    Pack<T> a[R::NP], b[R::NP], wt[R::NP];
#pragma unroll
    for (int i = 0; i < R::NP; ++i) {
        int64_t start;
        int skip;
        R::place(i, lane, D, start, skip);
        a[i].load(x + row * xr + start);
        if (res) b[i].load(res + row * rr + start);
        if (w) wt[i].load(w + start);
    }
    float ss = 0.0f;
#pragma unroll
    for (int i = 0; i < R::NP; ++i) {
        int64_t start;
        int skip;
        R::place(i, lane, D, start, skip);
        float own = 0.0f;
#pragma unroll
        for (int j = 0; j < R::V; ++j) {
            const float s = a[i].get(j) + (res ? b[i].get(j) : 0.0f);
            own += j >= skip ? s * s : 0.0f;
        }
        ss += own;
    }
    const float inv = 1.0f / sqrtf(row_sum<GROUP>(ss, red) / (float)D + eps);
#pragma unroll
    for (int i = 0; i < R::NP; ++i) {
        int64_t start;
        int skip;
        R::place(i, lane, D, start, skip);
        if (skip >= R::V) continue;
        float s[R::V], n[R::V];
#pragma unroll
        for (int j = 0; j < R::V; ++j) {
            s[j] = a[i].get(j) + (res ? b[i].get(j) : 0.0f);
            n[j] = s[j] * inv * (w ? wt[i].get(j) : 1.0f);
        }
        Pack<T> v;
        if (res) {
            v.set(s);
            store_own(out + row * D + start, v, skip);
        }
        v.set(n);
        store_own(y + row * D + start, v, skip);
    }
    if (rstd && lane == 0) rstd[row] = inv;
}

template <typename T, int GROUP, int EPT>
__global__ __launch_bounds__((Row<T, GROUP, EPT>::kThreads), 4) void norm_bwd_kernel(
    int64_t rows, int64_t D, const T* __restrict__ x, int64_t xr, const T* __restrict__ res, int64_t rr,
    const T* __restrict__ w, const float* __restrict__ rstd, const T* __restrict__ dy, int64_t dyr, const T* __restrict__ ds, int64_t dsr,
    T* __restrict__ dx, float* __restrict__ partials) {
    using R = Row<T, GROUP, EPT>;
    __shared__ float red[R::kWaves];
    extern __shared__ float sums[];     // [kRows][D]: the workgroup's weight gradient, where it has several rows
    const int lane = threadIdx.x % GROUP, group = threadIdx.x / GROUP;
    float dw[R::NP][R::V];
#pragma unroll
    for (int i = 0; i < R::NP; ++i)
#pragma unroll
        for (int j = 0; j < R::V; ++j) dw[i][j] = 0.0f;
    // GROUP > 64: every thread of the workgroup has the same row, so the barriers of row_sum are reached by all
    for (int64_t row = (int64_t)blockIdx.x * R::kRows + group; row < rows; row += (int64_t)gridDim.x * R::kRows) {
        const float inv = rstd[row];
        Pack<T> a[R::NP], b[R::NP], g[R::NP], e[R::NP], wt[R::NP];
#pragma unroll
        for (int i = 0; i < R::NP; ++i) {
            int64_t start;
            int skip;
            R::place(i, lane, D, start, skip);
            a[i].load(x + row * xr + start);
            if (res) b[i].load(res + row * rr + start);
            g[i].load(dy + row * dyr + start);
            if (ds) e[i].load(ds + row * dsr + start);
            if (w) wt[i].load(w + start);
        }
        float dot = 0.0f;
#pragma unroll
        for (int i = 0; i < R::NP; ++i) {
            int64_t start;
            int skip;
            R::place(i, lane, D, start, skip);
            float own = 0.0f;
#pragma unroll
            for (int j = 0; j < R::V; ++j) {
                const float n = (a[i].get(j) + (res ? b[i].get(j) : 0.0f)) * inv, t = g[i].get(j) * n;
                dw[i][j] += t;
                own += j >= skip ? t * (w ? wt[i].get(j) : 1.0f) : 0.0f;
            }
            dot += own;
        }
        const float mean = row_sum<GROUP>(dot, red) / (float)D;
#pragma unroll
        for (int i = 0; i < R::NP; ++i) {
            int64_t start;
            int skip;
            R::place(i, lane, D, start, skip);
            if (skip >= R::V) continue;
            float v[R::V];
#pragma unroll
            for (int j = 0; j < R::V; ++j) {
                const float n = (a[i].get(j) + (res ? b[i].get(j) : 0.0f)) * inv;
                v[j] = inv * (g[i].get(j) * (w ? wt[i].get(j) : 1.0f) - n * mean);
                if (ds) v[j] += e[i].get(j);
            }
            Pack<T> out;
            out.set(v);
            store_own(dx + row * D + start, out, skip);
        }
    }
    if (!partials) return;
#pragma unroll
    for (int i = 0; i < R::NP; ++i) {
        int64_t start;
        int skip;
        R::place(i, lane, D, start, skip);
        float* to = R::kRows > 1 ? sums + group * D + start : partials + blockIdx.x * D + start;
#pragma unroll
        for (int j = 0; j < R::V; ++j)
            if (j >= skip) to[j] = dw[i][j];
    }
    if constexpr (R::kRows > 1) {
        __syncthreads();
        for (int64_t d = threadIdx.x; d < D; d += R::kThreads) {
            float t = sums[d];
#pragma unroll
            for (int k = 1; k < R::kRows; ++k) t += sums[k * D + d];
            partials[blockIdx.x * D + d] = t;
        }
    }
}

// d_w = column sums of the workgroups' partial sums, each column by kFinish / kFinishCols threads
template <typename T>
__global__ __launch_bounds__(kFinish) void weight_finish_kernel(int64_t count, int64_t D, const float* __restrict__ partials,
                                                                T* __restrict__ dw) {
    constexpr int kParts = kFinish / kFinishCols;
    __shared__ float red[kParts][kFinishCols];
    const int col = threadIdx.x % kFinishCols, part = threadIdx.x / kFinishCols;
    const int64_t d = (int64_t)blockIdx.x * kFinishCols + col;
    float acc = 0.0f;
    if (d < D) {
#pragma unroll 8
        for (int64_t k = part; k < count; k += kParts) acc += partials[k * D + d];
    }
    red[part][col] = acc;
    __syncthreads();
    if (part != 0 || d >= D) return;
#pragma unroll
    for (int k = 1; k < kParts; ++k) acc += red[k][col];
    dw[d] = (T)acc;
}

// Rows narrower than a pack: one thread each. (A workgroup each, as for the widest, took 589 + 876 us for 10^6 rows of
// 6 in bf16, forward and backward.)
template <typename T>
struct NarrowRow {
    static constexpr int kMost = 16 / sizeof(T) - 1;
    float v[kMost];
    __device__ __forceinline__ void load(const T* p, int D) {
#pragma unroll
        for (int j = 0; j < kMost; ++j) v[j] = p && j < D ? (float)p[j] : 0.0f;
    }
    __device__ __forceinline__ void store(T* p, int D) const {
#pragma unroll
        for (int j = 0; j < kMost; ++j)
            if (j < D) p[j] = (T)v[j];
    }
};

constexpr int kNarrow = 256;

template <typename T>
__global__ __launch_bounds__(kNarrow) void narrow_fwd_kernel(int64_t rows, int D, const T* __restrict__ x, int64_t xr,
                                                             const T* __restrict__ res, int64_t rr,
                                                             const T* __restrict__ w, float eps, T* __restrict__ y,
                                                             T* __restrict__ out, float* __restrict__ rstd) {
    using R = NarrowRow<T>;
    R wt;
    wt.load(w, D);
    for (int64_t r = (int64_t)blockIdx.x * kNarrow + threadIdx.x; r < rows; r += (int64_t)gridDim.x * kNarrow) {
        R s, b;
        s.load(x + r * xr, D);
        b.load(res ? res + r * rr : nullptr, D);
        float ss = 0.0f;
#pragma unroll
        for (int j = 0; j < R::kMost; ++j) {
            s.v[j] += b.v[j];
            ss += s.v[j] * s.v[j];
        }
        const float inv = 1.0f / sqrtf(ss / (float)D + eps);
        if (res) s.store(out + r * D, D);
#pragma unroll
        for (int j = 0; j < R::kMost; ++j) s.v[j] *= inv * (w ? wt.v[j] : 1.0f);
        s.store(y + r * D, D);
        if (rstd) rstd[r] = inv;
    }
}

template <typename T>
__global__ __launch_bounds__(kNarrow) void narrow_bwd_kernel(int64_t rows, int D, const T* __restrict__ x, int64_t xr,
                                                             const T* __restrict__ res, int64_t rr,
                                                             const T* __restrict__ w, const float* __restrict__ rstd,
                                                             const T* __restrict__ dy, int64_t dyr,
                                                             const T* __restrict__ ds, int64_t dsr, T* __restrict__ dx,
                                                             float* __restrict__ partials) {
    using R = NarrowRow<T>;
    __shared__ float red[kNarrow / 64][R::kMost];
    R wt;
    wt.load(w, D);
    float dw[R::kMost] = {};
    for (int64_t r = (int64_t)blockIdx.x * kNarrow + threadIdx.x; r < rows; r += (int64_t)gridDim.x * kNarrow) {
        const float inv = rstd[r];
        R n, b, g, e;
        n.load(x + r * xr, D);
        b.load(res ? res + r * rr : nullptr, D);
        g.load(dy + r * dyr, D);
        e.load(ds ? ds + r * dsr : nullptr, D);
        float dot = 0.0f;
#pragma unroll
        for (int j = 0; j < R::kMost; ++j) {
            n.v[j] = (n.v[j] + b.v[j]) * inv;
            dw[j] += g.v[j] * n.v[j];
            g.v[j] *= w ? wt.v[j] : 1.0f;
            dot += g.v[j] * n.v[j];
        }
        const float mean = dot / (float)D;
#pragma unroll
        for (int j = 0; j < R::kMost; ++j) e.v[j] += inv * (g.v[j] - n.v[j] * mean);
        e.store(dx + r * D, D);
    }
    if (!partials) return;
#pragma unroll
    for (int j = 0; j < R::kMost; ++j) {
        const float v = lanes_reduce<64>(dw[j], Add{});
        if (threadIdx.x % 64 == 0) red[threadIdx.x / 64][j] = v;
    }
    __syncthreads();
    if (threadIdx.x >= (unsigned)D) return;
    float v = 0.0f;
    for (int k = 0; k < kNarrow / 64; ++k) v += red[k][threadIdx.x];
    partials[(int64_t)blockIdx.x * D + threadIdx.x] = v;
}

// Rows wider than a workgroup's registers: element by element, the row read again for the second use.
constexpr int kPlain = 256;

template <typename T>
__global__ __launch_bounds__(kPlain) void plain_fwd_kernel(int64_t rows, int64_t D, const T* __restrict__ x, int64_t xr,
                                                           const T* __restrict__ res, int64_t rr,
                                                           const T* __restrict__ w, float eps, T* __restrict__ y,
                                                           T* __restrict__ out, float* __restrict__ rstd) {
    __shared__ float red[kPlain / 64];
    for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
        float ss = 0.0f;
        for (int64_t d = threadIdx.x; d < D; d += kPlain) {
            const float s = (float)x[r * xr + d] + (res ? (float)res[r * rr + d] : 0.0f);
            ss += s * s;
        }
        const float inv = 1.0f / sqrtf(row_sum<kPlain>(ss, red) / (float)D + eps);
        for (int64_t d = threadIdx.x; d < D; d += kPlain) {
            const float s = (float)x[r * xr + d] + (res ? (float)res[r * rr + d] : 0.0f);
            if (res) out[r * D + d] = (T)s;
            y[r * D + d] = (T)(s * inv * (w ? (float)w[d] : 1.0f));
        }
        if (rstd && threadIdx.x == 0) rstd[r] = inv;
    }
}

template <typename T>
__global__ __launch_bounds__(kPlain) void plain_bwd_kernel(int64_t rows, int64_t D, const T* __restrict__ x, int64_t xr,
                                                           const T* __restrict__ res, int64_t rr,
                                                           const T* __restrict__ w, const float* __restrict__ rstd,
                                                           const T* __restrict__ dy, int64_t dyr,
                                                           const T* __restrict__ ds, int64_t dsr,
                                                           T* __restrict__ dx) {
    __shared__ float red[kPlain / 64];
    for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
        const float inv = rstd[r];
        float dot = 0.0f;
        for (int64_t d = threadIdx.x; d < D; d += kPlain)
            dot += (float)dy[r * dyr + d] * (w ? (float)w[d] : 1.0f) *
                   (((float)x[r * xr + d] + (res ? (float)res[r * rr + d] : 0.0f)) * inv);
        const float mean = row_sum<kPlain>(dot, red) / (float)D;
        for (int64_t d = threadIdx.x; d < D; d += kPlain) {
            const float g = (float)dy[r * dyr + d] * (w ? (float)w[d] : 1.0f);
            const float s = (float)x[r * xr + d] + (res ? (float)res[r * rr + d] : 0.0f);
            float v = inv * (g - s * inv * mean);
            if (ds) v += (float)ds[r * dsr + d];
            dx[r * D + d] = (T)v;
        }
    }
}

// partials[slab][d] = sum over the slab's rows of dy n
template <typename T>
__global__ __launch_bounds__(kPlain) void plain_weight_kernel(int64_t rows, int64_t D, int64_t slab,
                                                              const T* __restrict__ x, int64_t xr,
                                                              const T* __restrict__ res, int64_t rr,
                                                              const float* __restrict__ rstd,
                                                              const T* __restrict__ dy, int64_t dyr,
                                                              float* __restrict__ partials) {
    const int64_t d = (int64_t)blockIdx.x * kPlain + threadIdx.x;
    if (d >= D) return;
    const int64_t r0 = blockIdx.y * slab, r1 = r0 + slab < rows ? r0 + slab : rows;
    float acc = 0.0f;
    for (int64_t r = r0; r < r1; ++r) {
        const float s = (float)x[r * xr + d] + (res ? (float)res[r * rr + d] : 0.0f);
        acc += (float)dy[r * dyr + d] * (s * rstd[r]);
    }
    partials[blockIdx.y * D + d] = acc;
}

// Threads and elements a row takes. Forward: few threads with many loads each, so that rows up to 2048 need no
// barrier. Backward: 8 elements a thread, since a thread also holds the weight and its sums of them; with 16 the
// kernel took 135 registers, three waves a SIMD, and 123 us against 109 (16384 x 4096, bf16, without a residual).
struct Plan {
    int group, ept;      // group 1: the narrow kernels, 0: the plain ones
};

Plan plan_of(int64_t D, int64_t V, bool backward) {
    if (D < V) return {1, 0};
    if (D > 16384) return {0, 0};
    if (D <= 32) return {4, 8};
    if (D <= 128) return {16, 8};
    if (D <= 512) return {64, 8};
    if (D <= 1024) return backward ? Plan{128, 8} : Plan{64, 16};
    if (D <= 2048) return backward ? Plan{256, 8} : Plan{64, 32};
    if (D <= 4096) return backward ? Plan{512, 8} : Plan{256, 16};
    if (D <= 8192) return backward ? Plan{1024, 8} : Plan{512, 16};
    return {1024, 16};
}

template <bool BACKWARD, typename F>
void with_plan(const Plan& p, F&& fn) {
    using std::integral_constant;
    auto call = [&](auto g, auto n) {
        if (p.group == g && p.ept == n) fn(g, n);
    };
    call(integral_constant<int, 4>{}, integral_constant<int, 8>{});
    call(integral_constant<int, 16>{}, integral_constant<int, 8>{});
    call(integral_constant<int, 64>{}, integral_constant<int, 8>{});
    call(integral_constant<int, 1024>{}, integral_constant<int, 16>{});
    if constexpr (BACKWARD) {
        call(integral_constant<int, 128>{}, integral_constant<int, 8>{});
        call(integral_constant<int, 256>{}, integral_constant<int, 8>{});
        call(integral_constant<int, 512>{}, integral_constant<int, 8>{});
        call(integral_constant<int, 1024>{}, integral_constant<int, 8>{});
    } else {
        call(integral_constant<int, 64>{}, integral_constant<int, 16>{});
        call(integral_constant<int, 64>{}, integral_constant<int, 32>{});
        call(integral_constant<int, 256>{}, integral_constant<int, 16>{});
        call(integral_constant<int, 512>{}, integral_constant<int, 16>{});
    }
}

int64_t at_a_time(const Plan& p) { return p.group > 0 && p.group <= 64 ? 256 / p.group : 1; }

// Partial sums of the weight gradient: one for each workgroup of the backward pass.
int64_t partials_of(int64_t rows, const Plan& p) {
    const int64_t per = at_a_time(p), blocks = (rows + per - 1) / per;
    const int64_t most = kResident / (p.group <= 64 ? 256 : p.group);
    return blocks < most ? blocks : most;
}

}  // namespace

extern "C" {

int64_t swarm_residual_norm_workspace(int64_t rows, int64_t D) {
    if (rows < 0 || D < 1 || !sane(rows, D)) return SWARM_ERR_ARG;
    int64_t most = 0;
    for (int64_t V : {4, 8}) {
        const int64_t n = partials_of(rows, plan_of(D, V, true));
        if (n > most) most = n;
    }
    return most * D;
}

int32_t swarm_residual_norm_forward(int32_t dtype, int64_t rows, int64_t D, const void* x, int64_t x_row,
                                    const void* residual, int64_t res_row, const void* weight, float eps, void* y,
                                    void* stream_out, float* rstd, void* stream) {
    if (!known_type(dtype) || rows < 0 || D < 1 || !sane(rows, D) || !(eps >= 0.0f)) return SWARM_ERR_ARG;
    if (rows == 0) return SWARM_OK;
    const Plan plan = plan_of(D, dtype == SWARM_F32 ? 4 : 8, false);
    if (!x || !y || (residual && !stream_out) || x_row < 0 || res_row < 0) return SWARM_ERR_ARG;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    with_type(dtype, [&](auto e) {
        using E = decltype(e);
        const E *xp = static_cast<const E*>(x), *rp = static_cast<const E*>(residual);
        const E* wp = static_cast<const E*>(weight);
        E *yp = static_cast<E*>(y), *op = static_cast<E*>(stream_out);
        if (plan.group == 1) {
            const int64_t blocks = (rows + kNarrow - 1) / kNarrow;
            narrow_fwd_kernel<E><<<(unsigned)(blocks < 65536 ? blocks : 65536), kNarrow, 0, st>>>(
                rows, (int)D, xp, x_row, rp, res_row, wp, eps, yp, op, rstd);
            return;
        }
        if (plan.group == 0) {
            plain_fwd_kernel<E><<<(unsigned)(rows < 65536 ? rows : 65536), kPlain, 0, st>>>(rows, D, xp, x_row, rp, res_row,
                                                                                        wp, eps, yp, op, rstd);
            return;
        }
        with_plan<false>(plan, [&](auto g, auto n) {
            constexpr int G = decltype(g)::value, N = decltype(n)::value;
            using R = Row<E, G, N>;
            constexpr int64_t most = kLaunch / R::kThreads * R::kRows;      // rows of a launch
            for (int64_t r = 0; r < rows; r += most) {
                const int64_t part = rows - r < most ? rows - r : most;
                norm_fwd_kernel<E, G, N><<<(unsigned)((part + R::kRows - 1) / R::kRows), R::kThreads, 0, st>>>(
                    part, D, xp + r * x_row, x_row, rp ? rp + r * res_row : nullptr, res_row, wp, eps, yp + r * D,
                    op ? op + r * D : nullptr, rstd ? rstd + r : nullptr);
            }
        });
    });
    return swarm::record_hip_status();
}

int32_t swarm_residual_norm_backward(int32_t dtype, int64_t rows, int64_t D, const void* x, int64_t x_row,
                                     const void* residual, int64_t res_row, const void* weight, const float* rstd,
                                     const void* d_y, int64_t dy_row, const void* d_stream, int64_t ds_row, void* d_x,
                                     void* d_weight, float* work, void* stream) {
    if (!known_type(dtype) || rows < 0 || D < 1 || !sane(rows, D)) return SWARM_ERR_ARG;
    const int64_t cols = (D + kFinishCols - 1) / kFinishCols;
    if (d_weight && ((rows > 0 && !work) || cols > kLaunch / kFinish)) return SWARM_ERR_ARG;
    if (rows == 0 && !d_weight) return SWARM_OK;
    if (rows > 0 && (!x || !rstd || !d_y || !d_x || x_row < 0 || res_row < 0 || dy_row < 0 || ds_row < 0)) return SWARM_ERR_ARG;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    const Plan plan = plan_of(D, dtype == SWARM_F32 ? 4 : 8, true);
    int64_t count = partials_of(rows, plan);
    with_type(dtype, [&](auto e) {
        using E = decltype(e);
        const E *xp = static_cast<const E*>(x), *rp = static_cast<const E*>(residual);
        const E *wp = static_cast<const E*>(weight), *yp = static_cast<const E*>(d_y);
        const E* dp = static_cast<const E*>(d_stream);
        E* out = static_cast<E*>(d_x);
        float* partials = d_weight ? work : nullptr;
        if (rows > 0 && plan.group == 1) {
            narrow_bwd_kernel<E><<<(unsigned)count, kNarrow, 0, st>>>(rows, (int)D, xp, x_row, rp, res_row, wp, rstd, yp,
                                                                     dy_row, dp, ds_row, out, partials);
        } else if (rows > 0 && plan.group == 0) {
            plain_bwd_kernel<E><<<(unsigned)(rows < 65536 ? rows : 65536), kPlain, 0, st>>>(rows, D, xp, x_row, rp, res_row,
                                                                                        wp, rstd, yp, dy_row, dp, ds_row, out);
            const int64_t slab = (rows + count - 1) / count;
            count = (rows + slab - 1) / slab;
            if (d_weight)
                plain_weight_kernel<E><<<dim3((unsigned)((D + kPlain - 1) / kPlain), (unsigned)count), kPlain, 0, st>>>(
                    rows, D, slab, xp, x_row, rp, res_row, rstd, yp, dy_row, work);
        } else if (rows > 0) {
            with_plan<true>(plan, [&](auto g, auto n) {
                constexpr int G = decltype(g)::value, N = decltype(n)::value;
                using R = Row<E, G, N>;
                const size_t lds = partials && R::kRows > 1 ? R::kRows * (size_t)D * sizeof(float) : 0;
                norm_bwd_kernel<E, G, N><<<(unsigned)count, R::kThreads, lds, st>>>(rows, D, xp, x_row, rp, res_row, wp, rstd,
                                                                                  yp, dy_row, dp, ds_row, out, partials);
            });
        }
        if (d_weight)
            weight_finish_kernel<E><<<(unsigned)cols, kFinish, 0, st>>>(count, D, work, static_cast<E*>(d_weight));
    });
    return swarm::record_hip_status();
}

}  // extern "C"
