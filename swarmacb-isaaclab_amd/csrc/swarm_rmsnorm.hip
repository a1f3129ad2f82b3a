// swarm_rmsnorm.hip — root-mean-square norm of a residual sum (include/swarmseq.h: swarm_residual_norm_*).
//
//   s = x + r,  rstd = (mean(s^2) + eps)^-1/2,  n = s rstd,  y = n w
//   d_x = d_r = rstd (w dy - n mean(w dy n)) + d_stream,   d_w = sum over rows of dy n
#include "swarm_seq.h"

using namespace swarm_seq;

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int64_t kSlabs = 512;   // row slabs of the weight gradient's partial sums

// the sum of v over the workgroup, in every thread
__device__ __forceinline__ float block_sum(float v, float* red) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    float s = 0.0f;
    for (int k = 0; k < kWaves; ++k) s += red[k];
    return s;
}

template <typename T>
__global__ __launch_bounds__(kThreads) void norm_fwd_kernel(int64_t rows, int64_t D, const T* __restrict__ x, int64_t xr,
                                                            const T* __restrict__ res, int64_t rr,
                                                            const T* __restrict__ w, float eps, T* __restrict__ y,
                                                            T* __restrict__ out, float* __restrict__ rstd) {
    __shared__ float red[kWaves];
    for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
        float ss = 0.0f;
        for (int64_t d = threadIdx.x; d < D; d += kThreads) {
            const float s = (float)x[r * xr + d] + (res ? (float)res[r * rr + d] : 0.0f);
            ss += s * s;
        }
        const float inv = 1.0f / sqrtf(block_sum(ss, red) / (float)D + eps);
        for (int64_t d = threadIdx.x; d < D; d += kThreads) {
            const float s = (float)x[r * xr + d] + (res ? (float)res[r * rr + d] : 0.0f);
            if (res) out[r * D + d] = (T)s;
            y[r * D + d] = (T)(s * inv * (w ? (float)w[d] : 1.0f));
        }
        if (rstd && threadIdx.x == 0) rstd[r] = inv;
    }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void norm_bwd_kernel(int64_t rows, int64_t D, const T* __restrict__ s, int64_t sr,
                                                            const T* __restrict__ w, const float* __restrict__ rstd,
                                                            const T* __restrict__ dy, int64_t dyr,
                                                            const T* __restrict__ ds, int64_t dsr,
                                                            T* __restrict__ dx) {
    __shared__ float red[kWaves];
    for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
        const float inv = rstd[r];
        float dot = 0.0f;
        for (int64_t d = threadIdx.x; d < D; d += kThreads)
            dot += (float)dy[r * dyr + d] * (w ? (float)w[d] : 1.0f) * ((float)s[r * sr + d] * inv);
        const float mean = block_sum(dot, red) / (float)D;
        for (int64_t d = threadIdx.x; d < D; d += kThreads) {
            const float g = (float)dy[r * dyr + d] * (w ? (float)w[d] : 1.0f);
            float v = inv * (g - (float)s[r * sr + d] * inv * mean);
            if (ds) v += (float)ds[r * dsr + d];
            dx[r * D + d] = (T)v;
        }
    }
}

// partials[slab][d] = sum over the slab's rows of dy n
template <typename T>
__global__ __launch_bounds__(kThreads) void weight_partial_kernel(int64_t rows, int64_t D, int64_t slab,
                                                                  const T* __restrict__ s, int64_t sr,
                                                                  const float* __restrict__ rstd,
                                                                  const T* __restrict__ dy, int64_t dyr,
                                                                  float* __restrict__ partials) {
    const int64_t d = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    if (d >= D) return;
    const int64_t r0 = blockIdx.y * slab, r1 = r0 + slab < rows ? r0 + slab : rows;
    float acc = 0.0f;
    for (int64_t r = r0; r < r1; ++r) acc += (float)dy[r * dyr + d] * ((float)s[r * sr + d] * rstd[r]);
    partials[blockIdx.y * D + d] = acc;
}

template <typename T>
__global__ __launch_bounds__(kThreads) void weight_finish_kernel(int64_t slabs, int64_t D,
                                                                 const float* __restrict__ partials,
                                                                 T* __restrict__ dw) {
    const int64_t d = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    if (d >= D) return;
    float acc = 0.0f;
    for (int64_t k = 0; k < slabs; ++k) acc += partials[k * D + d];
    dw[d] = (T)acc;
}

void slabs_of(int64_t rows, int64_t& slab, int64_t& slabs) {
    slab = (rows + kSlabs - 1) / kSlabs;
    slabs = slab ? (rows + slab - 1) / slab : 0;
}

}  // namespace

extern "C" {

int64_t swarm_residual_norm_workspace(int64_t rows, int64_t D) {
    if (rows < 0 || D < 1 || !sane(rows, D)) return SWARM_ERR_ARG;
    int64_t slab, slabs;
    slabs_of(rows, slab, slabs);
    return slabs * D;
}

int32_t swarm_residual_norm_forward(int32_t dtype, int64_t rows, int64_t D, const void* x, int64_t x_row,
                                    const void* residual, int64_t res_row, const void* weight, float eps, void* y,
                                    void* stream_out, float* rstd, void* stream) {
    if (!known_type(dtype) || rows < 0 || D < 1 || !sane(rows, D) || !(eps >= 0.0f)) return SWARM_ERR_ARG;
    if (rows == 0) return SWARM_OK;
    if (!x || !y || (residual && !stream_out) || x_row < 0 || res_row < 0) return SWARM_ERR_ARG;
    const unsigned blocks = (unsigned)(rows < 65536 ? rows : 65536);
    with_type(dtype, [&](auto e) {
        using E = decltype(e);
        norm_fwd_kernel<E><<<blocks, kThreads, 0, static_cast<hipStream_t>(stream)>>>(
            rows, D, static_cast<const E*>(x), x_row, static_cast<const E*>(residual), res_row,
            static_cast<const E*>(weight), eps, static_cast<E*>(y), static_cast<E*>(stream_out), rstd);
    });
    return swarm::record_hip_status();
}

int32_t swarm_residual_norm_backward(int32_t dtype, int64_t rows, int64_t D, const void* sum, int64_t sum_row,
                                     const void* weight, const float* rstd, const void* d_y, int64_t dy_row,
                                     const void* d_stream, int64_t ds_row, void* d_x, void* d_weight, float* work,
                                     void* stream) {
    if (!known_type(dtype) || rows < 0 || D < 1 || !sane(rows, D) || D > 0x7fffffffLL * kThreads) return SWARM_ERR_ARG;
    if (d_weight && rows > 0 && !work) return SWARM_ERR_ARG;
    if (rows == 0 && !d_weight) return SWARM_OK;
    if (rows > 0 && (!sum || !rstd || !d_y || !d_x || sum_row < 0 || dy_row < 0 || ds_row < 0)) return SWARM_ERR_ARG;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    const unsigned blocks = (unsigned)(rows < 65536 ? rows : 65536);
    const unsigned cols = (unsigned)((D + kThreads - 1) / kThreads);
    int64_t slab, slabs;
    slabs_of(rows, slab, slabs);
    with_type(dtype, [&](auto e) {
        using E = decltype(e);
        if (rows > 0)
            norm_bwd_kernel<E><<<blocks, kThreads, 0, st>>>(
                rows, D, static_cast<const E*>(sum), sum_row, static_cast<const E*>(weight), rstd,
                static_cast<const E*>(d_y), dy_row, static_cast<const E*>(d_stream), ds_row, static_cast<E*>(d_x));
        if (!d_weight) return;
        if (rows > 0)
            weight_partial_kernel<E><<<dim3(cols, (unsigned)slabs), kThreads, 0, st>>>(
                rows, D, slab, static_cast<const E*>(sum), sum_row, rstd, static_cast<const E*>(d_y), dy_row, work);
        weight_finish_kernel<E><<<cols, kThreads, 0, st>>>(slabs, D, work, static_cast<E*>(d_weight));
    });
    return swarm::record_hip_status();
}

}  // extern "C"
