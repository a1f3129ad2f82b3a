// swarm_gated.hip — gated linear recurrence (include/swarmseq.h: swarm_gated_scan_*, swarm_gated_step).
//
//   c_t = f_t p_t + (1 - f_t) z_t,  p_t = keep_{t-1} c_{t-1},  h_t = o_t c_t,  f, o = sigmoid of their gates.
// With a_t = f_t keep_{t-1} the gradient E_t of p_t (times keep: of c_{t-1}) runs the same recurrence backwards:
//   D_t = o_t dh_t + E_{t+1},  E_t = a_t D_t,
//   d xf = D (p - z) f (1 - f),  d xz = D (1 - f),  d xo = dh c o (1 - o),  d c0 = E_0.
// Padding steps are the identity: a = 1, nothing added, zero outputs.
#include "swarm_seq.h"

using namespace swarm_seq;

namespace {

constexpr int kThreads = 256;

template <typename T>
__global__ __launch_bounds__(kThreads) void scan_fwd_kernel(int64_t n, int64_t steps, int64_t U, const T* __restrict__ gates,
                                                            int64_t gn, int64_t gt, const float* __restrict__ c0,
                                                            const float* __restrict__ keep,
                                                            const int64_t* __restrict__ lengths, T* __restrict__ h,
                                                            float* __restrict__ c_last, float* __restrict__ states) {
    const int64_t id = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    if (id >= n * U) return;
    const int64_t i = id / U, u = id - i * U;
    const int64_t len = lengths ? lengths[i] : steps;
    float c = c0 ? c0[id] : 0.0f;
    for (int64_t t = 0; t < steps; ++t) {
        if (states) states[(i * steps + t) * U + u] = c;
        float out = 0.0f;
        if (t < len) {
            const T* g = gates + i * gn + t * gt + u;
            float f, b;
            sigmoid_pair((float)g[0], f, b);
            const float p = (keep && t > 0) ? c * keep[i * steps + t - 1] : c;
            c = f * p + b * (float)g[U];
            out = sigmoid((float)g[2 * U]) * c;
        }
        h[(i * steps + t) * U + u] = (T)out;
    }
    c_last[id] = c;
}

template <typename T>
__global__ __launch_bounds__(kThreads) void scan_bwd_kernel(int64_t n, int64_t steps, int64_t U, const T* __restrict__ gates,
                                                            int64_t gn, int64_t gt, const float* __restrict__ keep,
                                                            const int64_t* __restrict__ lengths,
                                                            const float* __restrict__ states, const T* __restrict__ dh,
                                                            int64_t dn, int64_t dt, const float* __restrict__ d_last,
                                                            T* __restrict__ dg, float* __restrict__ d_c0) {
    const int64_t id = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    if (id >= n * U) return;
    const int64_t i = id / U, u = id - i * U;
    const int64_t len = lengths ? lengths[i] : steps;
    float E = d_last ? d_last[id] : 0.0f;
    for (int64_t t = steps - 1; t >= 0; --t) {
        float df = 0.0f, dz = 0.0f, dO = 0.0f;
        if (t < len) {
            const T* g = gates + i * gn + t * gt + u;
            float f, b, o, ob;
            sigmoid_pair((float)g[0], f, b);
            const float z = (float)g[U];
            sigmoid_pair((float)g[2 * U], o, ob);
            const float k = (keep && t > 0) ? keep[i * steps + t - 1] : 1.0f;
            const float p = states[(i * steps + t) * U + u] * k;
            const float c = f * p + b * z;
            const float d = dh ? (float)dh[i * dn + t * dt + u] : 0.0f;
            const float D = o * d + E;
            df = D * (p - z) * f * b;
            dz = D * b;
            dO = d * c * o * ob;
            E = f * k * D;
        }
        T* out = dg + (i * steps + t) * 3 * U + u;
        out[0] = (T)df;
        out[U] = (T)dz;
        out[2 * U] = (T)dO;
    }
    if (d_c0) d_c0[id] = E;
}

template <typename T>
__global__ __launch_bounds__(kThreads) void step_kernel(int64_t rows, int64_t U, const T* __restrict__ gates, int64_t gr,
                                                        const float* c, const float* __restrict__ keep,
                                                        T* __restrict__ h, float* c_out) {
    const int64_t id = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    if (id >= rows * U) return;
    const int64_t i = id / U, u = id - i * U;
    const T* g = gates + i * gr + u;
    float f, b;
    sigmoid_pair((float)g[0], f, b);
    const float p = keep ? c[id] * keep[i] : c[id];
    const float now = f * p + b * (float)g[U];
    c_out[id] = now;
    h[id] = (T)(sigmoid((float)g[2 * U]) * now);
}

bool blocks_of(int64_t items, unsigned& blocks) {
    const int64_t b = (items + kThreads - 1) / kThreads;
    blocks = (unsigned)b;
    return b <= 0x7fffffff;
}

}  // namespace

extern "C" {

int64_t swarm_gated_scan_workspace(int64_t, int64_t, int64_t) { return 0; }

int32_t swarm_gated_scan_forward(int32_t dtype, int64_t n, int64_t T, int64_t U, const void* gates, int64_t gates_n,
                                 int64_t gates_t, const float* c0, const float* keep, const int64_t* lengths, void* h,
                                 float* c_last, float* tile_states, float* work, void* stream) {
    (void)work;
    if (!known_type(dtype) || n < 0 || T < 1 || U < 1 || !sane(n, T, U)) return SWARM_ERR_ARG;
    if (n == 0) return SWARM_OK;
    unsigned blocks;
    if (!gates || !h || !c_last || gates_t < 0 || gates_n < 0 || !blocks_of(n * U, blocks)) return SWARM_ERR_ARG;
    with_type(dtype, [&](auto e) {
        using E = decltype(e);
        scan_fwd_kernel<E><<<blocks, kThreads, 0, static_cast<hipStream_t>(stream)>>>(
            n, T, U, static_cast<const E*>(gates), gates_n, gates_t, c0, keep, lengths, static_cast<E*>(h), c_last,
            tile_states);
    });
    return swarm::record_hip_status();
}

int32_t swarm_gated_scan_backward(int32_t dtype, int64_t n, int64_t T, int64_t U, const void* gates, int64_t gates_n,
                                  int64_t gates_t, const float* keep, const int64_t* lengths,
                                  const float* tile_states, const void* d_h, int64_t d_h_n, int64_t d_h_t,
                                  const float* d_last, void* d_gates, float* d_c0, float* work, void* stream) {
    (void)work;
    if (!known_type(dtype) || n < 0 || T < 1 || U < 1 || !sane(n, T, U)) return SWARM_ERR_ARG;
    if (n == 0) return SWARM_OK;
    unsigned blocks;
    if (!gates || !tile_states || !d_gates || gates_t < 0 || gates_n < 0 || d_h_n < 0 || d_h_t < 0 ||
        !blocks_of(n * U, blocks))
        return SWARM_ERR_ARG;
    with_type(dtype, [&](auto e) {
        using E = decltype(e);
        scan_bwd_kernel<E><<<blocks, kThreads, 0, static_cast<hipStream_t>(stream)>>>(
            n, T, U, static_cast<const E*>(gates), gates_n, gates_t, keep, lengths, tile_states,
            static_cast<const E*>(d_h), d_h_n, d_h_t, d_last, static_cast<E*>(d_gates), d_c0);
    });
    return swarm::record_hip_status();
}

int32_t swarm_gated_step(int32_t dtype, int64_t rows, int64_t U, const void* gates, int64_t gates_row, const float* c,
                         const float* keep, void* h, float* c_out, void* stream) {
    if (!known_type(dtype) || rows < 0 || U < 1 || !sane(rows, U)) return SWARM_ERR_ARG;
    if (rows == 0) return SWARM_OK;
    unsigned blocks;
    if (!gates || !c || !h || !c_out || gates_row < 0 || !blocks_of(rows * U, blocks)) return SWARM_ERR_ARG;
    with_type(dtype, [&](auto e) {
        using E = decltype(e);
        step_kernel<E><<<blocks, kThreads, 0, static_cast<hipStream_t>(stream)>>>(
            rows, U, static_cast<const E*>(gates), gates_row, c, keep, static_cast<E*>(h), c_out);
    });
    return swarm::record_hip_status();
}

}  // extern "C"
