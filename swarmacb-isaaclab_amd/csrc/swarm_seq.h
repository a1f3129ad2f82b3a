// swarm_seq.h — element types and small helpers of the sequence-policy kernels (include/swarmseq.h).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/swarmseq.h"
#include "../../include/swarmstep.h"
#include "swarm_launch.h"

namespace swarm_seq {

using f32 = float;
using bf16 = __bf16;
using f16 = _Float16;

constexpr float kLog2e = 1.44269504088896340736f;

// sigmoid(x) and 1 - sigmoid(x), both to a few units in the last place: e = exp(-x) stays finite (x is
// held above -87, where the sigmoid is 1e-38) and 1 - s = e s keeps the small side exact.
__device__ __forceinline__ void sigmoid_pair(float x, float& s, float& one_minus) {
    // not fmaxf: a NaN has to stay one
    const float e = __builtin_amdgcn_exp2f((x < -87.0f ? -87.0f : x) * -kLog2e);
    s = __builtin_amdgcn_rcpf(1.0f + e);
    one_minus = e * s;
}

__device__ __forceinline__ float sigmoid(float x) {
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f((x < -87.0f ? -87.0f : x) * -kLog2e));
}

// 16 bytes of elements at any address: global loads and stores of 16 bytes need no alignment on gfx950, so rows
// of odd width and unaligned views take the same path. `valid` < V at the end of a row goes element by element.
template <typename T>
struct Pack {
    static constexpr int V = 16 / sizeof(T);
    T e[V];
};

template <typename T>
__device__ __forceinline__ Pack<T> load_pack(const T* __restrict__ p, int valid) {
    Pack<T> r;
    if (valid >= Pack<T>::V) {
        __builtin_memcpy(&r, p, 16);
    } else {
#pragma unroll
        for (int j = 0; j < Pack<T>::V; ++j) r.e[j] = j < valid ? p[j] : (T)0.0f;
    }
    return r;
}

template <typename T>
__device__ __forceinline__ void store_pack(T* __restrict__ p, const Pack<T>& v, int valid) {
    if (valid >= Pack<T>::V) {
        __builtin_memcpy(p, &v, 16);
    } else {
#pragma unroll
        for (int j = 0; j < Pack<T>::V; ++j)
            if (j < valid) p[j] = v.e[j];
    }
}

// Calls fn with a value of the element type that `dtype` names; false for an unknown dtype.
template <typename F>
bool with_type(int32_t dtype, F&& fn) {
    switch (dtype) {
        case SWARM_F32: fn(f32{}); return true;
        case SWARM_BF16: fn(bf16{}); return true;
        case SWARM_F16: fn(f16{}); return true;
    }
    return false;
}

inline bool known_type(int32_t dtype) { return dtype == SWARM_F32 || dtype == SWARM_BF16 || dtype == SWARM_F16; }

// Largest element count of any operand: byte offsets stay far inside 63 bits.
constexpr int64_t kMaxElements = int64_t(1) << 48;

inline bool sane(int64_t a, int64_t b, int64_t c = 1) {
    if (a < 0 || b < 0 || c < 0) return false;
    if (a == 0 || b == 0 || c == 0) return true;
    return a <= kMaxElements / b && a * b <= kMaxElements / c;
}

}  // namespace swarm_seq
