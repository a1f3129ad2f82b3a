// swarm_seq.h — element types and small helpers of the sequence-policy kernels (include/swarmseq.h).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "../../include/swarmseq.h"
#include "../../include/swarmstep.h"
#include "swarm_launch.h"

namespace swarm_seq {

using f32 = float;
using bf16 = __bf16;
using f16 = _Float16;

constexpr int64_t kLaunch = 0xffffffff;      // threads of a launch, at most: a grid's size is counted in threads

constexpr float kLog2e = 1.44269504088896340736f;

constexpr float kLn2 = 0.69314718055994530942f;

// exp(y) from h = y log2 e, rounded: 2^h alone is off by |y| 2^-24 relative, since h is; d = y - h ln 2, formed in one
// rounding, is what it left out.
__device__ __forceinline__ float exp_from(float h, float d) {
    const float e = __builtin_amdgcn_exp2f(h);
    return __builtin_fmaf(e, d, e);
}

// Element types whose own rounding does not cover that error. (Bounded by memory in float32, where it costs nothing:
// 32 x 1000 x 2048, backward 391 us either way. In 16 bits 1 x 32768 x 1024 took 104 + 161 us forward and backward with it
// against 98 + 151 without, for errors far below the gates' own steps.)
template <typename T>
constexpr bool kExact = sizeof(T) == 4;

// sigmoid(x) and 1 - sigmoid(x) = e s with e = exp(-x), which keeps the small side exact: in float32 both are good to
// 7 + |x| / 20 units of 2^-24, else to 6 + 2 |x|. e is held below 2^126, with its remainder too: the reciprocal of more
// is no normal number and becomes 0, and e s with it; the sigmoid stays at 1.3e-38 there. An infinite x, or one beyond
// that bound, would leave no number in the remainder, which is below 2^-16 elsewhere; a NaN stays one.
template <typename T>
__device__ __forceinline__ void sigmoid_pair(float x, float& s, float& one_minus) {
    const float h = __builtin_elementwise_minimum(x * -kLog2e, 125.9f);
    const float e = kExact<T> ? exp_from(h, __builtin_amdgcn_fmed3f(__builtin_fmaf(h, -kLn2, -x), -0x1p-16f, 0x1p-16f))
                              : __builtin_amdgcn_exp2f(h);
    s = __builtin_amdgcn_rcpf(1.0f + e);
    one_minus = e * s;
}

template <typename T>
__device__ __forceinline__ float sigmoid(float x) {
    if constexpr (kExact<T>) {
        float s, rest;
        sigmoid_pair<T>(x, s, rest);
        return s;
    }
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(x * -kLog2e));
}

// N elements at any address, held as words (a 16-bit element in a register of its own would double what a tile
// takes). Global loads and stores of up to 16 bytes need no alignment on gfx950, so rows of odd width and
// unaligned views take the same path as aligned ones.
template <typename T, int N = 16 / sizeof(T)>
struct Pack {
    static constexpr int kWords = (N * (int)sizeof(T) + 3) / 4;
    uint32_t w[kWords];

    __device__ __forceinline__ void load(const T* __restrict__ p) {
        w[kWords - 1] = 0u;
        __builtin_memcpy(w, p, N * sizeof(T));
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int k = 0; k < kWords; ++k) w[k] = 0u;
    }
    __device__ __forceinline__ void store(T* __restrict__ p) const { __builtin_memcpy(p, w, N * sizeof(T)); }

    __device__ __forceinline__ float get(int j) const {
        if constexpr (sizeof(T) == 4) {
            return __builtin_bit_cast(float, w[j]);
        } else if constexpr (__is_same(T, bf16)) {
            return __builtin_bit_cast(float, j & 1 ? w[j / 2] & 0xffff0000u : w[j / 2] << 16);
        } else {
            return (float)__builtin_bit_cast(f16, (uint16_t)(j & 1 ? w[j / 2] >> 16 : w[j / 2] & 0xffffu));
        }
    }
    // rounds to nearest even
    __device__ __forceinline__ void set(const float (&v)[N]) {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int j = 0; j < N; ++j) w[j] = __builtin_bit_cast(uint32_t, v[j]);
        } else {
            typedef float F2 __attribute__((ext_vector_type(2)));
            typedef T T2 __attribute__((ext_vector_type(2)));
#pragma unroll
            for (int j = 0; j < N; j += 2)
                w[j / 2] = __builtin_bit_cast(uint32_t, __builtin_convertvector((F2{v[j], j + 1 < N ? v[j + 1 < N ? j + 1 : j] : 0.0f}), T2));
        }
    }
};

// op over groups of GROUP <= 64 consecutive lanes, in every lane: within 16 by DPP moves, then the 16- and 32-lane
// swaps, none of which goes through LDS.
template <int GROUP, typename Op>
__device__ __forceinline__ float lanes_reduce(float v, Op&& op) {
    static_assert(GROUP <= 64 && (GROUP & (GROUP - 1)) == 0, "a power of two");
    auto moved = [&](auto ctrl) {
        const int w = __builtin_bit_cast(int, v);
        return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(w, w, decltype(ctrl)::value, 0xf, 0xf, false));
    };
    if constexpr (GROUP >= 2) v = op(v, moved(std::integral_constant<int, 0xB1>{}));     // neighbours
    if constexpr (GROUP >= 4) v = op(v, moved(std::integral_constant<int, 0x4E>{}));     // pairs of a quad
    if constexpr (GROUP >= 8) v = op(v, moved(std::integral_constant<int, 0x141>{}));    // quads of 8, mirrored
    if constexpr (GROUP >= 16) v = op(v, moved(std::integral_constant<int, 0x140>{}));   // halves of 16, mirrored
    if constexpr (GROUP >= 32) {
        const uint32_t w = __builtin_bit_cast(uint32_t, v);
        const auto r = __builtin_amdgcn_permlane16_swap(w, w, false, false);
        const uint32_t one = r[0], other = r[1];      // __builtin_bit_cast of r[1] itself reads r[0]
        v = op(__builtin_bit_cast(float, one), __builtin_bit_cast(float, other));
    }
    if constexpr (GROUP >= 64) {
        const uint32_t w = __builtin_bit_cast(uint32_t, v);
        const auto r = __builtin_amdgcn_permlane32_swap(w, w, false, false);
        const uint32_t one = r[0], other = r[1];      // __builtin_bit_cast of r[1] itself reads r[0]
        v = op(__builtin_bit_cast(float, one), __builtin_bit_cast(float, other));
    }
    return v;
}

struct Add {
    __device__ __forceinline__ float operator()(float a, float b) const { return a + b; }
};

// the larger one, or a NaN
struct Maximum {
    __device__ __forceinline__ float operator()(float a, float b) const { return __builtin_elementwise_maximum(a, b); }
};

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
