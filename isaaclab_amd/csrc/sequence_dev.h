// What the sequence kernels share: element types, their conversions, and the scalar functions of a gate and a step size.
#pragma once

#include "common.h"

#include "../../include/isaaclab_amd_sequence.h"

namespace ilx {

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

template <typename T> __device__ __forceinline__ float to_f32(T v) { return static_cast<float>(v); }
template <typename T> __device__ __forceinline__ T from_f32(float v) { return static_cast<T>(v); }   // to nearest, ties to even

constexpr float kLog2e = 1.44269504088896340736f;

// e^x and 1/x on the hardware's exponential and reciprocal (1 ulp each; the product with log2 e adds |x| 2^-24 relative).
__device__ __forceinline__ float exp_fast(float x) { return __builtin_amdgcn_exp2f(x * kLog2e); }
__device__ __forceinline__ float rcp_fast(float x) { return __builtin_amdgcn_rcpf(x); }

__device__ __forceinline__ float sigmoid_fast(float x) { return rcp_fast(1.0f + exp_fast(-x)); }

// log(1 + e^x) = max(x, 0) + log1p(e^-|x|), the second term as 2 artanh(s), s = e / (2 + e) with e in (0, 1] (a logarithm of 1 + e
// would lose e's last bits, which for a step size of 1e-4 are all it has).  s is at most 1/3; the polynomial in s^2 is the one of degree
// 4 with the least largest relative error on [0, 1/9], 2^-27.9.  Relative error in units of 2^-24: at most 9 for x >= 0 and 9 + 1.3 |x|
// below (|x| from the product with log2 e and a quarter of it from log2 e itself; exponential and reciprocal 2 each, five roundings).
// Measured: 4 above -1, 10 down to -10, 32 down to -40.
__device__ __forceinline__ float softplus_f(float x) {
    const float e = exp_fast(-__builtin_fabsf(x));
    const float s = e * rcp_fast(2.0f + e), q = s * s;
    float p = 0.281783342f;
    p = __builtin_fmaf(p, q, 0.279606014f);
    p = __builtin_fmaf(p, q, 0.400249094f);
    p = __builtin_fmaf(p, q, 0.66666317f);
    p = __builtin_fmaf(p, q, 2.0f);
    return __builtin_fmaf(p, s, __builtin_fmaxf(x, 0.0f));   // (a NaN comes through e)
}

// V elements on their own boundary, up to 16 bytes.
template <typename T, int V> struct alignas(sizeof(T) * V < 16 ? sizeof(T) * V : 16) Pack { T v[V]; };

// V neighbouring channels of one row, as one load or store of up to 16 bytes on any element's boundary (the chip reads and writes
// global memory unaligned).
template <typename T, int V> struct __attribute__((packed, aligned(sizeof(T)))) Channels { T v[V]; };

template <int V, typename T> __device__ __forceinline__ void load_channels(const T* p, float (&v)[V]) {
    const Channels<T, V> w = *reinterpret_cast<const Channels<T, V>*>(p);
#pragma unroll
    for (int k = 0; k < V; ++k) v[k] = to_f32(w.v[k]);
}
template <int V, typename T> __device__ __forceinline__ void store_channels(T* p, const float (&v)[V]) {
    Channels<T, V> w;
#pragma unroll
    for (int k = 0; k < V; ++k) w.v[k] = from_f32<T>(v[k]);
    *reinterpret_cast<Channels<T, V>*>(p) = w;
}

constexpr int64_t kMostThreads = (int64_t{1} << 32) - 1024;   // of one launch
constexpr int32_t kMostChannels = 1 << 23;

inline bool aligned_to(const void* p, size_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

// Rows that one thread's or wave's sums of a parameter's gradient span in 32 bits: n adds are off by up to n 2^-24 of their terms'
// magnitudes, so a longer chain ends in another row of partial sums, and those are added in 64 bits.
constexpr int kChainRows = 512;

// The end of a parameter's gradient: `count` rows of (n0 + extra) x channels partial sums, one row per workgroup that kept
// some, are added in a fixed order, in 64 bits.  Value k of channel d goes to out0[d, k] for k < n0, then out1[d], out2[d];
// outputs that are NULL are left out.
void launch_parameter_sums(const float* partial, int64_t count, int32_t channels, int32_t n0, int32_t extra, float* out0, float* out1, float* out2,
                           hipStream_t stream);

}  // namespace ilx
