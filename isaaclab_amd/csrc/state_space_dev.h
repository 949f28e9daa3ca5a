// What the state space kernels share: their arguments, the split of channels over workgroups, and the wave-uniform reads
// of B and C.
#pragma once

#include "sequence_dev.h"

namespace ilx {

struct ScanArgs {
    ilx_state_space s;
    int group_channels;  // channels / groups
    int group_blocks;    // blocks of 64 channels per group
    int blocks;          // groups * group_blocks
    int64_t saved_blocks;  // blocks of ILX_SCAN_BLOCK rows per sequence
    int64_t slots;         // backward, step: workgroups per block of channels
    float* sums;           // backward: (slots, states + 2, channels) partial sums of dA, dD and d delta_bias
    float* shared;         // backward: (group_blocks, batch, length, groups, 2 * padded states) partial sums of dB, dC
};

// A wave holds 64 channels of one group, a lane each; lanes past the group's end repeat its last channel and store nothing.
struct ChannelLane {
    int group, d;
    bool active;
};
__device__ __forceinline__ ChannelLane channel_lane(const ScanArgs& a, int block, int lane) {
    ChannelLane c;
    c.group = block / a.group_blocks;
    const int within = (block - c.group * a.group_blocks) * 64 + lane;
    c.active = within < a.group_channels;
    c.d = c.group * a.group_channels + (c.active ? within : a.group_channels - 1);
    return c;
}

__device__ __forceinline__ int64_t scan_length(const ilx_state_space& s, int64_t b) {
    if (!s.lengths) return s.length;
    const int64_t n = s.lengths[b];
    return n < 0 ? 0 : (n > s.length ? s.length : n);
}

// B or C of one row, the states n0 .. n0 + S - 1 (zeros past the last): the same for all lanes, so it is read through the
// scalar cache and enters the arithmetic as scalar operands.  16-bit pairs are split by scalar instructions.
template <typename T> struct UniformWord { typedef float type; };
template <> struct UniformWord<bf16_t> { typedef uint32_t type; };
template <> struct UniformWord<f16_t> { typedef uint32_t type; };

template <int S, bool FULL> __device__ __forceinline__ void load_uniform(const float* row, int n0, int states, float (&v)[S]) {
    typedef const float __attribute__((address_space(4))) * Ptr;
    const Ptr p = (Ptr)(row);
#pragma unroll
    for (int i = 0; i < S; ++i) {
        if (FULL)
            v[i] = p[n0 + i];
        else
            v[i] = n0 + i < states ? p[n0 + i < states ? n0 + i : states - 1] : 0.0f;
    }
}
__device__ __forceinline__ float low_half(uint32_t w, bf16_t) { return __builtin_bit_cast(float, w << 16); }
__device__ __forceinline__ float high_half(uint32_t w, bf16_t) { return __builtin_bit_cast(float, w & 0xffff0000u); }
__device__ __forceinline__ float low_half(uint32_t w, f16_t) {
    return static_cast<float>(__builtin_bit_cast(f16_t, static_cast<uint16_t>(w)));
}
__device__ __forceinline__ float high_half(uint32_t w, f16_t) {
    return static_cast<float>(__builtin_bit_cast(f16_t, static_cast<uint16_t>(w >> 16)));
}
template <int S, bool FULL, typename T> __device__ __forceinline__ void load_uniform(const T* row, int n0, int states, float (&v)[S]) {
    typedef const uint32_t __attribute__((address_space(4))) * Ptr;
    const Ptr p = (Ptr)(row);
#pragma unroll
    for (int i = 0; i < S; i += 2) {   // (states is even: a pair is inside or outside)
        const bool in = FULL || n0 + i < states;
        const uint32_t w = p[(in ? n0 + i : states - 2) >> 1];
        v[i] = in ? low_half(w, T()) : 0.0f;
        v[i + 1] = in ? high_half(w, T()) : 0.0f;
    }
}

// Bit i: an episode begins at row t0 + i (i < count <= 64).
__device__ __forceinline__ uint64_t start_bits(const ilx_state_space& s, int64_t b, int64_t t0, int count, int lane) {
    if (!s.starts) return 0;
    bool on = false;
    if (lane < count) on = s.starts[b * s.starts_batch + (t0 + lane) * s.starts_time] != 0;
    return __ballot(on);
}

int scan_check(const ilx_state_space& s, const char* name);
ScanArgs scan_args(const ilx_state_space& s);

}  // namespace ilx
