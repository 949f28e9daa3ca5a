// What the state space kernels share: their arguments, the split of channels over workgroups and of sequences into parts,
// and the broadcasts of B and C inside a wave.
#pragma once

#include "sequence_dev.h"

#include <utility>

namespace ilx {

struct ScanArgs {
    ilx_state_space s;
    int group_channels;    // channels / groups
    int group_blocks;      // blocks of 64 channels per group
    int blocks;            // groups * group_blocks
    int64_t saved_blocks;  // blocks of ILX_SCAN_BLOCK rows per sequence
    // a long sequence in parts of part_rows rows (a multiple of ILX_SCAN_BLOCK); parts == 1: not divided
    int64_t parts, part_rows;
    float* part_state;   // (batch, parts, states, channels): what a part adds; after the join what enters it
    float* part_decay;   // (batch, parts, channels): sum of dt over a part, infinity if a start lies in it
    int64_t slots;       // backward, step: workgroups per block of channels
    float* sums;         // backward: (slots, states + 2, channels) partial sums of dA, dD and d delta_bias
    float* shared;       // backward: (group_blocks, batch, length, groups, 2 * padded states) partial sums of dB, dC
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

// Offset of a row: row and stride below 2^32, so one 32 x 32 bit product (scalar instructions).
__device__ __forceinline__ int64_t row_offset(uint32_t row, int64_t stride) {
    return static_cast<int64_t>(static_cast<uint64_t>(row) * static_cast<uint32_t>(stride));
}

// Bit i: an episode begins at row t0 + i (i < count <= 64).
__device__ __forceinline__ uint64_t start_bits(const ilx_state_space& s, int64_t b, int64_t t0, int count, int lane) {
    if (!s.starts) return 0;
    bool on = false;
    if (lane < count) on = s.starts[b * s.starts_batch + (t0 + lane) * s.starts_time] != 0;
    return __ballot(on);
}

template <typename F, int... I> __device__ __forceinline__ void static_for_(F f, std::integer_sequence<int, I...>) {
    (f(std::integral_constant<int, I>{}), ...);
}
template <int N, typename F> __device__ __forceinline__ void static_for(F f) { static_for_(f, std::make_integer_sequence<int, N>{}); }

// B and C of a row are the same for all channels of a wave.  They are held with state n in lane n of every 16 lanes, and an
// instruction that multiplies by one of them takes it from that lane (a row broadcast in its operand): no instruction, scalar
// register or LDS access of its own.
template <int L> __device__ __forceinline__ float from_lane(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0x150 + L, 0xf, 0xf, true));
}

// y0 + y1 += sum_n c[lane n] h[n] and r[n] += c[lane L + n] x.  The compiler does not give a fused multiply-add the
// broadcast operand, hence the assembly; a broadcast may not read what one of the two instructions ahead wrote, hence s_nop.
#define ILX_BCAST(n) " row_newbcast:" #n " row_mask:0xf bank_mask:0xf\n"
__device__ __forceinline__ void dot_states(float& y0, float& y1, float c, const float (&h)[4]) {
    asm("s_nop 1\n"
        "v_fmac_f32_dpp %0, %2, %3" ILX_BCAST(0) "v_fmac_f32_dpp %1, %2, %4" ILX_BCAST(1)
        "v_fmac_f32_dpp %0, %2, %5" ILX_BCAST(2) "v_fmac_f32_dpp %1, %2, %6" ILX_BCAST(3)
        : "+&v"(y0), "+&v"(y1)
        : "v"(c), "v"(h[0]), "v"(h[1]), "v"(h[2]), "v"(h[3]));
}
__device__ __forceinline__ void dot_states(float& y0, float& y1, float c, const float (&h)[8]) {
    asm("s_nop 1\n"
        "v_fmac_f32_dpp %0, %2, %3" ILX_BCAST(0) "v_fmac_f32_dpp %1, %2, %4" ILX_BCAST(1)
        "v_fmac_f32_dpp %0, %2, %5" ILX_BCAST(2) "v_fmac_f32_dpp %1, %2, %6" ILX_BCAST(3)
        "v_fmac_f32_dpp %0, %2, %7" ILX_BCAST(4) "v_fmac_f32_dpp %1, %2, %8" ILX_BCAST(5)
        "v_fmac_f32_dpp %0, %2, %9" ILX_BCAST(6) "v_fmac_f32_dpp %1, %2, %10" ILX_BCAST(7)
        : "+&v"(y0), "+&v"(y1)
        : "v"(c), "v"(h[0]), "v"(h[1]), "v"(h[2]), "v"(h[3]), "v"(h[4]), "v"(h[5]), "v"(h[6]), "v"(h[7]));
}
template <int O, int S> __device__ __forceinline__ void dot_sixteen(float& y0, float& y1, float c, const float (&h)[S]) {
    asm("s_nop 1\n"
        "v_fmac_f32_dpp %0, %2, %3" ILX_BCAST(0) "v_fmac_f32_dpp %1, %2, %4" ILX_BCAST(1)
        "v_fmac_f32_dpp %0, %2, %5" ILX_BCAST(2) "v_fmac_f32_dpp %1, %2, %6" ILX_BCAST(3)
        "v_fmac_f32_dpp %0, %2, %7" ILX_BCAST(4) "v_fmac_f32_dpp %1, %2, %8" ILX_BCAST(5)
        "v_fmac_f32_dpp %0, %2, %9" ILX_BCAST(6) "v_fmac_f32_dpp %1, %2, %10" ILX_BCAST(7)
        "v_fmac_f32_dpp %0, %2, %11" ILX_BCAST(8) "v_fmac_f32_dpp %1, %2, %12" ILX_BCAST(9)
        "v_fmac_f32_dpp %0, %2, %13" ILX_BCAST(10) "v_fmac_f32_dpp %1, %2, %14" ILX_BCAST(11)
        "v_fmac_f32_dpp %0, %2, %15" ILX_BCAST(12) "v_fmac_f32_dpp %1, %2, %16" ILX_BCAST(13)
        "v_fmac_f32_dpp %0, %2, %17" ILX_BCAST(14) "v_fmac_f32_dpp %1, %2, %18" ILX_BCAST(15)
        : "+&v"(y0), "+&v"(y1)
        : "v"(c), "v"(h[O + 0]), "v"(h[O + 1]), "v"(h[O + 2]), "v"(h[O + 3]), "v"(h[O + 4]), "v"(h[O + 5]), "v"(h[O + 6]), "v"(h[O + 7]),
          "v"(h[O + 8]), "v"(h[O + 9]), "v"(h[O + 10]), "v"(h[O + 11]), "v"(h[O + 12]), "v"(h[O + 13]), "v"(h[O + 14]), "v"(h[O + 15]));
}
__device__ __forceinline__ void dot_states(float& y0, float& y1, float c, const float (&h)[16]) { dot_sixteen<0>(y0, y1, c, h); }
// four states from lane L on
template <int L> __device__ __forceinline__ void dot_four(float& y, float c, const float (&h)[4]) {
    asm("s_nop 1\n"
        "v_fmac_f32_dpp %0, %1, %2 row_newbcast:%6 row_mask:0xf bank_mask:0xf\n"
        "v_fmac_f32_dpp %0, %1, %3 row_newbcast:%7 row_mask:0xf bank_mask:0xf\n"
        "v_fmac_f32_dpp %0, %1, %4 row_newbcast:%8 row_mask:0xf bank_mask:0xf\n"
        "v_fmac_f32_dpp %0, %1, %5 row_newbcast:%9 row_mask:0xf bank_mask:0xf\n"
        : "+&v"(y)
        : "v"(c), "v"(h[0]), "v"(h[1]), "v"(h[2]), "v"(h[3]), "n"(L), "n"(L + 1), "n"(L + 2), "n"(L + 3));
}
template <int L> __device__ __forceinline__ void add_four(float (&r)[4], float c, float x) {
    asm("s_nop 1\n"
        "v_fmac_f32_dpp %0, %4, %5 row_newbcast:%6 row_mask:0xf bank_mask:0xf\n"
        "v_fmac_f32_dpp %1, %4, %5 row_newbcast:%7 row_mask:0xf bank_mask:0xf\n"
        "v_fmac_f32_dpp %2, %4, %5 row_newbcast:%8 row_mask:0xf bank_mask:0xf\n"
        "v_fmac_f32_dpp %3, %4, %5 row_newbcast:%9 row_mask:0xf bank_mask:0xf\n"
        : "+&v"(r[0]), "+&v"(r[1]), "+&v"(r[2]), "+&v"(r[3])
        : "v"(c), "v"(x), "n"(L), "n"(L + 1), "n"(L + 2), "n"(L + 3));
}

int scan_check(const ilx_state_space& s, const char* name);
ScanArgs scan_args(const ilx_state_space& s);
// parts of a sequence, and the floats their states and decays take
int64_t divide_scan(ScanArgs& a, float* workspace);
void launch_part_states(const ScanArgs& a, bool backward, hipStream_t stream);

}  // namespace ilx
