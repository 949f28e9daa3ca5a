// What the state space kernels share: their arguments, the split of channels over workgroups and of sequences into parts,
// and the broadcasts of B and C inside a wave.
#pragma once

#include "sequence_dev.h"
#include "uniform_access.h"

#include <utility>

namespace ilx {

struct StateSpaceArgs {
    ilx_state_space s;
    int group_channels;    // channels / groups
    int group_blocks;      // blocks of 64 channels per group
    int blocks;            // groups * group_blocks
    int64_t saved_blocks;  // blocks of ILX_SCAN_BLOCK rows per sequence
    // a long sequence in parts of part_rows rows (a multiple of ILX_SCAN_BLOCK); parts == 1: not divided
    int64_t parts, part_rows;
    float* part_state;   // (batch, parts, states, channels): what a part adds; after the join what enters it
    float* part_decay;   // (batch, parts, channels): sum of dt over a part, infinity if a start lies in it
    int64_t slots;       // workgroups per block of channels
    int units;           // waves of a launch whose waves are independent
    bool decays_aligned; // A on a 16-byte boundary
    int64_t chains;      // backward: partial sums of a workgroup, each over kChainRows rows at most
    float* sums;         // backward: (slots, chains, states + 2, channels) partial sums of dA, dD and d delta_bias
    float* shared;       // backward: (group_blocks, batch, length, groups, 2 * padded states) partial sums of dB, dC
};

// A wave holds 64 channels of one group, a lane each; lanes past the group's end repeat its last channel and store nothing.
struct ChannelLane {
    int group, d;
    bool active;
};
__device__ __forceinline__ ChannelLane channel_lane(const StateSpaceArgs& a, int block, int lane) {
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

// The kernel's arguments, read anew: a value that an item needs once must not hold scalar registers through all of its rows
// (the compiler would keep all of them, and spill into vector registers, two to four cycles an access).
typedef const __attribute__((address_space(4))) StateSpaceArgs* ArgsPtr;
__device__ __forceinline__ ArgsPtr arguments_again() {
    auto p = __builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
    return (ArgsPtr)p;
}

// Elements of a row that all lanes share, by buffer instructions: the row is a scalar base and a scalar offset, the lane's byte
// offset one vector register that never changes, so an access costs no address arithmetic in the vector unit.
template <typename T> __device__ __forceinline__ __amdgpu_buffer_rsrc_t row_buffer(const T* base) {
    const uint64_t p = uni(reinterpret_cast<uint64_t>(base));
    return __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>(p), 0, 0xffffffff, 0x00027000);
}
template <typename T> __device__ __forceinline__ T lane_load(__amdgpu_buffer_rsrc_t row, uint32_t lane_bytes, uint32_t row_bytes) {
    if constexpr (sizeof(T) == 4)
        return __builtin_bit_cast(T, __builtin_amdgcn_raw_buffer_load_b32(row, lane_bytes, row_bytes, 0));
    else
        return __builtin_bit_cast(T, static_cast<uint16_t>(__builtin_amdgcn_raw_buffer_load_b16(row, lane_bytes, row_bytes, 0)));
}
template <typename T> __device__ __forceinline__ void lane_store(__amdgpu_buffer_rsrc_t row, uint32_t lane_bytes, uint32_t row_bytes, T v) {
    if constexpr (sizeof(T) == 4)
        __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, v), row, lane_bytes, row_bytes, 0);
    else
        __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(uint16_t, v), row, lane_bytes, row_bytes, 0);
}

// Here the value has arrived.  Loads and stores come back in one order and a wait counts what may still be out, so a value read ahead is
// waited for before the stores that follow: a wait behind them, at the value's use, would be one for the stores as well.
template <typename T> __device__ __forceinline__ void arrive(T& v) {
    if constexpr (sizeof(T) == 4) {
        asm volatile("" : "+v"(v));
    } else if constexpr (sizeof(T) == 2) {
        uint32_t u = __builtin_bit_cast(uint16_t, v);
        asm volatile("" : "+v"(u));
        v = __builtin_bit_cast(T, static_cast<uint16_t>(u));
    } else {
        uint32_t u = v;
        asm volatile("" : "+v"(u));
        v = static_cast<T>(u);
    }
}
template <typename T, int N> __device__ __forceinline__ void arrive(T (&v)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) arrive(v[i]);
}

// Rows of one sequence, from a moving first one.  Time strides are below 2^27 elements, so that a lane's offset in one of the next
// seven rows fits 32 bits.
template <typename T> struct Stream {
    const T* p;
    uint32_t time;   // bytes
    __device__ __forceinline__ void set(const void* base, int64_t sequence, int t0, int64_t stride) {
        time = static_cast<uint32_t>(stride) * static_cast<uint32_t>(sizeof(T));
        p = static_cast<const T*>(base) + sequence;
        step(t0);
    }
    __device__ __forceinline__ void step(int rows) {
        p = reinterpret_cast<const T*>(reinterpret_cast<uintptr_t>(p) + static_cast<int64_t>(rows) * static_cast<int64_t>(time));
    }
    __device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer() const { return row_buffer(p); }
};

template <typename F, int... I> __device__ __forceinline__ void static_for_(F f, std::integer_sequence<int, I...>) {
    (f(std::integral_constant<int, I>{}), ...);
}
template <int N, typename F> __device__ __forceinline__ void static_for(F f) { static_for_(f, std::make_integer_sequence<int, N>{}); }

typedef float f32x4 __attribute__((ext_vector_type(4)));

// B and C of a row are the same for all channels of a wave, so they are kept spread over lanes and enter the arithmetic from
// there, without an instruction, scalar register or LDS access of their own:
//  * h[0..3] += B[0..3] u  for all 64 channels is one 4 x 4 x 1 matrix instruction of 16 blocks: a lane's four results are its
//    block's four values of the first operand times the lane's own second operand, and the first operand's block is the same
//    for all blocks (or all of a row of 16 lanes).  One register holds 64 such values: 16 states of 4 rows.
//  * y += sum_n C[n] h[n]  takes C[n] from lane n of every 16 lanes (a row broadcast in the multiply-add's operand).
// Measured rates at full occupancy, in cycles a SIMD: multiply-add 2.6, with a broadcast operand 4.3, the matrix instruction 9.4 (for
// four multiply-adds), exponential 8.2, a select 4.6, half a wave's exchange (permlane swap) 8.4.
template <int BLOCK> __device__ __forceinline__ f32x4 outer(float values, float u, f32x4 h) {   // any 4 lanes' values for all lanes
    return __builtin_amdgcn_mfma_f32_4x4x1f32(values, u, h, 4, BLOCK, 0);
}

// y0 + y1 += sum of the states times lanes 0 .. of c.  The compiler does not give a fused multiply-add the broadcast operand, hence
// the assembly; a broadcast may not read what one of the two instructions ahead wrote, and a matrix instruction's result may not be
// read within five, hence the wait ahead of each block.
#define ILX_BCAST(n) " row_newbcast:" #n " row_mask:0xf bank_mask:0xf\n"
#define ILX_WAIT "s_nop 7\n"
__device__ __forceinline__ void dot_states(float& y0, float& y1, float c, const f32x4& a) {
    asm(ILX_WAIT
        "v_fmac_f32_dpp %0, %2, %3" ILX_BCAST(0) "v_fmac_f32_dpp %1, %2, %4" ILX_BCAST(1)
        "v_fmac_f32_dpp %0, %2, %5" ILX_BCAST(2) "v_fmac_f32_dpp %1, %2, %6" ILX_BCAST(3)
        : "+&v"(y0), "+&v"(y1)
        : "v"(c), "v"(a[0]), "v"(a[1]), "v"(a[2]), "v"(a[3]));
}
__device__ __forceinline__ void dot_states(float& y0, float& y1, float c, const f32x4& a, const f32x4& b) {
    asm(ILX_WAIT
        "v_fmac_f32_dpp %0, %2, %3" ILX_BCAST(0) "v_fmac_f32_dpp %1, %2, %4" ILX_BCAST(1)
        "v_fmac_f32_dpp %0, %2, %5" ILX_BCAST(2) "v_fmac_f32_dpp %1, %2, %6" ILX_BCAST(3)
        "v_fmac_f32_dpp %0, %2, %7" ILX_BCAST(4) "v_fmac_f32_dpp %1, %2, %8" ILX_BCAST(5)
        "v_fmac_f32_dpp %0, %2, %9" ILX_BCAST(6) "v_fmac_f32_dpp %1, %2, %10" ILX_BCAST(7)
        : "+&v"(y0), "+&v"(y1)
        : "v"(c), "v"(a[0]), "v"(a[1]), "v"(a[2]), "v"(a[3]), "v"(b[0]), "v"(b[1]), "v"(b[2]), "v"(b[3]));
}
__device__ __forceinline__ void dot_states(float& y0, float& y1, float c, const f32x4& a, const f32x4& b, const f32x4& d, const f32x4& e) {
    asm(ILX_WAIT
        "v_fmac_f32_dpp %0, %2, %3" ILX_BCAST(0) "v_fmac_f32_dpp %1, %2, %4" ILX_BCAST(1)
        "v_fmac_f32_dpp %0, %2, %5" ILX_BCAST(2) "v_fmac_f32_dpp %1, %2, %6" ILX_BCAST(3)
        "v_fmac_f32_dpp %0, %2, %7" ILX_BCAST(4) "v_fmac_f32_dpp %1, %2, %8" ILX_BCAST(5)
        "v_fmac_f32_dpp %0, %2, %9" ILX_BCAST(6) "v_fmac_f32_dpp %1, %2, %10" ILX_BCAST(7)
        "v_fmac_f32_dpp %0, %2, %11" ILX_BCAST(8) "v_fmac_f32_dpp %1, %2, %12" ILX_BCAST(9)
        "v_fmac_f32_dpp %0, %2, %13" ILX_BCAST(10) "v_fmac_f32_dpp %1, %2, %14" ILX_BCAST(11)
        "v_fmac_f32_dpp %0, %2, %15" ILX_BCAST(12) "v_fmac_f32_dpp %1, %2, %16" ILX_BCAST(13)
        "v_fmac_f32_dpp %0, %2, %17" ILX_BCAST(14) "v_fmac_f32_dpp %1, %2, %18" ILX_BCAST(15)
        : "+&v"(y0), "+&v"(y1)
        : "v"(c), "v"(a[0]), "v"(a[1]), "v"(a[2]), "v"(a[3]), "v"(b[0]), "v"(b[1]), "v"(b[2]), "v"(b[3]), "v"(d[0]), "v"(d[1]), "v"(d[2]), "v"(d[3]),
          "v"(e[0]), "v"(e[1]), "v"(e[2]), "v"(e[3]));
}

// v where the state exists, else 0, without a select
__device__ __forceinline__ float masked(float v, uint32_t mask) { return __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, v) & mask); }

int scan_check(const ilx_state_space& s, const char* name);
StateSpaceArgs scan_args(const ilx_state_space& s);
void share_items(StateSpaceArgs& a, int64_t items);
// parts of a sequence, and the floats their states and decays take
int64_t divide_scan(StateSpaceArgs& a, float* workspace);
void launch_part_states(const StateSpaceArgs& a, bool backward, hipStream_t stream);

}  // namespace ilx
