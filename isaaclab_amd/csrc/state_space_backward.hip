// Backward pass of the selective state space recurrence.  With dy the gradient of y (before the gate) and r_t that of h_t,
//   r_t[n] = dy_t C_t[n] + a_{t+1}[n] r_{t+1}[n],   a_t = exp(dt_t A) (0 at a start),   p_t = a_t h_{t-1},
//   dB_t[n] = sum_d r dt x,   dC_t[n] = sum_d dy h,   dA[n] = sum_t r p dt,   dx = D dy + dt sum_n r B,
//   d dt = x sum_n r B + sum_n r p A,   d delta = d dt sigmoid(delta + bias).
// The states are not kept by the forward pass (they are `states` times the inputs); it saves one in ILX_SCAN_BLOCK rows, and a
// workgroup recomputes a block's forward from there, then walks it backwards.  A workgroup has 64 channels, a lane each, and a
// wave for every four states, so a lane holds a and p of a whole block in registers (2 x 8 x 4); what is summed over the
// states (sum r B, sum r p A, y) meets in LDS once per block, and what is summed over the channels (dB, dC) is added across the
// lanes by a halving exchange: eight values become one register in 8 + 4 + 2 lanes' worth of instructions, not 8 x 6.
#include "state_space_dev.h"

namespace ilx {

constexpr int kRows = ILX_SCAN_BLOCK;
constexpr int kStates = 4;   // per wave
constexpr float kLn2 = 0.693147180559945309417f;


template <int L> __device__ __forceinline__ float from_lane(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0x150 + L, 0xf, 0xf, true));
}
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

template <int CTRL> __device__ __forceinline__ float dpp_add(float v) {
    const int o = __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true);
    return v + __builtin_bit_cast(float, o);
}

// {a.lower half, b.lower half} + {a.upper half, b.upper half}: in the lower 32 lanes a folded onto itself, in the upper b.
__device__ __forceinline__ float fold32(float a, float b) {
    const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, a), __builtin_bit_cast(unsigned, b), false, false);
    return __builtin_bit_cast(float, static_cast<unsigned>(r[0])) + __builtin_bit_cast(float, static_cast<unsigned>(r[1]));
}
// the same between the rows of 16 lanes: even rows keep a, odd rows b
__device__ __forceinline__ float fold16(float a, float b) {
    const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, a), __builtin_bit_cast(unsigned, b), false, false);
    return __builtin_bit_cast(float, static_cast<unsigned>(r[0])) + __builtin_bit_cast(float, static_cast<unsigned>(r[1]));
}

// The sums over the 64 lanes of eight values: lane l gets the one numbered bit 5 of l + 2 * bit 4 + 4 * bit 3.
__device__ __forceinline__ float sum_lanes(const float (&v)[8], int lane) {
    const float a = fold16(fold32(v[0], v[1]), fold32(v[2], v[3]));
    const float b = fold16(fold32(v[4], v[5]), fold32(v[6], v[7]));
    const float a8 = dpp_add<0x128>(a), b8 = dpp_add<0x128>(b);   // row_ror:8
    float s = lane & 8 ? b8 : a8;
    s = dpp_add<0x141>(s);   // row_half_mirror: lane i and 7 - i
    s = dpp_add<0x4e>(s);    // quad_perm 2,3,0,1
    return dpp_add<0xb1>(s); // quad_perm 1,0,3,2
}

// A block of rows of one part of a sequence.
struct ScanBlock {
    int64_t item, b, begin, end, t0;   // begin .. end: the part's rows that exist
    int count;
};

template <typename T, typename TB, int NW>
__global__ void __launch_bounds__(64 * NW, 3) scan_backward_kernel(StateSpaceArgs a) {
    constexpr int E = kRows / NW;   // rows a wave prepares and finishes per block
    __shared__ float2 s_step[2][kRows][64];       // dt and dt x, of this block and the one before
    __shared__ float s_dy[2][kRows][64];
    __shared__ float2 s_sum[NW][kRows][64];       // sum r B and sum r p A log2 e over the wave's states
    __shared__ float s_y[NW][kRows][64];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n0 = w * kStates;
    const int block = blockIdx.x % a.blocks;
    const int64_t slot = blockIdx.x / a.blocks;
    const ChannelLane c = channel_lane(a, block, lane);
    const int group_block = block - c.group * a.group_blocks;
    const ilx_state_space& s = a.s;
    const int64_t channels = s.channels, items = s.batch * a.parts;
    float A2[kStates], dA[kStates];   // A2 = A log2 e
#pragma unroll
    for (int n = 0; n < kStates; ++n) {
        const bool in = n0 + n < s.states;
        A2[n] = in ? s.A[static_cast<int64_t>(c.d) * s.states + n0 + n] * kLog2e : 0.0f;
        dA[n] = 0.0f;
    }
    const float bias = s.delta_bias ? s.delta_bias[c.d] : 0.0f, skip = s.D ? s.D[c.d] : 0.0f;
    float dD = 0.0f, dbias = 0.0f;
    const int value = (lane >> 5 & 1) + 2 * (lane >> 4 & 1) + 4 * (lane >> 3 & 1);   // what sum_lanes leaves here
    const int shared_column = (value >> 2) * (NW * kStates) + n0 + (value & 3);
    // B and C of four rows and the wave's four states in every 16 lanes
    const int bc_row = lane >> 2 & 3, bc_state = n0 + (lane & 3);
    const bool bc_in = bc_state < s.states;
    const int bc_at = bc_in ? bc_state : s.states - 1;
    const uint32_t parts = static_cast<uint32_t>(a.parts);

    // the last block of an item, with count 0 if the item has no rows
    auto item_end = [&](int64_t item) {
        ScanBlock k;
        k.item = item, k.b = static_cast<uint32_t>(item) / parts, k.begin = static_cast<uint32_t>(item) % parts * a.part_rows;
        const int64_t len = scan_length(s, k.b);
        k.end = k.begin + a.part_rows < len ? k.begin + a.part_rows : len;
        k.t0 = k.begin < k.end ? k.begin + (k.end - k.begin - 1) / kRows * kRows : k.begin;
        k.count = k.begin < k.end ? static_cast<int>(k.end - k.t0) : 0;
        return k;
    };
    // a block's inputs, read while the block ahead of it in this order is worked on
    T in_d[E], in_x[E], in_g[E], in_z[E];
    TB in_B[kRows / 4], in_C[kRows / 4];
    float in_h[kStates];
    uint64_t in_starts = 0;
    auto read = [&](const ScanBlock& k) {
        const T* px = static_cast<const T*>(s.x) + k.b * s.x_batch;
        const T* pd = static_cast<const T*>(s.delta) + k.b * s.delta_batch;
        const T* pz = static_cast<const T*>(s.gate) + k.b * s.gate_batch;
        const T* pg = static_cast<const T*>(s.grad_out) + k.b * s.grad_out_batch;
        const TB* pB = static_cast<const TB*>(s.B) + k.b * s.B_batch + c.group * s.states;
        const TB* pC = static_cast<const TB*>(s.C) + k.b * s.C_batch + c.group * s.states;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int i = e * NW + w;
            const uint32_t t = static_cast<uint32_t>(k.t0 + (i < k.count ? i : k.count - 1));
            in_d[e] = (pd + row_offset(t, s.delta_time))[c.d];
            in_x[e] = (px + row_offset(t, s.x_time))[c.d];
            in_g[e] = (pg + row_offset(t, s.grad_out_time))[c.d];
            if (s.gate) in_z[e] = (pz + row_offset(t, s.gate_time))[c.d];
        }
#pragma unroll
        for (int j = 0; j < kRows / 4; ++j) {
            const int i = 4 * j + bc_row;
            const uint32_t t = static_cast<uint32_t>(k.t0 + (i < k.count ? i : k.count - 1));
            in_B[j] = pB[row_offset(t, s.B_time) + bc_at];
            in_C[j] = pC[row_offset(t, s.C_time) + bc_at];
        }
        const float* save = s.saved + (k.b * a.saved_blocks + k.t0 / kRows) * s.states * channels;
#pragma unroll
        for (int n = 0; n < kStates; ++n) in_h[n] = (save + (n0 + n < s.states ? n0 + n : s.states - 1) * channels)[c.d];
        in_starts = start_bits(s, k.b, k.t0, k.count, lane);
    };

    ScanBlock k = item_end(slot);
    if (k.count > 0) read(k);
    float r[kStates];
    bool fresh = true;
    int buffer = 0;
    while (k.item < items) {
        if (fresh) {   // the item's last block: what enters the part from behind, and zeros for the rows that do not exist
            const float* enters = a.parts > 1 ? a.part_state + k.item * s.states * channels : s.grad_last ? s.grad_last + k.b * s.states * channels : nullptr;
#pragma unroll
            for (int n = 0; n < kStates; ++n) r[n] = enters && c.active && n0 + n < s.states ? (enters + (n0 + n) * channels)[c.d] : 0.0f;
            const int64_t limit = k.begin + a.part_rows < s.length ? k.begin + a.part_rows : s.length;
            for (int64_t t = (k.end > k.begin ? k.end : k.begin) + w; t < limit; t += NW) {
                const int64_t at = k.b * s.grad_batch + t * s.grad_time + c.d;
                if (!c.active) break;
                static_cast<T*>(s.grad_x)[at] = from_f32<T>(0.0f);
                static_cast<T*>(s.grad_delta)[at] = from_f32<T>(0.0f);
                if (s.gate) static_cast<T*>(s.grad_gate)[at] = from_f32<T>(0.0f);
            }
        }
        ScanBlock next = k;
        if (k.t0 > k.begin) {
            next.t0 = k.t0 - kRows, next.count = kRows;
        } else if (k.item + a.slots < items) {
            next = item_end(k.item + a.slots);
        } else {
            next.item = items, next.count = 0;
        }
        if (k.count > 0) {
            // rows past the end act as rows that leave the state alone: dt = x = dy = 0
            float slope[E], dgate[E], x[E];
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const int i = e * NW + w;
                const bool in = i < k.count && c.active;
                const float raw = to_f32(in_d[e]) + bias, g = to_f32(in_g[e]);
                x[e] = in ? to_f32(in_x[e]) : 0.0f;
                float dy = g;
                dgate[e] = 0.0f;
                if (s.gate) {
                    const float z = to_f32(in_z[e]), sig = sigmoid_fast(z);
                    dy = g * z * sig;
                    dgate[e] = g * sig * __builtin_fmaf(z, 1.0f - sig, 1.0f);
                }
                slope[e] = s.softplus ? sigmoid_fast(raw) : 1.0f;
                const float dt = in ? (s.softplus ? softplus_f(raw) : raw) : 0.0f;
                s_step[buffer][i][lane] = make_float2(dt, dt * x[e]);
                s_dy[buffer][i][lane] = in ? dy : 0.0f;
            }
            float B[kRows / 4], C[kRows / 4], h0[kStates], decay[kRows][kStates], h[kRows][kStates];
#pragma unroll
            for (int j = 0; j < kRows / 4; ++j) B[j] = bc_in ? to_f32(in_B[j]) : 0.0f, C[j] = bc_in ? to_f32(in_C[j]) : 0.0f;
#pragma unroll
            for (int n = 0; n < kStates; ++n) h0[n] = n0 + n < s.states ? in_h[n] : 0.0f;
            const uint64_t starts = in_starts;
            __syncthreads();
            if (next.count > 0) read(next);
            float kept = 0.0f;
            auto walk = [&](auto with_starts) {
                static_for<kRows>([&](auto row) {
                    constexpr int i = row;
                    __builtin_amdgcn_sched_barrier(0);
                    const float2 v = s_step[buffer][i][lane];
                    const bool start = decltype(with_starts)::value && (starts >> i & 1);
                    static_for<kStates>([&](auto state) {
                        constexpr int n = state;
                        const float before = i == 0 ? h0[n] : h[i == 0 ? 0 : i - 1][n];
                        const float e = __builtin_amdgcn_exp2f(v.x * A2[n]);
                        decay[i][n] = start ? 0.0f : e;
                        h[i][n] = __builtin_fmaf(decay[i][n], start ? 0.0f : before, v.y * from_lane<4 * (i & 3) + n>(B[i >> 2]));
                    });
                    float y = 0.0f;
                    dot_four<4 * (i & 3)>(y, C[i >> 2], h[i]);
                    s_y[w][i][lane] = y;
                });
                uint64_t starts_again = starts;   // (kept apart: the compiler would hold what the two walks share in registers)
                asm volatile("" : "+s"(starts_again) : : "memory");
                static_for<kRows>([&](auto row) {
                    constexpr int i = kRows - 1 - row;
                    __builtin_amdgcn_sched_barrier(0);
                    const float2 u = s_step[buffer][i][lane];
                    const float dy = s_dy[buffer][i][lane];
                    const bool start = decltype(with_starts)::value && (starts_again >> i & 1);
                    float v[2 * kStates], rb = 0.0f, ra = 0.0f;
                    add_four<4 * (i & 3)>(r, C[i >> 2], dy);
                    dot_four<4 * (i & 3)>(rb, B[i >> 2], r);
                    static_for<kStates>([&](auto state) {
                        constexpr int n = state;
                        v[n] = r[n] * u.y;
                        v[kStates + n] = dy * h[i][n];
                        r[n] = start ? 0.0f : r[n] * decay[i][n];
                        const float q = r[n] * (start ? 0.0f : i == 0 ? h0[n] : h[i == 0 ? 0 : i - 1][n]);
                        ra = __builtin_fmaf(q, A2[n], ra);
                        dA[n] = __builtin_fmaf(q, u.x, dA[n]);
                    });
                    s_sum[w][i][lane] = make_float2(rb, ra);
                    const float sum = sum_lanes(v, lane);
                    kept = (lane & 7) == i ? sum : kept;
                });
            };
            if (starts)
                walk(std::true_type{});
            else
                walk(std::false_type{});
            if ((lane & 7) < k.count) {
                const int64_t at = ((group_block * s.batch + k.b) * s.length + k.t0 + (lane & 7)) * s.groups + c.group;
                a.shared[at * (2 * NW * kStates) + shared_column] = kept;
            }
            __syncthreads();
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const int i = e * NW + w;
                if (i < k.count && c.active) {
                    float rb = 0.0f, ra = 0.0f, y = 0.0f;
#pragma unroll
                    for (int j = 0; j < NW; ++j) {
                        const float2 v = s_sum[j][i][lane];
                        rb += v.x, ra += v.y;
                        y += s_y[j][i][lane];
                    }
                    const float dt = s_step[buffer][i][lane].x, dy = s_dy[buffer][i][lane], draw = __builtin_fmaf(x[e], rb, ra * kLn2) * slope[e];
                    const int64_t at = k.b * s.grad_batch + row_offset(static_cast<uint32_t>(k.t0 + i), s.grad_time);
                    (static_cast<T*>(s.grad_x) + at)[c.d] = from_f32<T>(__builtin_fmaf(dt, rb, skip * dy));
                    (static_cast<T*>(s.grad_delta) + at)[c.d] = from_f32<T>(draw);
                    if (s.gate) (static_cast<T*>(s.grad_gate) + at)[c.d] = from_f32<T>(dgate[e] * __builtin_fmaf(skip, x[e], y));
                    dD = __builtin_fmaf(dy, x[e], dD);
                    dbias += draw;
                }
            }
            buffer ^= 1;   // (the next block's rows go where nobody still reads; its sums are written behind a barrier)
        } else if (next.count > 0) {
            read(next);
        }
        fresh = next.item != k.item;
        if (fresh && k.begin == 0 && s.grad_state && c.active) {
#pragma unroll
            for (int n = 0; n < kStates; ++n)
                if (n0 + n < s.states) (s.grad_state + (k.b * s.states + n0 + n) * channels)[c.d] = r[n];
        }
        k = next;
    }
    __syncthreads();
    s_sum[0][w][lane] = make_float2(dD, dbias);
    __syncthreads();
    if (!c.active) return;
    float* sums = a.sums + slot * (s.states + 2) * channels;
#pragma unroll
    for (int n = 0; n < kStates; ++n)
        if (n0 + n < s.states) sums[(n0 + n) * channels + c.d] = dA[n];
    if (w == 0) {
        for (int j = 1; j < NW; ++j) dD += s_sum[0][j][lane].x, dbias += s_sum[0][j][lane].y;
        sums[s.states * channels + c.d] = dD;
        sums[(s.states + 1) * channels + c.d] = dbias;
    }
}

// dB and dC: the sums of the blocks of channels of a group, in order; rows past a sequence's end are zeros.
template <typename TB> __global__ void __launch_bounds__(256) scan_shared_sums_kernel(StateSpaceArgs a, int padded) {
    const ilx_state_space& s = a.s;
    const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x, rows = s.batch * s.length * s.groups;
    if (i >= rows * s.states) return;
    const int64_t row = i / s.states;
    const int n = static_cast<int>(i - row * s.states);
    const int64_t bt = row / s.groups, b = bt / s.length, t = bt - b * s.length;
    float dB = 0.0f, dC = 0.0f;
    if (t < scan_length(s, b))
        for (int k = 0; k < a.group_blocks; ++k) {
            const float* p = a.shared + (k * rows + row) * 2 * padded + n;
            dB += p[0];
            dC += p[padded];
        }
    static_cast<TB*>(s.grad_B)[i] = from_f32<TB>(dB);
    static_cast<TB*>(s.grad_C)[i] = from_f32<TB>(dC);
}

}  // namespace ilx

using namespace ilx;

namespace {

int waves_for(int states) { return states <= 4 ? 1 : states <= 8 ? 2 : states <= 16 ? 4 : 8; }

StateSpaceArgs backward_args(const ilx_state_space& s, int64_t* floats) {
    StateSpaceArgs a = scan_args(s);
    const int64_t part_floats = divide_scan(a, s.workspace);
    const int64_t most = 2048 / a.blocks > 0 ? 2048 / a.blocks : 1, items = s.batch * a.parts;
    a.slots = items < most ? items : most;
    const int64_t sums = a.slots * (s.states + 2) * s.channels;
    const int64_t shared = a.group_blocks * s.batch * s.length * s.groups * 2 * waves_for(s.states) * kStates;
    a.sums = s.workspace + part_floats;
    a.shared = a.sums + sums;
    *floats = part_floats + sums + shared;
    return a;
}

template <typename T, typename TB, int NW> void backward_launch(const StateSpaceArgs& a, hipStream_t s) {
    ILX_LAUNCH((scan_backward_kernel<T, TB, NW>), dim3(static_cast<unsigned>(a.slots * a.blocks)), dim3(64 * NW), 0, s, a);
}

template <typename T, typename TB> void backward_states(const StateSpaceArgs& a, hipStream_t s) {
    const int waves = waves_for(a.s.states);
    switch (waves) {
        case 1: backward_launch<T, TB, 1>(a, s); break;
        case 2: backward_launch<T, TB, 2>(a, s); break;
        case 4: backward_launch<T, TB, 4>(a, s); break;
        default: backward_launch<T, TB, 8>(a, s); break;
    }
    const int64_t values = a.s.batch * a.s.length * a.s.groups * a.s.states;
    if (values > 0) ILX_LAUNCH((scan_shared_sums_kernel<TB>), dim3(blocks_for(values)), dim3(256), 0, s, a, waves * kStates);
}

}  // namespace

extern "C" int ilx_state_space_workspace(const ilx_state_space* scan, int backward, int64_t* floats) {
    ILX_REQUIRE(scan && floats, ILX_EINVAL, "ilx_state_space_workspace: NULL argument");
    const int rc = scan_check(*scan, "ilx_state_space_workspace");
    if (rc != ILX_OK) return rc;
    if (backward) {
        backward_args(*scan, floats);
    } else {
        StateSpaceArgs a = scan_args(*scan);
        *floats = divide_scan(a, nullptr);
    }
    return ILX_OK;
}

extern "C" int ilx_state_space_backward(const ilx_state_space* scan, void* stream) {
    ILX_REQUIRE(scan, ILX_EINVAL, "ilx_state_space_backward: descriptor is NULL");
    const ilx_state_space& s = *scan;
    const int rc = scan_check(s, "ilx_state_space_backward");
    if (rc != ILX_OK) return rc;
    const bool some = s.batch > 0 && s.length > 0;
    ILX_REQUIRE(s.A && s.grad_A && (!some || (s.x && s.delta && s.B && s.C && s.grad_out && s.grad_x && s.grad_delta && s.grad_B && s.grad_C && s.saved)),
                ILX_EINVAL, "ilx_state_space_backward: NULL operand");
    ILX_REQUIRE(!some || (s.gate != nullptr) == (s.grad_gate != nullptr), ILX_EINVAL, "ilx_state_space_backward: gate and grad_gate come together");
    int64_t needed = 0;
    const StateSpaceArgs a = backward_args(s, &needed);
    ILX_REQUIRE(s.workspace_floats >= needed && (s.workspace || needed == 0), ILX_EINVAL,
                "ilx_state_space_backward: workspace of %lld floats, %lld needed", (long long)s.workspace_floats, (long long)needed);
    ILX_REQUIRE(s.batch * a.parts * a.blocks <= INT32_MAX && s.batch * s.length * s.groups * s.states / 256 < INT32_MAX, ILX_ESHAPE,
                "ilx_state_space_backward: shape too large for one launch");
    hipStream_t st = as_stream(stream);
    if (s.batch > 0) {
        if (a.parts > 1) launch_part_states(a, true, st);
        const bool wide = s.bc_dtype == ILX_F32;
        switch (s.dtype) {
            case ILX_F32: backward_states<float, float>(a, st); break;
            case ILX_BF16: wide ? backward_states<bf16_t, float>(a, st) : backward_states<bf16_t, bf16_t>(a, st); break;
            default: wide ? backward_states<f16_t, float>(a, st) : backward_states<f16_t, f16_t>(a, st); break;
        }
    }
    launch_parameter_sums(a.sums, a.slots, s.channels, s.states, s.grad_A, s.grad_D, s.grad_delta_bias, st);
    ILX_LAUNCH_CHECK("ilx_state_space_backward");
    return ILX_OK;
}
