// Backward pass of the selective state space recurrence.  With dy the gradient of y (before the gate) and r_t that of h_t,
//   r_t[n] = dy_t C_t[n] + a_{t+1}[n] r_{t+1}[n],   a_t = exp(dt_t A) (0 at a start),   p_t = a_t h_{t-1},
//   dB_t[n] = sum_d r dt x,   dC_t[n] = sum_d dy h,   dA[n] = sum_t r p dt,   dx = D dy + dt sum_n r B,
//   d dt = x sum_n r B + sum_n r p A,   d delta = d dt sigmoid(delta + bias).
// The states are not kept by the forward pass (they are `states` times the inputs); it saves one in ILX_SCAN_BLOCK rows, and a
// workgroup recomputes a block's forward from there, then walks it backwards.  A workgroup has 64 channels, a lane each, and a
// wave for every four states, so a lane holds a and p of a whole block in registers (2 x 16 x 4); what is summed over the
// states (sum r B, sum r p A, y) meets in LDS once per block, and what is summed over the channels (dB, dC) is added across the
// lanes by a halving exchange: eight values become one register in 8 + 4 + 2 lanes' worth of instructions, not 8 x 6.
#include "state_space_dev.h"

namespace ilx {

constexpr int kRows = ILX_SCAN_BLOCK;
constexpr int kStates = 4;   // per wave

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

template <typename T, typename TB, int NW, bool FULL>
__global__ void __launch_bounds__(64 * NW) scan_backward_kernel(ScanArgs a) {
    constexpr int E = kRows / NW;   // rows a wave prepares and finishes per block
    __shared__ float s_dt[kRows][64], s_x[kRows][64], s_dy[kRows][64];
    __shared__ float s_rb[NW][kRows][64], s_ra[NW][kRows][64], s_y[NW][kRows][64];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n0 = w * kStates;
    const int block = blockIdx.x % a.blocks;
    const int64_t slot = blockIdx.x / a.blocks;
    const ChannelLane c = channel_lane(a, block, lane);
    const int group_block = block - c.group * a.group_blocks;
    const ilx_state_space& s = a.s;
    const int64_t channels = s.channels;
    float A[kStates], A2[kStates], dA[kStates];
#pragma unroll
    for (int n = 0; n < kStates; ++n) {
        A[n] = FULL || n0 + n < s.states ? s.A[static_cast<int64_t>(c.d) * s.states + n0 + n] : 0.0f;
        A2[n] = A[n] * kLog2e;
        dA[n] = 0.0f;
    }
    const float bias = s.delta_bias ? s.delta_bias[c.d] : 0.0f, skip = s.D ? s.D[c.d] : 0.0f;
    float dD = 0.0f, dbias = 0.0f;
    const int value = (lane >> 5 & 1) + 2 * (lane >> 4 & 1) + 4 * (lane >> 3 & 1);   // what sum_lanes leaves here
    const int shared_column = (value >> 2) * (NW * kStates) + n0 + (value & 3);

    for (int64_t b = slot; b < s.batch; b += a.slots) {
        const int64_t len = scan_length(s, b);
        const T* px = static_cast<const T*>(s.x) + b * s.x_batch + c.d;
        const T* pd = static_cast<const T*>(s.delta) + b * s.delta_batch + c.d;
        const T* pz = s.gate ? static_cast<const T*>(s.gate) + b * s.gate_batch + c.d : nullptr;
        const T* pg = static_cast<const T*>(s.grad_out) + b * s.grad_out_batch + c.d;
        const TB* pB = static_cast<const TB*>(s.B) + b * s.B_batch + c.group * s.states;
        const TB* pC = static_cast<const TB*>(s.C) + b * s.C_batch + c.group * s.states;
        T* gx = static_cast<T*>(s.grad_x) + b * s.grad_x_batch + c.d;
        T* gd = static_cast<T*>(s.grad_delta) + b * s.grad_delta_batch + c.d;
        T* gz = s.gate ? static_cast<T*>(s.grad_gate) + b * s.grad_gate_batch + c.d : nullptr;
        float r[kStates];
#pragma unroll
        for (int n = 0; n < kStates; ++n)
            r[n] = s.grad_last && c.active && (FULL || n0 + n < s.states) ? s.grad_last[(b * s.states + n0 + n) * channels + c.d] : 0.0f;
        for (int64_t t = len + w; t < s.length; t += NW) {
            if (!c.active) break;
            gx[t * s.grad_x_time] = from_f32<T>(0.0f);
            gd[t * s.grad_delta_time] = from_f32<T>(0.0f);
            if (gz) gz[t * s.grad_gate_time] = from_f32<T>(0.0f);
        }
        for (int64_t blk = (len + kRows - 1) / kRows - 1; blk >= 0; --blk) {
            const int64_t t0 = blk * kRows;
            const int count = len - t0 < kRows ? static_cast<int>(len - t0) : kRows;
            // rows past the end act as rows that leave the state alone: dt = x = dy = 0
            float slope[E], dgate[E];
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const int i = e * NW + w;
                const bool in = i < count && c.active;
                const int64_t t = t0 + (i < count ? i : count - 1);
                const float raw = to_f32(pd[t * s.delta_time]) + bias, x = to_f32(px[t * s.x_time]), g = to_f32(pg[t * s.grad_out_time]);
                float dy = g;
                dgate[e] = 0.0f;
                if (pz) {
                    const float z = to_f32(pz[t * s.gate_time]), sig = sigmoid_fast(z);
                    dy = g * z * sig;
                    dgate[e] = g * sig * __builtin_fmaf(z, 1.0f - sig, 1.0f);
                }
                slope[e] = s.softplus ? sigmoid_fast(raw) : 1.0f;
                s_dt[i][lane] = in ? (s.softplus ? softplus_f(raw) : raw) : 0.0f;
                s_x[i][lane] = in ? x : 0.0f;
                s_dy[i][lane] = in ? dy : 0.0f;
            }
            const uint64_t starts = start_bits(s, b, t0, count, lane);
            float h[kStates], decay[kRows][kStates], p[kRows][kStates];
            const float* save = s.saved + (b * a.saved_blocks + blk) * s.states * channels + c.d;
#pragma unroll
            for (int n = 0; n < kStates; ++n) h[n] = FULL || n0 + n < s.states ? save[(n0 + n) * channels] : 0.0f;
            __syncthreads();
#pragma unroll
            for (int i = 0; i < kRows; ++i) {
                const int64_t t = t0 + (i < count ? i : count - 1);
                float B[kStates], C[kStates];
                load_uniform<kStates, FULL>(pB + t * s.B_time, n0, s.states, B);
                load_uniform<kStates, FULL>(pC + t * s.C_time, n0, s.states, C);
                const float dt = s_dt[i][lane], u = dt * s_x[i][lane];
                const bool start = starts >> i & 1;
                float y = 0.0f;
#pragma unroll
                for (int n = 0; n < kStates; ++n) {
                    decay[i][n] = start ? 0.0f : __builtin_amdgcn_exp2f(dt * A2[n]);
                    p[i][n] = start ? 0.0f : decay[i][n] * h[n];
                    h[n] = __builtin_fmaf(u, B[n], p[i][n]);
                    y = __builtin_fmaf(C[n], h[n], y);
                }
                s_y[w][i][lane] = y;
            }
            float kept = 0.0f;
#pragma unroll
            for (int i = kRows - 1; i >= 0; --i) {
                const int64_t t = t0 + (i < count ? i : count - 1);
                float B[kStates], C[kStates], v[2 * kStates];
                load_uniform<kStates, FULL>(pB + t * s.B_time, n0, s.states, B);
                load_uniform<kStates, FULL>(pC + t * s.C_time, n0, s.states, C);
                const float dt = s_dt[i][lane], u = dt * s_x[i][lane], dy = s_dy[i][lane];
                float rb = 0.0f, ra = 0.0f;
#pragma unroll
                for (int n = 0; n < kStates; ++n) {
                    r[n] = __builtin_fmaf(dy, C[n], r[n]);
                    rb = __builtin_fmaf(r[n], B[n], rb);
                    const float q = r[n] * p[i][n];
                    ra = __builtin_fmaf(q, A[n], ra);
                    dA[n] = __builtin_fmaf(q, dt, dA[n]);
                    v[n] = r[n] * u;
                    v[kStates + n] = dy * __builtin_fmaf(u, B[n], p[i][n]);
                    r[n] *= decay[i][n];
                }
                s_rb[w][i][lane] = rb;
                s_ra[w][i][lane] = ra;
                const float sum = sum_lanes(v, lane);
                kept = (lane & 7) == (i & 7) ? sum : kept;
                if ((i & 7) == 0 && i + (lane & 7) < count) {
                    const int64_t row = ((group_block * s.batch + b) * s.length + t0 + i + (lane & 7)) * s.groups + c.group;
                    a.shared[row * (2 * NW * kStates) + shared_column] = kept;
                }
            }
            __syncthreads();
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const int i = e * NW + w;
                if (i < count && c.active) {
                    const int64_t t = t0 + i;
                    float rb = 0.0f, ra = 0.0f, y = 0.0f;
#pragma unroll
                    for (int k = 0; k < NW; ++k) rb += s_rb[k][i][lane], ra += s_ra[k][i][lane], y += s_y[k][i][lane];
                    const float dt = s_dt[i][lane], x = s_x[i][lane], dy = s_dy[i][lane];
                    const float draw = __builtin_fmaf(x, rb, ra) * slope[e];
                    gx[t * s.grad_x_time] = from_f32<T>(__builtin_fmaf(dt, rb, skip * dy));
                    gd[t * s.grad_delta_time] = from_f32<T>(draw);
                    if (gz) gz[t * s.grad_gate_time] = from_f32<T>(dgate[e] * __builtin_fmaf(skip, x, y));
                    dD = __builtin_fmaf(dy, x, dD);
                    dbias += draw;
                }
            }
            __syncthreads();
        }
        if (s.grad_state && c.active) {
#pragma unroll
            for (int n = 0; n < kStates; ++n)
                if (FULL || n0 + n < s.states) s.grad_state[(b * s.states + n0 + n) * channels + c.d] = r[n];
        }
    }
    s_dt[w][lane] = dD;
    s_x[w][lane] = dbias;
    __syncthreads();
    if (!c.active) return;
    float* sums = a.sums + slot * (s.states + 2) * channels + c.d;
#pragma unroll
    for (int n = 0; n < kStates; ++n)
        if (FULL || n0 + n < s.states) sums[(n0 + n) * channels] = dA[n];
    if (w == 0) {
        for (int k = 1; k < NW; ++k) dD += s_dt[k][lane], dbias += s_x[k][lane];
        sums[s.states * channels] = dD;
        sums[(s.states + 1) * channels] = dbias;
    }
}

// dB and dC: the sums of the blocks of channels of a group, in order; rows past a sequence's end are zeros.
template <typename TB> __global__ void __launch_bounds__(256) scan_shared_sums_kernel(ScanArgs a, int padded) {
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

ScanArgs backward_args(const ilx_state_space& s, int64_t* floats) {
    ScanArgs a = scan_args(s);
    const int64_t most = 1024 / a.blocks > 0 ? 1024 / a.blocks : 1;
    a.slots = s.batch < most ? s.batch : most;
    const int64_t sums = a.slots * (s.states + 2) * s.channels;
    const int64_t shared = a.group_blocks * s.batch * s.length * s.groups * 2 * waves_for(s.states) * kStates;
    a.sums = s.workspace;
    a.shared = s.workspace + sums;
    *floats = sums + shared;
    return a;
}

template <typename T, typename TB, int NW> void backward_launch(const ScanArgs& a, hipStream_t s) {
    const dim3 grid(static_cast<unsigned>(a.slots * a.blocks)), threads(64 * NW);
    if (a.s.states == NW * kStates)
        ILX_LAUNCH((scan_backward_kernel<T, TB, NW, true>), grid, threads, 0, s, a);
    else
        ILX_LAUNCH((scan_backward_kernel<T, TB, NW, false>), grid, threads, 0, s, a);
}

template <typename T, typename TB> void backward_states(const ScanArgs& a, hipStream_t s) {
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
    *floats = 0;
    if (backward) backward_args(*scan, floats);
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
    const ScanArgs a = backward_args(s, &needed);
    ILX_REQUIRE(s.workspace_floats >= needed && (s.workspace || needed == 0), ILX_EINVAL,
                "ilx_state_space_backward: workspace of %lld floats, %lld needed", (long long)s.workspace_floats, (long long)needed);
    ILX_REQUIRE(a.slots * a.blocks <= INT32_MAX && s.batch * s.length * s.groups * s.states / 256 < INT32_MAX, ILX_ESHAPE,
                "ilx_state_space_backward: shape too large for one launch");
    hipStream_t st = as_stream(stream);
    if (s.batch > 0) {
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
