// Selective state space recurrence, forward and one step:
//   h[n] <- exp(dt A[n]) h[n] + dt B[n] x,   y = sum_n C[n] h[n] + D x,   dt = softplus(delta + bias)
// per channel, with B and C shared by the channels of a group.
// A lane owns a channel and all its states, a wave 64 channels: the recurrence needs no exchange between lanes, B and C
// are scalars of the wave, and a row's x, delta, gate and out are one access of 64 neighbours each.  Per state and row
// there is one multiply, one exponential (which issues at a quarter of the rate) and three more instructions.
#include "state_space_dev.h"

namespace ilx {

constexpr int kScanRows = 8;   // rows whose inputs are in registers together

template <typename T, typename TB, int S, bool FULL>
__global__ void __launch_bounds__(64) scan_forward_kernel(ScanArgs a) {
    const int lane = threadIdx.x;
    const int block = blockIdx.x % a.blocks;
    const int64_t b = blockIdx.x / a.blocks;
    const ChannelLane c = channel_lane(a, block, lane);
    const ilx_state_space& s = a.s;
    const int64_t len = scan_length(s, b), channels = s.channels;
    float A2[S], h[S];
#pragma unroll
    for (int n = 0; n < S; ++n) {
        const bool in = FULL || n < s.states;
        A2[n] = in ? s.A[static_cast<int64_t>(c.d) * s.states + n] * kLog2e : 0.0f;
        h[n] = in && s.state ? s.state[(b * s.states + n) * channels + c.d] : 0.0f;
    }
    const float bias = s.delta_bias ? s.delta_bias[c.d] : 0.0f, skip = s.D ? s.D[c.d] : 0.0f;
    const T* px = static_cast<const T*>(s.x) + b * s.x_batch;
    const T* pd = static_cast<const T*>(s.delta) + b * s.delta_batch;
    const T* pz = s.gate ? static_cast<const T*>(s.gate) + b * s.gate_batch : nullptr;
    const TB* pB = static_cast<const TB*>(s.B) + b * s.B_batch + c.group * s.states;
    const TB* pC = static_cast<const TB*>(s.C) + b * s.C_batch + c.group * s.states;
    T* po = static_cast<T*>(s.out) + b * s.out_batch;
    for (int64_t t0 = 0; t0 < len; t0 += kScanRows) {
        const int count = len - t0 < kScanRows ? static_cast<int>(len - t0) : kScanRows;
        float x[kScanRows], dt[kScanRows], z[kScanRows];
#pragma unroll
        for (int i = 0; i < kScanRows; ++i) {
            const int64_t t = t0 + (i < count ? i : count - 1);
            x[i] = to_f32(px[t * s.x_time + c.d]);
            dt[i] = to_f32(pd[t * s.delta_time + c.d]);
            z[i] = pz ? to_f32(pz[t * s.gate_time + c.d]) : 0.0f;
        }
        const uint64_t starts = start_bits(s, b, t0, count, lane);
        if (s.saved && t0 % ILX_SCAN_BLOCK == 0 && c.active) {
            float* save = s.saved + (b * a.saved_blocks + t0 / ILX_SCAN_BLOCK) * s.states * channels + c.d;
#pragma unroll
            for (int n = 0; n < S; ++n)
                if (FULL || n < s.states) save[n * channels] = h[n];
        }
#pragma unroll
        for (int i = 0; i < kScanRows; ++i) {
            dt[i] += bias;
            if (s.softplus) dt[i] = softplus_f(dt[i]);
        }
#pragma unroll
        for (int i = 0; i < kScanRows; ++i) {
            if (i < count) {
                const int64_t t = t0 + i;
                float B[S], C[S];
                load_uniform<S, FULL>(pB + t * s.B_time, 0, s.states, B);
                load_uniform<S, FULL>(pC + t * s.C_time, 0, s.states, C);
                const float u = dt[i] * x[i];
                float y = skip * x[i];
                if (starts >> i & 1) {
#pragma unroll
                    for (int n = 0; n < S; ++n) h[n] = 0.0f;
                }
#pragma unroll
                for (int n = 0; n < S; ++n) {
                    const float decay = __builtin_amdgcn_exp2f(dt[i] * A2[n]);
                    h[n] = __builtin_fmaf(decay, h[n], u * B[n]);
                    y = __builtin_fmaf(C[n], h[n], y);
                }
                if (pz) y *= z[i] * sigmoid_fast(z[i]);
                if (c.active) po[t * s.out_time + c.d] = from_f32<T>(y);
            }
        }
    }
    if (!c.active) return;
    for (int64_t t = len; t < s.length; ++t) po[t * s.out_time + c.d] = from_f32<T>(0.0f);
    if (s.last) {
#pragma unroll
        for (int n = 0; n < S; ++n)
            if (FULL || n < s.states) s.last[(b * s.states + n) * channels + c.d] = h[n];
    }
}

// One row per sequence: the recurrence above with sequences in the place of rows, so that A stays in registers.  Bound by
// the state, read and written once.
template <typename T, typename TB, int S, bool FULL>
__global__ void __launch_bounds__(64) scan_step_kernel(ScanArgs a) {
    const int lane = threadIdx.x;
    const ChannelLane c = channel_lane(a, blockIdx.x % a.blocks, lane);
    const ilx_state_space& s = a.s;
    const int64_t channels = s.channels;
    float A2[S];
#pragma unroll
    for (int n = 0; n < S; ++n) A2[n] = FULL || n < s.states ? s.A[static_cast<int64_t>(c.d) * s.states + n] * kLog2e : 0.0f;
    const float bias = s.delta_bias ? s.delta_bias[c.d] : 0.0f, skip = s.D ? s.D[c.d] : 0.0f;
    for (int64_t b = blockIdx.x / a.blocks; b < s.batch; b += a.slots) {
        float h[S], B[S], C[S];
        float* state = s.last + b * s.states * channels + c.d;
#pragma unroll
        for (int n = 0; n < S; ++n) h[n] = FULL || n < s.states ? state[n * channels] : 0.0f;
        const float x = to_f32(static_cast<const T*>(s.x)[b * s.x_batch + c.d]);
        float dt = to_f32(static_cast<const T*>(s.delta)[b * s.delta_batch + c.d]) + bias;
        const float z = s.gate ? to_f32(static_cast<const T*>(s.gate)[b * s.gate_batch + c.d]) : 0.0f;
        const bool start = s.starts && s.starts[b * s.starts_batch];
        load_uniform<S, FULL>(static_cast<const TB*>(s.B) + b * s.B_batch + c.group * s.states, 0, s.states, B);
        load_uniform<S, FULL>(static_cast<const TB*>(s.C) + b * s.C_batch + c.group * s.states, 0, s.states, C);
        if (s.softplus) dt = softplus_f(dt);
        const float u = dt * x;
        float y = skip * x;
#pragma unroll
        for (int n = 0; n < S; ++n) {
            const float decay = __builtin_amdgcn_exp2f(dt * A2[n]);
            h[n] = __builtin_fmaf(decay, start ? 0.0f : h[n], u * B[n]);
            y = __builtin_fmaf(C[n], h[n], y);
        }
        if (s.gate) y *= z * sigmoid_fast(z);
        if (!c.active) continue;
#pragma unroll
        for (int n = 0; n < S; ++n)
            if (FULL || n < s.states) state[n * channels] = h[n];
        static_cast<T*>(s.out)[b * s.out_batch + c.d] = from_f32<T>(y);
    }
}

int scan_check(const ilx_state_space& s, const char* name) {
    ILX_REQUIRE(s.batch >= 0 && s.length >= 0 && s.channels > 0 && s.groups > 0, ILX_EINVAL, "%s: bad shape (%lld, %lld, %d), %d groups", name,
                (long long)s.batch, (long long)s.length, s.channels, s.groups);
    ILX_REQUIRE(s.channels % s.groups == 0, ILX_ESHAPE, "%s: %d channels do not split into %d groups", name, s.channels, s.groups);
    ILX_REQUIRE(s.states >= 1 && s.states <= ILX_SCAN_MAX_STATES, ILX_ESHAPE, "%s: %d states (1..%d supported)", name, s.states,
                ILX_SCAN_MAX_STATES);
    ILX_REQUIRE(s.dtype >= ILX_F32 && s.dtype <= ILX_F16, ILX_EINVAL, "%s: unknown type %d", name, s.dtype);
    ILX_REQUIRE(s.bc_dtype == ILX_F32 || s.bc_dtype == s.dtype, ILX_EINVAL, "%s: B and C of type %d beside activations of type %d", name,
                s.bc_dtype, s.dtype);
    ILX_REQUIRE(s.batch <= INT32_MAX && s.length <= INT32_MAX && s.batch * (s.length + 1) < (int64_t{1} << 40), ILX_ESHAPE,
                "%s: shape (%lld, %lld) too large", name, (long long)s.batch, (long long)s.length);
    if (s.bc_dtype != ILX_F32)
        ILX_REQUIRE(s.states % 2 == 0 && s.B_batch % 2 == 0 && s.B_time % 2 == 0 && s.C_batch % 2 == 0 && s.C_time % 2 == 0 && aligned_to(s.B, 4) &&
                        aligned_to(s.C, 4),
                    ILX_ESHAPE, "%s: 16-bit B and C are read in pairs: states, strides and pointers must be even", name);
    return ILX_OK;
}

ScanArgs scan_args(const ilx_state_space& s) {
    ScanArgs a{};
    a.s = s;
    a.group_channels = s.channels / s.groups;
    a.group_blocks = (a.group_channels + 63) / 64;
    a.blocks = s.groups * a.group_blocks;
    a.saved_blocks = (s.length + ILX_SCAN_BLOCK - 1) / ILX_SCAN_BLOCK;
    return a;
}

}  // namespace ilx

using namespace ilx;

namespace {

enum ScanKind { kForward, kStep };

template <typename T, typename TB, int S, bool FULL> void scan_launch(ScanKind kind, const ScanArgs& a, hipStream_t s) {
    if (kind == kStep)
        ILX_LAUNCH((scan_step_kernel<T, TB, S, FULL>), dim3(static_cast<unsigned>(a.slots * a.blocks)), dim3(64), 0, s, a);
    else
        ILX_LAUNCH((scan_forward_kernel<T, TB, S, FULL>), dim3(static_cast<unsigned>(a.s.batch * a.blocks)), dim3(64), 0, s, a);
}

template <typename T, typename TB> void scan_states(ScanKind kind, const ScanArgs& a, hipStream_t s) {
    const int n = a.s.states;
    if (n == 4) return scan_launch<T, TB, 4, true>(kind, a, s);
    if (n == 8) return scan_launch<T, TB, 8, true>(kind, a, s);
    if (n == 16) return scan_launch<T, TB, 16, true>(kind, a, s);
    if (n == 32) return scan_launch<T, TB, 32, true>(kind, a, s);
    if (n < 4) return scan_launch<T, TB, 4, false>(kind, a, s);
    if (n < 8) return scan_launch<T, TB, 8, false>(kind, a, s);
    if (n < 16) return scan_launch<T, TB, 16, false>(kind, a, s);
    scan_launch<T, TB, 32, false>(kind, a, s);
}

void scan_dispatch(ScanKind kind, const ScanArgs& a, hipStream_t s) {
    const bool wide = a.s.bc_dtype == ILX_F32;
    switch (a.s.dtype) {
        case ILX_F32: return scan_states<float, float>(kind, a, s);
        case ILX_BF16: return wide ? scan_states<bf16_t, float>(kind, a, s) : scan_states<bf16_t, bf16_t>(kind, a, s);
        default: return wide ? scan_states<f16_t, float>(kind, a, s) : scan_states<f16_t, f16_t>(kind, a, s);
    }
}

}  // namespace

extern "C" int ilx_state_space_forward(const ilx_state_space* scan, void* stream) {
    ILX_REQUIRE(scan, ILX_EINVAL, "ilx_state_space_forward: descriptor is NULL");
    const ilx_state_space& s = *scan;
    const int rc = scan_check(s, "ilx_state_space_forward");
    if (rc != ILX_OK) return rc;
    if (s.batch == 0) return ILX_OK;
    ILX_REQUIRE(s.A && (s.length == 0 || (s.x && s.delta && s.B && s.C && s.out)), ILX_EINVAL, "ilx_state_space_forward: NULL operand");
    ILX_REQUIRE(!s.last || s.last != s.state, ILX_EINVAL, "ilx_state_space_forward: last and state are the same buffer");
    const ScanArgs a = scan_args(s);
    ILX_REQUIRE(s.batch * a.blocks <= INT32_MAX, ILX_ESHAPE, "ilx_state_space_forward: shape too large for one launch");
    scan_dispatch(kForward, a, as_stream(stream));
    ILX_LAUNCH_CHECK("ilx_state_space_forward");
    return ILX_OK;
}

extern "C" int ilx_state_space_step(const ilx_state_space* scan, void* stream) {
    ILX_REQUIRE(scan, ILX_EINVAL, "ilx_state_space_step: descriptor is NULL");
    ilx_state_space s = *scan;
    s.length = 1;
    s.B_time = s.C_time = 0;
    const int rc = scan_check(s, "ilx_state_space_step");
    if (rc != ILX_OK) return rc;
    if (s.batch == 0) return ILX_OK;
    ILX_REQUIRE(s.x && s.delta && s.A && s.B && s.C && s.out && s.state, ILX_EINVAL, "ilx_state_space_step: NULL operand");
    ILX_REQUIRE(s.state == s.last, ILX_EINVAL, "ilx_state_space_step: the state is updated in place, last must be state");
    ILX_REQUIRE(!s.lengths && !s.saved, ILX_EINVAL, "ilx_state_space_step: lengths and saved must be NULL");
    ScanArgs a = scan_args(s);
    const int64_t most = 8192 / a.blocks > 0 ? 8192 / a.blocks : 1;
    a.slots = s.batch < most ? s.batch : most;
    ILX_REQUIRE(a.slots * a.blocks <= INT32_MAX, ILX_ESHAPE, "ilx_state_space_step: shape too large for one launch");
    scan_dispatch(kStep, a, as_stream(stream));
    ILX_LAUNCH_CHECK("ilx_state_space_step");
    return ILX_OK;
}
