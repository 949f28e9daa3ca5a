// Selective state space recurrence, forward and one step:
//   h[n] <- exp(dt A[n]) h[n] + dt B[n] x,   y = sum_n C[n] h[n] + D x,   dt = softplus(delta + bias)
// per channel, with B and C shared by the channels of a group.
// A lane owns a channel and all its states, a wave 64 channels: the recurrence needs no exchange between lanes, a row's x,
// delta, gate and out are one access of 64 neighbours each, and B and C come out of one register a row by broadcast.  Per state
// and row that leaves a multiply, an exponential (a quarter of the rate), a multiply by B and two multiply-adds.  The next four
// rows are on their way while four are worked on.
// Where that makes too few waves (few sequences, long ones), a sequence is divided into parts: every part runs from a zero state
// for what it adds to the state, a join passes the states through all parts (a part as a whole multiplies a state by
// exp(A sum dt)), and every part runs again from the state that enters it.  That costs a second pass of exponentials and buys
// up to 256 times the waves.
#include "state_space_dev.h"

namespace ilx {

constexpr int kScanRows = 4;    // rows whose inputs are in registers together; divides ILX_SCAN_BLOCK
constexpr int kMostParts = 256;

// One row's inputs as they are in memory.
template <typename T, typename TB, int W> struct ScanRow {
    T x, delta, gate;
    TB B[W], C[W];
};

template <typename T, typename TB, int S> struct ScanReader {
    static constexpr int W = (S + 15) / 16;
    const T *x, *delta, *gate;
    const TB *B, *C;
    int64_t x_time, delta_time, gate_time, B_time, C_time;
    int d, n[W];
    bool in[W];

    __device__ __forceinline__ ScanReader(const ScanArgs& a, const ChannelLane& c, int64_t b, int lane, const void* px, int64_t px_batch, int64_t px_time) {
        const ilx_state_space& s = a.s;
        x = static_cast<const T*>(px) + b * px_batch, x_time = px_time;
        delta = static_cast<const T*>(s.delta) + b * s.delta_batch, delta_time = s.delta_time;
        gate = s.gate ? static_cast<const T*>(s.gate) + b * s.gate_batch : nullptr, gate_time = s.gate_time;
        B = static_cast<const TB*>(s.B) + b * s.B_batch + c.group * s.states, B_time = s.B_time;
        C = static_cast<const TB*>(s.C) + b * s.C_batch + c.group * s.states, C_time = s.C_time;
        d = c.d;
#pragma unroll
        for (int k = 0; k < W; ++k) {
            const int at = 16 * k + (lane & 15);
            in[k] = at < s.states;
            n[k] = in[k] ? at : s.states - 1;
        }
    }
    template <bool WITH_B, bool WITH_C, bool WITH_GATE> __device__ __forceinline__ void read(ScanRow<T, TB, W>& r, uint32_t t) const {
        r.x = x[row_offset(t, x_time) + d];
        r.delta = delta[row_offset(t, delta_time) + d];
        if (WITH_GATE && gate) r.gate = gate[row_offset(t, gate_time) + d];
#pragma unroll
        for (int k = 0; k < W; ++k) {
            if (WITH_B) r.B[k] = B[row_offset(t, B_time) + n[k]];
            if (WITH_C) r.C[k] = C[row_offset(t, C_time) + n[k]];
        }
    }
    __device__ __forceinline__ float state_lane(const TB (&v)[W], int k) const { return in[k] ? to_f32(v[k]) : 0.0f; }
};

// h <- exp(dt A) h + u B  for all states of the lane
template <int S, int W> __device__ __forceinline__ void advance(float (&h)[S], const float (&A2)[S], const float (&B)[W], float dt, float u) {
    static_for<S>([&](auto i) {
        constexpr int n = i;
        h[n] = __builtin_fmaf(__builtin_amdgcn_exp2f(dt * A2[n]), h[n], u * from_lane<(n & 15)>(B[n >> 4]));
    });
}

template <int S, int W> __device__ __forceinline__ float dot(const float (&C)[W], const float (&h)[S], float y) {
    float y1 = 0.0f;
    if constexpr (S <= 16)
        dot_states(y, y1, C[0], h);
    else {
        dot_sixteen<0>(y, y1, C[0], h);
        dot_sixteen<16>(y, y1, C[1], h);
    }
    return y + y1;
}

template <typename T, typename TB, int S>
__global__ void __launch_bounds__(64) scan_forward_kernel(ScanArgs a) {
    constexpr int W = (S + 15) / 16;
    const int lane = threadIdx.x;
    const uint32_t item = blockIdx.x / a.blocks, parts = static_cast<uint32_t>(a.parts);
    const int64_t b = item / parts, part = item % parts;
    const ChannelLane c = channel_lane(a, blockIdx.x % a.blocks, lane);
    const ilx_state_space& s = a.s;
    const int64_t len = scan_length(s, b), channels = s.channels, begin = part * a.part_rows;
    const int64_t limit = begin + a.part_rows < s.length ? begin + a.part_rows : s.length, end = limit < len ? limit : len;
    float A2[S], h[S];
    const float* enters = a.parts > 1 ? a.part_state + static_cast<int64_t>(item) * s.states * channels : s.state ? s.state + b * s.states * channels : nullptr;
#pragma unroll
    for (int n = 0; n < S; ++n) {
        const bool in = n < s.states;
        A2[n] = in ? s.A[static_cast<int64_t>(c.d) * s.states + n] * kLog2e : 0.0f;
        h[n] = in && enters ? enters[n * channels + c.d] : 0.0f;
    }
    const float bias = s.delta_bias ? s.delta_bias[c.d] : 0.0f, skip = s.D ? s.D[c.d] : 0.0f;
    const ScanReader<T, TB, S> in(a, c, b, lane, s.x, s.x_batch, s.x_time);
    T* po = static_cast<T*>(s.out) + b * s.out_batch + c.d;
    ScanRow<T, TB, W> rows[kScanRows];
    auto read = [&](int64_t t0) {
#pragma unroll
        for (int i = 0; i < kScanRows; ++i)
            in.template read<true, true, true>(rows[i], static_cast<uint32_t>(t0 + i < end ? t0 + i : end - 1));
    };
    if (begin < end) read(begin);
    for (int64_t t0 = begin; t0 < end; t0 += kScanRows) {
        const int count = end - t0 < kScanRows ? static_cast<int>(end - t0) : kScanRows;
        float x[kScanRows], dt[kScanRows], z[kScanRows], B[kScanRows][W], C[kScanRows][W];
#pragma unroll
        for (int i = 0; i < kScanRows; ++i) {
            x[i] = to_f32(rows[i].x);
            dt[i] = to_f32(rows[i].delta) + bias;
            if (in.gate) z[i] = to_f32(rows[i].gate);
#pragma unroll
            for (int k = 0; k < W; ++k) B[i][k] = in.state_lane(rows[i].B, k), C[i][k] = in.state_lane(rows[i].C, k);
        }
        const uint64_t starts = start_bits(s, b, t0, count, lane);
        if (t0 + kScanRows < end) read(t0 + kScanRows);
        if (s.saved && t0 % ILX_SCAN_BLOCK == 0 && c.active) {
            float* save = s.saved + (b * a.saved_blocks + t0 / ILX_SCAN_BLOCK) * s.states * channels + c.d;
#pragma unroll
            for (int n = 0; n < S; ++n)
                if (n < s.states) save[n * channels] = h[n];
        }
        if (s.softplus) {
#pragma unroll
            for (int i = 0; i < kScanRows; ++i) dt[i] = softplus_f(dt[i]);
        }
#pragma unroll
        for (int i = 0; i < kScanRows; ++i) {
            if (i < count) {
                if (starts >> i & 1) {
#pragma unroll
                    for (int n = 0; n < S; ++n) h[n] = 0.0f;
                }
                advance(h, A2, B[i], dt[i], dt[i] * x[i]);
                float y = dot<S>(C[i], h, skip * x[i]);
                if (in.gate) y *= z[i] * sigmoid_fast(z[i]);
                if (c.active) po[row_offset(static_cast<uint32_t>(t0 + i), s.out_time)] = from_f32<T>(y);
            }
        }
    }
    if (!c.active) return;
    for (int64_t t = begin > len ? begin : len; t < limit; ++t) po[t * s.out_time] = from_f32<T>(0.0f);
    if (s.last && ((begin < len && len <= limit) || (len == 0 && part == 0))) {   // the part that ends the sequence
#pragma unroll
        for (int n = 0; n < S; ++n)
            if (n < s.states) s.last[(b * s.states + n) * channels + c.d] = h[n];
    }
}

// What a part of a sequence adds to the state, from zeros: forward the state behind it, backward (REVERSE) the gradient of the
// state ahead of it, r <- a (r + dy C) from its last row to its first.
template <typename T, typename TB, int S, bool REVERSE>
__global__ void __launch_bounds__(64) scan_part_kernel(ScanArgs a) {
    constexpr int W = (S + 15) / 16;
    const int lane = threadIdx.x;
    const uint32_t item = blockIdx.x / a.blocks, parts = static_cast<uint32_t>(a.parts);
    const int64_t b = item / parts, part = item % parts;
    const ChannelLane c = channel_lane(a, blockIdx.x % a.blocks, lane);
    const ilx_state_space& s = a.s;
    const int64_t len = scan_length(s, b), channels = s.channels, begin = part * a.part_rows;
    const int64_t limit = begin + a.part_rows < s.length ? begin + a.part_rows : s.length, end = limit < len ? limit : len;
    float A2[S], h[S], sum = 0.0f;
    bool any = false;
#pragma unroll
    for (int n = 0; n < S; ++n) {
        A2[n] = n < s.states ? s.A[static_cast<int64_t>(c.d) * s.states + n] * kLog2e : 0.0f;
        h[n] = 0.0f;
    }
    const float bias = s.delta_bias ? s.delta_bias[c.d] : 0.0f;
    const ScanReader<T, TB, S> in(a, c, b, lane, REVERSE ? s.grad_out : s.x, REVERSE ? s.grad_out_batch : s.x_batch, REVERSE ? s.grad_out_time : s.x_time);
    ScanRow<T, TB, W> rows[kScanRows];
    auto read = [&](int64_t t0) {
#pragma unroll
        for (int i = 0; i < kScanRows; ++i)
            in.template read<!REVERSE, REVERSE, REVERSE>(rows[i], static_cast<uint32_t>(t0 + i < end ? t0 + i : end - 1));
    };
    const int64_t steps = begin < end ? (end - begin + kScanRows - 1) / kScanRows : 0;
    if (steps > 0) read(begin + (REVERSE ? steps - 1 : 0) * kScanRows);
    for (int64_t j = 0; j < steps; ++j) {
        const int64_t t0 = begin + (REVERSE ? steps - 1 - j : j) * kScanRows;
        const int count = end - t0 < kScanRows ? static_cast<int>(end - t0) : kScanRows;
        float x[kScanRows], dt[kScanRows], z[kScanRows], M[kScanRows][W];
#pragma unroll
        for (int i = 0; i < kScanRows; ++i) {
            x[i] = to_f32(rows[i].x);
            dt[i] = to_f32(rows[i].delta) + bias;
            if (REVERSE && in.gate) z[i] = to_f32(rows[i].gate);
#pragma unroll
            for (int k = 0; k < W; ++k) M[i][k] = in.state_lane(REVERSE ? rows[i].C : rows[i].B, k);
        }
        const uint64_t starts = start_bits(s, b, t0, count, lane);
        any = any || starts != 0;
        if (j + 1 < steps) read(REVERSE ? t0 - kScanRows : t0 + kScanRows);
        if (s.softplus) {
#pragma unroll
            for (int i = 0; i < kScanRows; ++i) dt[i] = softplus_f(dt[i]);
        }
        if (REVERSE && in.gate) {
#pragma unroll
            for (int i = 0; i < kScanRows; ++i) x[i] *= z[i] * sigmoid_fast(z[i]);
        }
#pragma unroll
        for (int k = 0; k < kScanRows; ++k) {
            const int i = REVERSE ? kScanRows - 1 - k : k;
            if (i < count) {
                sum += dt[i];
                if (REVERSE) {
                    static_for<S>([&](auto m) {
                        constexpr int n = m;
                        h[n] = __builtin_amdgcn_exp2f(dt[i] * A2[n]) * (h[n] + x[i] * from_lane<(n & 15)>(M[i][n >> 4]));
                    });
                }
                if (starts >> i & 1) {
#pragma unroll
                    for (int n = 0; n < S; ++n) h[n] = 0.0f;
                }
                if (!REVERSE) advance(h, A2, M[i], dt[i], dt[i] * x[i]);
            }
        }
    }
    if (!c.active) return;
#pragma unroll
    for (int n = 0; n < S; ++n)
        if (n < s.states) a.part_state[(static_cast<int64_t>(item) * s.states + n) * channels + c.d] = h[n];
    a.part_decay[static_cast<int64_t>(item) * channels + c.d] = any ? __builtin_inff() : sum;
}

// Passes the states through the parts: part_state becomes what enters each part (backward: the gradient that enters it from
// the part behind).  64 states of a sequence to a workgroup, a sixteenth of the parts to each of its waves: a wave joins its own
// parts, the waves' joins meet in LDS, and each wave passes what enters it through its parts again, out of registers.
__global__ void __launch_bounds__(1024) scan_join_kernel(ScanArgs a, int backward, const float* first) {
    constexpr int kWaves = 16, kPer = kMostParts / kWaves;
    __shared__ float s_decay[kWaves][64], s_state[kWaves][64];
    const ilx_state_space& s = a.s;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int columns = s.states * s.channels, column_blocks = (columns + 63) / 64;
    const int64_t b = blockIdx.x / column_blocks;
    const int column = static_cast<int>(blockIdx.x % column_blocks) * 64 + lane;
    const bool active = column < columns;
    const int at = active ? column : columns - 1, n = at / s.channels, d = at - n * s.channels;
    const int parts = static_cast<int>(a.parts), per = (parts + kWaves - 1) / kWaves, p0 = w * per;
    const float A2 = s.A[static_cast<int64_t>(d) * s.states + n] * kLog2e;
    float decay[kPer], state[kPer];
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        const bool in = j < per && p0 + j < parts;
        const int64_t p = b * parts + (backward ? parts - 1 - (p0 + j) : p0 + j);
        decay[j] = in ? a.part_decay[p * s.channels + d] : 0.0f;
        state[j] = in ? a.part_state[p * columns + at] : 0.0f;
    }
    float D = 1.0f, H = 0.0f;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        decay[j] = decay[j] == __builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(decay[j] * A2);   // a start cuts: exactly 0
        H = decay[j] == 0.0f ? state[j] : __builtin_fmaf(decay[j], H, state[j]);
        D *= decay[j];
    }
    s_decay[w][lane] = D;
    s_state[w][lane] = H;
    __syncthreads();
    float h = first ? first[b * columns + at] : 0.0f;
    for (int k = 0; k < w; ++k) h = s_decay[k][lane] == 0.0f ? s_state[k][lane] : __builtin_fmaf(s_decay[k][lane], h, s_state[k][lane]);
    if (!active) return;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        if (j < per && p0 + j < parts) {
            const int64_t p = b * parts + (backward ? parts - 1 - (p0 + j) : p0 + j);
            a.part_state[p * columns + at] = h;
            h = decay[j] == 0.0f ? state[j] : __builtin_fmaf(decay[j], h, state[j]);
        }
    }
}

// One row per sequence: the recurrence above with sequences in the place of rows, so that A stays in registers.  Bound by
// the state, read and written once.
template <typename T, typename TB, int S>
__global__ void __launch_bounds__(64) scan_step_kernel(ScanArgs a) {
    constexpr int W = (S + 15) / 16;
    const int lane = threadIdx.x;
    const ChannelLane c = channel_lane(a, blockIdx.x % a.blocks, lane);
    const ilx_state_space& s = a.s;
    const int64_t channels = s.channels;
    float A2[S];
#pragma unroll
    for (int n = 0; n < S; ++n) A2[n] = n < s.states ? s.A[static_cast<int64_t>(c.d) * s.states + n] * kLog2e : 0.0f;
    const float bias = s.delta_bias ? s.delta_bias[c.d] : 0.0f, skip = s.D ? s.D[c.d] : 0.0f;
    for (int64_t b = blockIdx.x / a.blocks; b < s.batch; b += a.slots) {
        float h[S], B[W], C[W];
        float* state = s.last + b * s.states * channels + c.d;
#pragma unroll
        for (int n = 0; n < S; ++n) h[n] = n < s.states ? state[n * channels] : 0.0f;
        const ScanReader<T, TB, S> in(a, c, b, lane, s.x, s.x_batch, 0);
        ScanRow<T, TB, W> row;
        in.template read<true, true, true>(row, 0);
        const bool start = s.starts && s.starts[b * s.starts_batch];
#pragma unroll
        for (int k = 0; k < W; ++k) B[k] = in.state_lane(row.B, k), C[k] = in.state_lane(row.C, k);
        const float x = to_f32(row.x);
        float dt = to_f32(row.delta) + bias;
        if (s.softplus) dt = softplus_f(dt);
        if (start) {
#pragma unroll
            for (int n = 0; n < S; ++n) h[n] = 0.0f;
        }
        advance(h, A2, B, dt, dt * x);
        float y = dot<S>(C, h, skip * x);
        if (in.gate) {
            const float z = to_f32(row.gate);
            y *= z * sigmoid_fast(z);
        }
        if (!c.active) continue;
#pragma unroll
        for (int n = 0; n < S; ++n)
            if (n < s.states) state[n * channels] = h[n];
        static_cast<T*>(s.out)[b * s.out_batch + c.d] = from_f32<T>(y);
    }
}

int scan_check(const ilx_state_space& s, const char* name) {
    ILX_REQUIRE(s.batch >= 0 && s.length >= 0 && s.channels > 0 && s.groups > 0, ILX_EINVAL, "%s: bad shape (%lld, %lld, %d), %d groups", name,
                (long long)s.batch, (long long)s.length, s.channels, s.groups);
    ILX_REQUIRE(s.channels % s.groups == 0, ILX_ESHAPE, "%s: %d channels do not split into %d groups", name, s.channels, s.groups);
    ILX_REQUIRE(s.states >= 1 && s.states <= ILX_SCAN_MAX_STATES, ILX_ESHAPE, "%s: %d states (1..%d supported)", name, s.states,
                ILX_SCAN_MAX_STATES);
    ILX_REQUIRE(s.channels <= INT32_MAX / ILX_SCAN_MAX_STATES - 64, ILX_ESHAPE, "%s: %d channels", name, s.channels);
    ILX_REQUIRE(s.dtype >= ILX_F32 && s.dtype <= ILX_F16, ILX_EINVAL, "%s: unknown type %d", name, s.dtype);
    ILX_REQUIRE(s.bc_dtype == ILX_F32 || s.bc_dtype == s.dtype, ILX_EINVAL, "%s: B and C of type %d beside activations of type %d", name,
                s.bc_dtype, s.dtype);
    ILX_REQUIRE(s.batch <= INT32_MAX && s.length <= INT32_MAX - 64 && s.batch * (s.length + 1) < (int64_t{1} << 40), ILX_ESHAPE,
                "%s: shape (%lld, %lld) too large", name, (long long)s.batch, (long long)s.length);
    if (s.length > 1)
        for (const int64_t stride : {s.x_time, s.delta_time, s.gate_time, s.B_time, s.C_time, s.out_time, s.grad_out_time, s.grad_time})
            ILX_REQUIRE(stride >= 0 && stride <= UINT32_MAX, ILX_ESHAPE, "%s: a time stride of %lld elements", name, (long long)stride);
    return ILX_OK;
}

ScanArgs scan_args(const ilx_state_space& s) {
    ScanArgs a{};
    a.s = s;
    a.group_channels = s.channels / s.groups;
    a.group_blocks = (a.group_channels + 63) / 64;
    a.blocks = s.groups * a.group_blocks;
    a.saved_blocks = (s.length + ILX_SCAN_BLOCK - 1) / ILX_SCAN_BLOCK;
    a.parts = 1, a.part_rows = s.length;
    return a;
}

// Two waves per SIMD hide a row's latency well enough that a second pass does not pay; below that a sequence is divided towards
// four per SIMD, in parts of at least 32 rows (a part's cost ahead of its first row is that of about eight).
int64_t divide_scan(ScanArgs& a, float* workspace) {
    const ilx_state_space& s = a.s;
    const int64_t waves = s.batch * a.blocks, full = 4 * device_cu_count();   // one per SIMD
    if (waves == 0 || waves >= 2 * full || s.length < 64) return 0;
    int64_t parts = 4 * full / waves;
    if (parts > kMostParts) parts = kMostParts;
    int64_t rows = (s.length + parts - 1) / parts;
    if (rows < 32) rows = 32;
    rows = (rows + ILX_SCAN_BLOCK - 1) / ILX_SCAN_BLOCK * ILX_SCAN_BLOCK;
    a.part_rows = rows, a.parts = (s.length + rows - 1) / rows;
    if (a.parts == 1) return 0;
    const int64_t states = s.batch * a.parts * s.states * s.channels, decays = s.batch * a.parts * s.channels;
    a.part_state = workspace, a.part_decay = workspace + states;
    return states + decays;
}

}  // namespace ilx

using namespace ilx;

namespace {

enum ScanKind { kForward, kStep, kParts, kPartsBackward };

template <typename T, typename TB, int S> void scan_launch(ScanKind kind, const ScanArgs& a, hipStream_t s) {
    const dim3 grid(static_cast<unsigned>(kind == kStep ? a.slots * a.blocks : a.s.batch * a.parts * a.blocks)), threads(64);
    switch (kind) {
        case kStep: ILX_LAUNCH((scan_step_kernel<T, TB, S>), grid, threads, 0, s, a); break;
        case kParts: ILX_LAUNCH((scan_part_kernel<T, TB, S, false>), grid, threads, 0, s, a); break;
        case kPartsBackward: ILX_LAUNCH((scan_part_kernel<T, TB, S, true>), grid, threads, 0, s, a); break;
        default: ILX_LAUNCH((scan_forward_kernel<T, TB, S>), grid, threads, 0, s, a); break;
    }
}

template <typename T, typename TB> void scan_states(ScanKind kind, const ScanArgs& a, hipStream_t s) {
    const int n = a.s.states;
    if (n <= 4) return scan_launch<T, TB, 4>(kind, a, s);
    if (n <= 8) return scan_launch<T, TB, 8>(kind, a, s);
    if (n <= 16) return scan_launch<T, TB, 16>(kind, a, s);
    scan_launch<T, TB, 32>(kind, a, s);
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

void ilx::launch_part_states(const ScanArgs& a, bool backward, hipStream_t s) {
    scan_dispatch(backward ? kPartsBackward : kParts, a, s);
    const int64_t column_blocks = (static_cast<int64_t>(a.s.states) * a.s.channels + 63) / 64;
    ILX_LAUNCH(scan_join_kernel, dim3(static_cast<unsigned>(a.s.batch * column_blocks)), dim3(1024), 0, s, a, backward ? 1 : 0,
               backward ? a.s.grad_last : a.s.state);
}

extern "C" int ilx_state_space_forward(const ilx_state_space* scan, void* stream) {
    ILX_REQUIRE(scan, ILX_EINVAL, "ilx_state_space_forward: descriptor is NULL");
    const ilx_state_space& s = *scan;
    const int rc = scan_check(s, "ilx_state_space_forward");
    if (rc != ILX_OK) return rc;
    if (s.batch == 0) return ILX_OK;
    ILX_REQUIRE(s.A && (s.length == 0 || (s.x && s.delta && s.B && s.C && s.out)), ILX_EINVAL, "ilx_state_space_forward: NULL operand");
    ILX_REQUIRE(!s.last || s.last != s.state, ILX_EINVAL, "ilx_state_space_forward: last and state are the same buffer");
    ScanArgs a = scan_args(s);
    const int64_t needed = divide_scan(a, s.workspace);
    ILX_REQUIRE(needed == 0 || (s.workspace && s.workspace_floats >= needed), ILX_EINVAL,
                "ilx_state_space_forward: workspace of %lld floats, %lld needed", (long long)s.workspace_floats, (long long)needed);
    ILX_REQUIRE(s.batch * a.parts * a.blocks <= INT32_MAX, ILX_ESHAPE, "ilx_state_space_forward: shape too large for one launch");
    if (a.parts > 1) launch_part_states(a, false, as_stream(stream));
    scan_dispatch(kForward, a, as_stream(stream));
    ILX_LAUNCH_CHECK("ilx_state_space_forward");
    return ILX_OK;
}

extern "C" int ilx_state_space_step(const ilx_state_space* scan, void* stream) {
    ILX_REQUIRE(scan, ILX_EINVAL, "ilx_state_space_step: descriptor is NULL");
    ilx_state_space s = *scan;
    s.length = 1;
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
