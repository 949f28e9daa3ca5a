// Backward pass of the selective state space recurrence.  With dy the gradient of y (before the gate) and r_t that of h_t,
//   r_t[n] = dy_t C_t[n] + a_{t+1}[n] r_{t+1}[n],   a_t = exp(dt_t A) (0 at a start),   q_t = a_t r_t h_{t-1},
//   dB_t[n] = sum_d r dt x,   dC_t[n] = sum_d dy h,   dA[n] = sum_t q dt,   dx = D dy + dt sum_n r B,
//   d dt = x sum_n r B + sum_n q A,   d delta = d dt sigmoid(delta + bias).
// The states are not kept by the forward pass (they are `states` times the inputs); it saves one in ILX_SCAN_BLOCK rows, and a
// wave recomputes a block's forward from there, a and h of all its rows in registers, then walks it backwards.
// A wave holds 16 channels times four quarters of the states: lane l has channel l % 16 and S states from S (l / 16) on.  So
// everything a row needs stays inside the wave:
//  * a row's dt, dt x and dy are made once, by the quarter of lanes whose turn the row is, and reach the others through LDS
//    without a barrier; the same lanes finish the row (dx, d delta, d gate);
//  * sums over the states (sum r B, sum q A, y) are added over the four quarters for four rows together, by exchanges that leave
//    each quarter its own row: three exchanges for four sums;
//  * sums over the channels (dB, dC) are first halved twice inside 16 lanes, each step leaving half of the lanes one value and
//    half another (twelve adds for eight values, where a plain tree takes 32); what is left, 16 numbers of a workgroup's four waves
//    (64 channels) to a result, is added from LDS behind the block's one barrier.
// Measured, 24 x 4096 x 256 f32 with gate and 16 states: 378 us (351 to 436 from pass to pass; and 15 for the sums of dB and dC over blocks
// of channels, 6 for the parameters), 0.97 GB, 2.6 TB/s.  Bound by instructions: 89 in the vector unit for a row and wave (four states a
// lane), which is busy 72 % of the time with three waves on a SIMD.  Waiting for reads behind the stores costs 10 us, running pointers in
// the place of the arguments read again 30 (they spill).
#include "state_space_dev.h"

namespace ilx {

constexpr int kRows = ILX_SCAN_BLOCK;
constexpr int kWaves = 4;
constexpr int kChannels = 16;   // per wave
constexpr int kChainBlocks = kChainRows / kRows;
constexpr float kLn2 = 0.693147180559945309417f;
static_assert(kRows == 8, "two sets of four rows");

__device__ __forceinline__ uint32_t bits(float v) { return __builtin_bit_cast(uint32_t, v); }
__device__ __forceinline__ float number(uint32_t v) { return __builtin_bit_cast(float, v); }

// Lanes below 32 get a folded onto itself, lanes from 32 on b; the same between neighbouring 16 lanes.
__device__ __forceinline__ float fold32(float a, float b) {
    const auto r = __builtin_amdgcn_permlane32_swap(bits(a), bits(b), false, false);
    return number(r[0]) + number(r[1]);
}
__device__ __forceinline__ float fold16(float a, float b) {
    const auto r = __builtin_amdgcn_permlane16_swap(bits(a), bits(b), false, false);
    return number(r[0]) + number(r[1]);
}
// Four rows' sums over the four quarters of the lanes: quarter g gets row g's.
__device__ __forceinline__ float fold_rows(const float (&v)[4]) { return fold16(fold32(v[0], v[2]), fold32(v[1], v[3])); }

// Inside 16 lanes: lanes 0-7 get a folded onto itself, lanes 8-15 b; inside 8 lanes: 0-3 a, 4-7 b.
__device__ __forceinline__ float fold8(float a, float b) {
    float r;
    asm("s_nop 1\n"
        "v_add_f32_dpp %0, %1, %1 row_ror:8 row_mask:0xf bank_mask:0x3\n"
        "v_add_f32_dpp %0, %2, %2 row_ror:8 row_mask:0xf bank_mask:0xc\n"
        : "=&v"(r)
        : "v"(a), "v"(b));
    return r;
}
__device__ __forceinline__ float fold4(float a, float b) {
    float r;
    asm("s_nop 1\n"
        "v_add_f32_dpp %0, %1, %1 row_half_mirror row_mask:0xf bank_mask:0x5\n"
        "v_add_f32_dpp %0, %2, %2 row_half_mirror row_mask:0xf bank_mask:0xa\n"
        : "=&v"(r)
        : "v"(a), "v"(b));
    return r;
}
// Of 2 S values per lane: register k, lanes 4 b .. 4 b + 3 of every 16 hold parts of value 4 k + order(b).
__device__ __forceinline__ constexpr int bank_of(int value) { return (value & 1) * 2 + (value >> 1 & 1); }
template <int N, int R> __device__ __forceinline__ void halve_twice(const float (&v)[N], float (&out)[R]) {
    if constexpr (N == 2) {
        const float t = fold8(v[0], v[1]);
        out[0] = fold4(t, t);
    } else {
#pragma unroll
        for (int k = 0; k < R; ++k) out[k] = fold4(fold8(v[4 * k], v[4 * k + 1]), fold8(v[4 * k + 2], v[4 * k + 3]));
    }
}

// Operands out of lanes: row Q of four, the quarter's own states (state_space_dev.h).
template <int L> __device__ __forceinline__ float from_lane(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0x150 + L, 0xf, 0xf, true));
}
// h += values u
template <int Q, int S, int O> __device__ __forceinline__ void add_outer(float (&h)[S], const float (&values)[O], float u) {
    if constexpr (S >= 4) {
#pragma unroll
        for (int m = 0; m < O; ++m) {
            f32x4 c = {h[4 * m], h[4 * m + 1], h[4 * m + 2], h[4 * m + 3]};
            c = __builtin_amdgcn_mfma_f32_4x4x1f32(values[m], u, c, 2, Q, 0);
#pragma unroll
            for (int j = 0; j < 4; ++j) h[4 * m + j] = c[j];
        }
    } else {
        static_for<S>([&](auto j) { h[j] = __builtin_fmaf(from_lane<4 * Q + j>(values[0]), u, h[j]); });
    }
}
// sum of values h over the lane's states
template <int Q, int S, int O> __device__ __forceinline__ float dot_quarter(const float (&values)[O], const float (&h)[S]) {
    float y = 0.0f;
    if constexpr (S < 4) {
        static_for<S>([&](auto j) { y = __builtin_fmaf(from_lane<4 * Q + j>(values[0]), h[j], y); });
    } else {
#pragma unroll
        for (int m = 0; m < O; ++m)
            asm(ILX_WAIT
                "v_fmac_f32_dpp %0, %1, %2 row_newbcast:%6 row_mask:0xf bank_mask:0xf\n"
                "v_fmac_f32_dpp %0, %1, %3 row_newbcast:%7 row_mask:0xf bank_mask:0xf\n"
                "v_fmac_f32_dpp %0, %1, %4 row_newbcast:%8 row_mask:0xf bank_mask:0xf\n"
                "v_fmac_f32_dpp %0, %1, %5 row_newbcast:%9 row_mask:0xf bank_mask:0xf\n"
                "s_nop 1\n"   // (an exchange between lanes may not read it sooner)
                : "+&v"(y)
                : "v"(values[m]), "v"(h[4 * m]), "v"(h[4 * m + 1]), "v"(h[4 * m + 2]), "v"(h[4 * m + 3]), "n"(4 * Q), "n"(4 * Q + 1), "n"(4 * Q + 2),
                  "n"(4 * Q + 3));
    }
    return y;
}

// The state ahead of row I of a block.
template <int I, int S> __device__ __forceinline__ float before(const float (&h0)[S], const float (&h)[kRows][S], int j) {
    if constexpr (I == 0)
        return h0[j];
    else
        return h[I - 1][j];
}

// A block of rows of one part of a sequence.
struct ScanBlock {
    int item, b, begin, end, t0;   // begin .. end: the part's rows that exist
    int count;
};

template <typename T, typename TB, int S>
__global__ void __launch_bounds__(64 * kWaves, S == 8 ? 2 : 3) scan_backward_kernel(StateSpaceArgs a) {
    constexpr int O = (S + 3) / 4, R = S / 2 > 0 ? S / 2 : 1;
    __shared__ float4 s_row[kWaves][kRows][kChannels];   // dt, dt x, dy
    alignas(16) __shared__ float s_part[2][kWaves][R][kRows][64];    // halved sums of this block and the one before
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), quarter = lane >> 4;
    const int block = blockIdx.x % a.blocks, slot = blockIdx.x / a.blocks;
    const int group = block / a.group_blocks, group_block = block - group * a.group_blocks;
    const int within = group_block * 64 + w * kChannels + (lane & 15);
    const bool active = within < a.group_channels;
    const int d = group * a.group_channels + (active ? within : a.group_channels - 1);
    const ilx_state_space& s = a.s;
    const int states = s.states, channels = s.channels, items = static_cast<int>(s.batch * a.parts);
    const bool gated = s.gate != nullptr;
    float A2[S], dA[S];   // A2 = A log2 e
#pragma unroll
    for (int j = 0; j < S; ++j) {
        const int n = S * quarter + j;
        A2[j] = n < states ? s.A[static_cast<int64_t>(d) * states + n] * kLog2e : 0.0f;
        dA[j] = 0.0f;
    }
    float bias = s.delta_bias ? s.delta_bias[d] : 0.0f, skip = s.D ? s.D[d] : 0.0f;
    arrive(A2), arrive(bias), arrive(skip);
    float dD = 0.0f, dbias = 0.0f;
    // where the lane's values are: its channel, its quarter's states (clamped to the last), its element of the operands
    const uint32_t channel = static_cast<uint32_t>(d) * sizeof(T);
    uint32_t state_at[S];
#pragma unroll
    for (int j = 0; j < S; ++j) state_at[j] = (static_cast<uint32_t>(S * quarter + j < states ? S * quarter + j : states - 1) * channels + d) * 4;
    uint32_t operand_at[O], operand_mask[O];
#pragma unroll
    for (int m = 0; m < O; ++m) {
        const int i = 4 * m + (lane & 3), n = S * quarter + (i < S ? i : S - 1);
        operand_at[m] = (n < states ? n : states - 1) * sizeof(TB);
        operand_mask[m] = i < S && n < states ? ~0u : 0u;
    }

    // the last block of an item, with count 0 if the item has no rows
    auto item_end = [&](int item) {
        const ArgsPtr p = arguments_again();
        const int parts = static_cast<int>(p->parts), part_rows = static_cast<int>(p->part_rows);
        ScanBlock k;
        k.item = item, k.b = item / parts, k.begin = (item - k.b * parts) * part_rows;
        int len = static_cast<int>(p->s.length);
        if (p->s.lengths) {
            const int n = uni(p->s.lengths[k.b]);
            len = n < 0 ? 0 : (n < len ? n : len);
        }
        k.end = k.begin + part_rows < len ? k.begin + part_rows : len;
        k.t0 = k.begin < k.end ? k.begin + (k.end - k.begin - 1) / kRows * kRows : k.begin;
        k.count = k.begin < k.end ? k.end - k.t0 : 0;
        return k;
    };
    // a block's inputs, read while the block ahead of it in this order is worked on
    T in_d[2], in_x[2], in_g[2], in_z[2];
    TB in_B[2][O], in_C[2][O];
    float in_h[S];
    uint8_t in_start = 0;   // of row `lane` of the block
    auto read = [&](const ScanBlock& k) {
        const ArgsPtr p = arguments_again();
        Stream<T> x, delta, gate, grad;
        Stream<TB> B, C;
        x.set(p->s.x, k.b * p->s.x_batch, k.t0, p->s.x_time);
        delta.set(p->s.delta, k.b * p->s.delta_batch, k.t0, p->s.delta_time);
        grad.set(p->s.grad_out, k.b * p->s.grad_out_batch, k.t0, p->s.grad_out_time);
        B.set(p->s.B, k.b * p->s.B_batch + group * p->s.states, k.t0, p->s.B_time);
        C.set(p->s.C, k.b * p->s.C_batch + group * p->s.states, k.t0, p->s.C_time);
        if (p->s.gate)
            gate.set(p->s.gate, k.b * p->s.gate_batch, k.t0, p->s.gate_time);
        else
            gate = grad;   // (read and not used)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const uint32_t row = 4 * e + quarter < k.count ? 4 * e + quarter : k.count - 1;
            in_d[e] = lane_load<T>(delta.buffer(), row * delta.time + channel, 0);
            in_x[e] = lane_load<T>(x.buffer(), row * x.time + channel, 0);
            in_g[e] = lane_load<T>(grad.buffer(), row * grad.time + channel, 0);
            in_z[e] = lane_load<T>(gate.buffer(), row * gate.time + channel, 0);
            const int q = 4 * e + (lane >> 2 & 3);
            const uint32_t operand_row = q < k.count ? q : k.count - 1;
#pragma unroll
            for (int m = 0; m < O; ++m) {
                in_B[e][m] = lane_load<TB>(B.buffer(), operand_row * B.time + operand_at[m], 0);
                in_C[e][m] = lane_load<TB>(C.buffer(), operand_row * C.time + operand_at[m], 0);
            }
        }
        const auto save = row_buffer(p->s.saved + (k.b * p->saved_blocks + k.t0 / kRows) * (static_cast<int64_t>(p->s.states) * p->s.channels));
#pragma unroll
        for (int j = 0; j < S; ++j) in_h[j] = lane_load<float>(save, state_at[j], 0);
        in_start = 0;
        if (p->s.starts && lane < k.count) in_start = (p->s.starts + k.b * p->s.starts_batch + k.t0 * p->s.starts_time)[lane * p->s.starts_time];
    };

    auto arrived = [&] {
        arrive(in_d), arrive(in_x), arrive(in_g), arrive(in_z), arrive(in_h), arrive(in_start);
#pragma unroll
        for (int e = 0; e < 2; ++e) arrive(in_B[e]), arrive(in_C[e]);
    };

    // a row of the workgroup's partial sums of the parameters' gradients
    int chain = 0, summed = 0;   // rows written; blocks in the sums
    auto end_chain = [&] {
        const ArgsPtr p = arguments_again();
        dD = fold32(dD, dD), dbias = fold32(dbias, dbias);
        dD = fold16(dD, dD), dbias = fold16(dbias, dbias);
        const uint32_t n = p->s.states, row = p->s.channels * 4;
        const auto to = row_buffer(p->sums + (slot * p->chains + chain) * (static_cast<int64_t>(n) + 2) * p->s.channels);
        if (active) {
#pragma unroll
            for (int j = 0; j < S; ++j)
                if (S * quarter + j < n) lane_store<float>(to, state_at[j], 0, dA[j]);
            uint32_t at = channel;   // (made here: the compiler would hold the channel's offset in another register through all rows)
            asm volatile("" : "+v"(at));
            at *= 4 / sizeof(T);
            if (quarter == 0) lane_store<float>(to, at, n * row, dD), lane_store<float>(to, at, (n + 1) * row, dbias);
        }
#pragma unroll
        for (int j = 0; j < S; ++j) dA[j] = 0.0f;
        dD = 0.0f, dbias = 0.0f;
        ++chain, summed = 0;
    };

    ScanBlock k = item_end(slot);
    if (k.count > 0) {
        read(k);
        arrived();
    }
    float r[S];
    bool fresh = true;
    int buffer = 0;
    while (k.item < items) {
        if (fresh) {   // the item's last block: what enters the part from behind, and zeros for the rows that do not exist
            const ArgsPtr p = arguments_again();
            const int64_t size = static_cast<int64_t>(p->s.states) * p->s.channels;
            const float* enters = p->parts > 1 ? p->part_state + k.item * size : p->s.grad_last ? p->s.grad_last + k.b * size : nullptr;
#pragma unroll
            for (int j = 0; j < S; ++j) r[j] = 0.0f;
            if (enters) {
                const auto from = row_buffer(enters);
#pragma unroll
                for (int j = 0; j < S; ++j) r[j] = active && S * quarter + j < states ? lane_load<float>(from, state_at[j], 0) : 0.0f;
                arrive(r);
            }
            const int length = static_cast<int>(p->s.length), part_rows = static_cast<int>(p->part_rows), limit = k.begin + part_rows < length ? k.begin + part_rows : length;
            for (int t = (k.end > k.begin ? k.end : k.begin) + quarter; t < limit; t += 4) {
                const int64_t at = k.b * p->s.grad_batch + t * p->s.grad_time + d;
                if (!active) break;
                static_cast<T*>(p->s.grad_x)[at] = from_f32<T>(0.0f);
                static_cast<T*>(p->s.grad_delta)[at] = from_f32<T>(0.0f);
                if (gated) static_cast<T*>(p->s.grad_gate)[at] = from_f32<T>(0.0f);
            }
        }
        ScanBlock next = k;
        if (k.t0 > k.begin) {
            next.t0 = k.t0 - kRows, next.count = kRows;
        } else if (k.item + static_cast<int>(a.slots) < items) {
            next = item_end(k.item + static_cast<int>(a.slots));
        } else {
            next.item = items, next.count = 0;
        }
        if (k.count > 0) {
            if (summed == kChainBlocks) end_chain();
            ++summed;
            // rows past the end act as rows that leave the state alone: dt = x = dy = 0
            float slope[2], dgate[2], x[2], dt[2], dy[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const bool in = 4 * e + quarter < k.count && active;
                const float raw = to_f32(in_d[e]) + bias, g = to_f32(in_g[e]);
                x[e] = in ? to_f32(in_x[e]) : 0.0f;
                dy[e] = g, dgate[e] = 0.0f, slope[e] = 1.0f, dt[e] = raw;
                if (gated) {
                    const float z = to_f32(in_z[e]), sig = sigmoid_fast(z);
                    dy[e] = g * z * sig;
                    dgate[e] = g * sig * __builtin_fmaf(z, 1.0f - sig, 1.0f);
                }
                if (s.softplus) slope[e] = sigmoid_fast(raw), dt[e] = softplus_f(raw);
                dy[e] = in ? dy[e] : 0.0f, dt[e] = in ? dt[e] : 0.0f;
                s_row[w][4 * e + quarter][lane & 15] = make_float4(dt[e], dt[e] * x[e], dy[e], 0.0f);
            }
            float B[2][O], C[2][O], h0[S], decay[kRows][S], h[kRows][S];
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
                for (int m = 0; m < O; ++m) B[e][m] = masked(to_f32(in_B[e][m]), operand_mask[m]), C[e][m] = masked(to_f32(in_C[e][m]), operand_mask[m]);
#pragma unroll
            for (int j = 0; j < S; ++j) h0[j] = in_h[j];
            const uint32_t starts = static_cast<uint32_t>(__ballot(in_start != 0));
            if (next.count > 0) read(next);
            float y[2], rb[2], ra[2];
            auto walk = [&](auto with_starts) {
                float four[4], four_a[4];
                static_for<kRows>([&](auto row) {
                    constexpr int i = row;
                    const float4 v = s_row[w][i][lane & 15];
                    const bool start = decltype(with_starts)::value && (starts >> i & 1);
                    if (start) {
                        asm volatile("; an episode starts");   // (a branch, not selects: nearly no row takes it)
                        static_for<S>([&](auto j) { decay[i][j] = 0.0f, h[i][j] = 0.0f; });
                    } else {
                        static_for<S>([&](auto j) {
                            decay[i][j] = __builtin_amdgcn_exp2f(v.x * A2[j]);
                            h[i][j] = decay[i][j] * before<i>(h0, h, j);
                        });
                    }
                    add_outer<(i & 3)>(h[i], B[i >> 2], v.y);
                    four[i & 3] = dot_quarter<(i & 3)>(C[i >> 2], h[i]);
                    if constexpr ((i & 3) == 3) y[i >> 2] = fold_rows(four);
                });
                uint32_t starts_again = starts;   // (kept apart: the compiler would hold what the two walks share in registers)
                asm volatile("" : "+s"(starts_again) : : "memory");
                static_for<kRows>([&](auto row) {
                    constexpr int i = kRows - 1 - row;
                    const float4 u = s_row[w][i][lane & 15];
                    const bool start = decltype(with_starts)::value && (starts_again >> i & 1);
                    float v[2 * S], sums[R];
                    add_outer<(i & 3)>(r, C[i >> 2], u.z);
                    four[i & 3] = dot_quarter<(i & 3)>(B[i >> 2], r);
                    four_a[i & 3] = 0.0f;
#pragma unroll
                    for (int j = 0; j < S; ++j) {
                        v[j] = r[j] * u.y;
                        v[S + j] = u.z * h[i][j];
                    }
                    if (start) {
                        asm volatile("; an episode starts");
                        static_for<S>([&](auto j) { r[j] = 0.0f; });
                    } else {
                        static_for<S>([&](auto j) {
                            r[j] *= decay[i][j];
                            const float q = r[j] * before<i>(h0, h, j);
                            four_a[i & 3] = __builtin_fmaf(q, A2[j], four_a[i & 3]);
                            dA[j] = __builtin_fmaf(q, u.x, dA[j]);
                        });
                    }
                    halve_twice(v, sums);
#pragma unroll
                    for (int m = 0; m < R; ++m) s_part[buffer][w][m][i][lane] = sums[m];
                    if constexpr ((i & 3) == 0) rb[i >> 2] = fold_rows(four), ra[i >> 2] = fold_rows(four_a);
                });
            };
            if (starts)
                walk(std::true_type{});
            else
                walk(std::false_type{});
            arrived();
            {
                const ArgsPtr p = arguments_again();
                const uint32_t time = static_cast<uint32_t>(p->s.grad_time) * sizeof(T);
                const int64_t at = k.b * p->s.grad_batch + static_cast<int64_t>(k.t0) * p->s.grad_time;
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int i = 4 * e + quarter;
                    if (i < k.count && active) {
                        const float draw = __builtin_fmaf(x[e], rb[e], ra[e] * kLn2) * slope[e];
                        const uint32_t to = i * time + channel;
                        lane_store<T>(row_buffer(static_cast<T*>(p->s.grad_x) + at), to, 0, from_f32<T>(__builtin_fmaf(dt[e], rb[e], skip * dy[e])));
                        lane_store<T>(row_buffer(static_cast<T*>(p->s.grad_delta) + at), to, 0, from_f32<T>(draw));
                        if (gated) lane_store<T>(row_buffer(static_cast<T*>(p->s.grad_gate) + at), to, 0, from_f32<T>(dgate[e] * __builtin_fmaf(skip, x[e], y[e])));
                        dD = __builtin_fmaf(dy[e], x[e], dD);
                        dbias += draw;
                    }
                }
            }
            __syncthreads();
            // dB and dC of the block's rows over the workgroup's channels
            float* to = a.shared + ((static_cast<int64_t>(group_block) * s.batch + k.b) * s.length + k.t0) * s.groups * (8 * S);
            for (int o = threadIdx.x; o < k.count * 8 * S; o += 64 * kWaves) {
                const int i = o / (8 * S), value = o - i * (8 * S), n = value % (4 * S), v = value / (4 * S) * S + n % S;
                const int at = 16 * (n / S) + 4 * bank_of(v & 3);
                float sum = 0.0f;
#pragma unroll
                for (int m = 0; m < kWaves; ++m) {
                    const float4 q = *reinterpret_cast<const float4*>(&s_part[buffer][m][v >> 2][i][at]);
                    sum += (q.x + q.y) + (q.z + q.w);
                }
                to[(static_cast<int64_t>(i) * s.groups + group) * (8 * S) + value] = sum;
            }
            buffer ^= 1;   // (this one is written again behind the next block's barrier)
        } else if (next.count > 0) {
            read(next);
            arrived();
        }
        fresh = next.item != k.item;
        if (fresh && k.begin == 0 && s.grad_state && active) {
#pragma unroll
            for (int j = 0; j < S; ++j)
                if (S * quarter + j < states) s.grad_state[k.b * static_cast<int64_t>(states) * channels + (state_at[j] >> 2)] = r[j];
        }
        k = next;
    }
    // the last sums, and zeros for the rows of partial sums that are left (sequences that end early)
    for (const int chains = static_cast<int>(a.chains); chain < chains;) end_chain();
}

// dB and dC: the sums of the blocks of channels of a group, in order and in 64 bits (there may be thousands of them); rows past a
// sequence's end are zeros.
template <typename TB> __global__ void __launch_bounds__(256) scan_shared_sums_kernel(StateSpaceArgs a, int padded) {
    const ilx_state_space& s = a.s;
    const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x, rows = s.batch * s.length * s.groups;
    if (i >= rows * s.states) return;
    const int64_t row = i / s.states;
    const int n = static_cast<int>(i - row * s.states);
    const int64_t bt = row / s.groups, b = bt / s.length, t = bt - b * s.length;
    double dB = 0.0, dC = 0.0;
    if (t < scan_length(s, b))
        for (int k = 0; k < a.group_blocks; ++k) {
            const float* p = a.shared + (k * rows + row) * 2 * padded + n;
            dB += static_cast<double>(p[0]);
            dC += static_cast<double>(p[padded]);
        }
    static_cast<TB*>(s.grad_B)[i] = from_f32<TB>(static_cast<float>(dB));
    static_cast<TB*>(s.grad_C)[i] = from_f32<TB>(static_cast<float>(dC));
}

}  // namespace ilx

using namespace ilx;

namespace {

int lane_states(int states) { return states <= 4 ? 1 : states <= 8 ? 2 : states <= 16 ? 4 : 8; }

StateSpaceArgs backward_args(const ilx_state_space& s, int64_t* floats) {
    StateSpaceArgs a = scan_args(s);
    const int64_t part_floats = divide_scan(a, s.workspace);
    // two workgroups in turn where three are resident, each with as many sequences as the next
    const int64_t items = s.batch * a.parts, wanted = 6 * device_cu_count(), most = wanted / a.blocks > 0 ? wanted / a.blocks : 1;
    const int64_t each = (items + most - 1) / most;
    a.slots = each > 0 ? (items + each - 1) / each : 0;
    const int64_t summed = each * ((a.part_rows + kRows - 1) / kRows);   // blocks of a workgroup
    a.chains = summed > kChainBlocks ? (summed + kChainBlocks - 1) / kChainBlocks : 1;
    const int64_t sums = a.slots * a.chains * (s.states + 2) * s.channels;
    const int64_t shared = a.group_blocks * s.batch * s.length * s.groups * 8 * lane_states(s.states);
    a.sums = s.workspace + part_floats;
    a.shared = a.sums + sums;
    *floats = part_floats + sums + shared;
    return a;
}

template <typename T, typename TB> void backward_states(const StateSpaceArgs& a, hipStream_t s) {
    const dim3 grid(static_cast<unsigned>(a.slots * a.blocks)), threads(64 * kWaves);
    const int each = lane_states(a.s.states);
    switch (each) {
        case 1: ILX_LAUNCH((scan_backward_kernel<T, TB, 1>), grid, threads, 0, s, a); break;
        case 2: ILX_LAUNCH((scan_backward_kernel<T, TB, 2>), grid, threads, 0, s, a); break;
        case 4: ILX_LAUNCH((scan_backward_kernel<T, TB, 4>), grid, threads, 0, s, a); break;
        default: ILX_LAUNCH((scan_backward_kernel<T, TB, 8>), grid, threads, 0, s, a); break;
    }
    const int64_t values = a.s.batch * a.s.length * a.s.groups * a.s.states;
    if (values > 0) ILX_LAUNCH((scan_shared_sums_kernel<TB>), dim3(blocks_for(values)), dim3(256), 0, s, a, 4 * each);
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
    ILX_REQUIRE(s.batch * a.parts * a.blocks <= INT32_MAX - 65536 && s.batch * s.length * s.groups * s.states < kMostThreads, ILX_ESHAPE,
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
    launch_parameter_sums(a.sums, a.slots * a.chains, s.channels, s.states, 2, s.grad_A, s.grad_D, s.grad_delta_bias, st);
    ILX_LAUNCH_CHECK("ilx_state_space_backward");
    return ILX_OK;
}
