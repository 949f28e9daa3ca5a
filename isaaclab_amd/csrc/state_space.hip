// Selective state space recurrence, forward and one step:
//   h[n] <- exp(dt A[n]) h[n] + dt B[n] x,   y = sum_n C[n] h[n] + D x,   dt = softplus(delta + bias)
// per channel, with B and C shared by the channels of a group.
// A lane owns a channel and all its states, a wave 64 channels: the recurrence needs no exchange between lanes, a row's x,
// delta, gate and out are one access of 64 neighbours each, and B and C enter from lanes (state_space_dev.h).  Per state and row
// that leaves a multiply, an exponential (a third to a quarter of the rate), a multiply, a quarter of a matrix instruction and a
// multiply-add.  The next four rows, of this sequence or the wave's next, are on their way while four are worked on.
// Where that makes too few waves (few sequences, long ones), a sequence is divided into parts: every part runs from a zero state
// for what it adds to the state, a join passes the states through all parts (a part as a whole multiplies a state by
// exp(A sum dt)), and every part runs again from the state that enters it.  That costs a second pass of exponentials and buys
// up to 256 times the waves.
// Measured with 16 states, against a large copy's 4.97 TB/s:
//   24 x 4096 x 256 f32, gate, state in and out: 133 us, 537 MB, 4.0 TB/s; with the states a backward pass needs 142 us, 738 MB, 5.2
//   TB/s: bound by memory
//   1 x 16384 x 1024 bf16 in 256 parts: 60 us for the parts, 11 for the join, 82 for the rows; 134 MB of operands, so bound by the
//   vector unit (part kernel: 78 instructions a row and wave, 52 of them the recurrence; the unit is busy 76 % of the time)
//   undivided, the same call takes 19 ms
//   step, 16384 x 256 bf16: 113 us on states that are not cached (571 MB, 5.1 TB/s), 91 in a loop on one state
#include "state_space_dev.h"
#include "uniform_access.h"

namespace ilx {

constexpr int kScanRows = 4;    // rows whose inputs are in registers together; divides ILX_SCAN_BLOCK
constexpr int kMostParts = 256;
constexpr int kJoinParts = 16;   // of a wave in the join
constexpr int kScanWaves = 4;   // to a workgroup: independent, but a workgroup puts one on each SIMD of its CU (single waves end up
                                // unevenly: two thirds of the waves that fit were resident on average)

__device__ __forceinline__ int wave_unit() { return uni(static_cast<int>(blockIdx.x * kScanWaves + (threadIdx.x >> 6))); }

enum { kHasGate = 1, kSoftplus = 2, kHasStarts = 4 };

// What stays in scalar registers through a wave's life; all else is read again where an item begins (arguments_again).
template <typename T, typename TB> struct ScanStreams {
    Stream<T> x, delta, gate;   // at the rows that are read next
    Stream<TB> o, c;            // operand of `outer` and of `dot`
    Stream<uint8_t> starts;
    int flags;
    int item, b, begin, end, t0;   // the item that is read, its rows that exist, the next row

    template <bool REVERSE> __device__ __forceinline__ void open(int which, int group) {
        const ArgsPtr a = arguments_again();
        const int parts = static_cast<int>(a->parts), rows = static_cast<int>(a->part_rows);
        item = which, b = item / parts, begin = (item - b * parts) * rows;
        int len = static_cast<int>(a->s.length);
        if (a->s.lengths) {
            const int n = uni(a->s.lengths[b]);
            len = n < 0 ? 0 : (n < len ? n : len);
        }
        end = begin + rows < len ? begin + rows : len;
        t0 = REVERSE && begin < end ? begin + (end - 1 - begin) / kScanRows * kScanRows : begin;
        if (REVERSE)
            x.set(a->s.grad_out, b * a->s.grad_out_batch, t0, a->s.grad_out_time), o.set(a->s.C, b * a->s.C_batch + group * a->s.states, t0, a->s.C_time);
        else
            x.set(a->s.x, b * a->s.x_batch, t0, a->s.x_time), o.set(a->s.B, b * a->s.B_batch + group * a->s.states, t0, a->s.B_time);
        delta.set(a->s.delta, b * a->s.delta_batch, t0, a->s.delta_time);
        if (a->s.gate)
            gate.set(a->s.gate, b * a->s.gate_batch, t0, a->s.gate_time);
        else
            gate = delta;   // (read and not used)
        c.set(a->s.C, b * a->s.C_batch + group * a->s.states, t0, a->s.C_time);
        starts.set(a->s.starts, b * a->s.starts_batch, t0, a->s.starts_time);
    }
    __device__ __forceinline__ int count() const { return end - t0 < kScanRows ? end - t0 : kScanRows; }
    template <bool REVERSE> __device__ __forceinline__ void step() {
        constexpr int n = REVERSE ? -kScanRows : kScanRows;
        x.step(n), delta.step(n), gate.step(n), o.step(n), c.step(n), starts.step(n);
        t0 += n;
    }
};

// The inputs of four rows, read while the four rows ahead of them are worked on.
template <typename T, typename TB, int W, bool WITH_GATE, bool WITH_DOT> struct ScanRows {
    T x[kScanRows], delta[kScanRows], gate[kScanRows];
    TB o[W], c[kScanRows][W];
    uint8_t start;   // of row `lane`

    // channel: the lane's channel, o_state, c_state: its states of the operands of `outer` and `dot`, all in bytes
    __device__ __forceinline__ void read(const ScanStreams<T, TB>& k, uint32_t channel, const uint32_t (&o_state)[W], const uint32_t (&c_state)[W], int lane) {
        const int count = k.count();
        const auto bx = k.x.buffer(), bd = k.delta.buffer(), bz = k.gate.buffer(), bo = k.o.buffer(), bc = k.c.buffer();
#pragma unroll
        for (int i = 0; i < kScanRows; ++i) {
            const uint32_t r = i < count ? i : count - 1;
            x[i] = lane_load<T>(bx, channel, r * k.x.time);
            delta[i] = lane_load<T>(bd, channel, r * k.delta.time);
            if (WITH_GATE) gate[i] = lane_load<T>(bz, channel, r * k.gate.time);
            if (WITH_DOT) {
#pragma unroll
                for (int j = 0; j < W; ++j) c[i][j] = lane_load<TB>(bc, c_state[j], r * k.c.time);
            }
        }
        const int at = lane >> 2 & 3;
        const uint32_t row = (at < count ? at : count - 1) * k.o.time;
#pragma unroll
        for (int j = 0; j < W; ++j) o[j] = lane_load<TB>(bo, row + o_state[j], 0);
        start = 0;
        if ((k.flags & kHasStarts) && lane < count) start = k.starts.p[lane * k.starts.time];
    }
    __device__ __forceinline__ void arrived() {
        arrive(x), arrive(delta), arrive(o), arrive(start);
        if (WITH_GATE) arrive(gate);
        if (WITH_DOT) {
#pragma unroll
            for (int i = 0; i < kScanRows; ++i) arrive(c[i]);
        }
    }
    __device__ __forceinline__ uint32_t starts() const { return static_cast<uint32_t>(__ballot(start != 0)); }   // a bit a row
};

// A start: a branch of its own, taken rarely, and no selects on the way past it.
template <int V> __device__ __forceinline__ void forget_if(bool start, f32x4 (&h)[V]) {
    if (start) {
        asm volatile("; an episode starts");
#pragma unroll
        for (int m = 0; m < V; ++m) h[m] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
}

// h <- exp(dt A) h + u B for all states of the lane; B from row ROW of the outer operand
template <int ROW, int V, int W> __device__ __forceinline__ void advance(f32x4 (&h)[V], const f32x4 (&A2)[V], const float (&B)[W], float dt, float u) {
    static_for<V>([&](auto i) {
        constexpr int m = i;
        f32x4 p;
#pragma unroll
        for (int j = 0; j < 4; ++j) p[j] = __builtin_amdgcn_exp2f(dt * A2[m][j]) * h[m][j];
        h[m] = outer<4 * (m & 3) + ROW>(B[m >> 2], u, p);
    });
}

template <int V, int W> __device__ __forceinline__ float dot(const float (&C)[W], const f32x4 (&h)[V], float y) {
    float y1 = 0.0f;
    if constexpr (V == 1)
        dot_states(y, y1, C[0], h[0]);
    else if constexpr (V == 2)
        dot_states(y, y1, C[0], h[0], h[1]);
    else
        dot_states(y, y1, C[0], h[0], h[1], h[2], h[3]);
    if constexpr (V == 8) dot_states(y, y1, C[1], h[4], h[5], h[6], h[7]);
    return y + y1;
}

// The lane's row of A times log2 e, zeros past the last state.
template <int V> __device__ __forceinline__ void load_decays(const StateSpaceArgs& a, int d, f32x4 (&A2)[V]) {
    const float* A = a.s.A + static_cast<int64_t>(d) * a.s.states;
    if (a.s.states == 4 * V && a.decays_aligned) {
#pragma unroll
        for (int m = 0; m < V; ++m) A2[m] = reinterpret_cast<const f32x4*>(A)[m] * kLog2e;
    } else {
#pragma unroll
        for (int n = 0; n < 4 * V; ++n) A2[n >> 2][n & 3] = n < a.s.states ? A[n] * kLog2e : 0.0f;
    }
}

// The states of the lane's channel (its byte offset), `channels` apart.
template <int V> __device__ __forceinline__ void load_state(const float* from, int states, int channels, uint32_t channel, f32x4 (&h)[V]) {
#pragma unroll
    for (int m = 0; m < V; ++m) h[m] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    if (!from) return;
    const auto row = row_buffer(from);
    const uint32_t step = static_cast<uint32_t>(channels) * 4;
    if (states == 4 * V) {
#pragma unroll
        for (int n = 0; n < 4 * V; ++n) h[n >> 2][n & 3] = lane_load<float>(row, channel, n * step);
    } else {
#pragma unroll
        for (int n = 0; n < 4 * V; ++n)
            if (n < states) h[n >> 2][n & 3] = lane_load<float>(row, channel, n * step);
    }
}
template <int V> __device__ __forceinline__ void store_state(float* to, int states, int channels, uint32_t channel, const f32x4 (&h)[V]) {
    const auto row = row_buffer(to);
    const uint32_t step = static_cast<uint32_t>(channels) * 4;
    if (states == 4 * V) {
#pragma unroll
        for (int n = 0; n < 4 * V; ++n) lane_store<float>(row, channel, n * step, h[n >> 2][n & 3]);
    } else {
#pragma unroll
        for (int n = 0; n < 4 * V; ++n)
            if (n < states) lane_store<float>(row, channel, n * step, h[n >> 2][n & 3]);
    }
}

// Which states a lane holds of the operands of `outer` and `dot` (clamped to the last), and masks that zero what does not exist.
template <typename TB, int W> struct SharedStates {
    uint32_t o[W], c[W], o_mask[W], c_mask[W];   // o, c in bytes
    __device__ __forceinline__ SharedStates(int lane, int states) {
#pragma unroll
        for (int j = 0; j < W; ++j) {
            const int p = 16 * j + 4 * (lane >> 4) + (lane & 3), q = 16 * j + (lane & 15);
            o[j] = (p < states ? p : states - 1) * sizeof(TB), c[j] = (q < states ? q : states - 1) * sizeof(TB);
            o_mask[j] = p < states ? ~0u : 0u, c_mask[j] = q < states ? ~0u : 0u;
        }
    }
};

__device__ __forceinline__ int scan_flags(const ilx_state_space& s) {
    return (s.gate ? kHasGate : 0) | (s.softplus ? kSoftplus : 0) | (s.starts ? kHasStarts : 0);
}

template <typename T, typename TB, int S>
__global__ void __launch_bounds__(64 * kScanWaves) scan_forward_kernel(StateSpaceArgs a) {
    constexpr int V = S / 4, W = (S + 15) / 16;
    const int lane = threadIdx.x & 63, unit = wave_unit();
    if (unit >= a.units) return;
    const ChannelLane c = channel_lane(a, unit % a.blocks, lane);
    const uint32_t channel = c.d * sizeof(T), channel4 = c.d * 4;
    const SharedStates<TB, W> shared(lane, a.s.states);
    const int items = static_cast<int>(a.s.batch * a.parts), slots = static_cast<int>(a.slots);
    f32x4 A2[V], h[V];
    load_decays<V>(a, c.d, A2);
    float bias = a.s.delta_bias ? a.s.delta_bias[c.d] : 0.0f, skip = a.s.D ? a.s.D[c.d] : 0.0f;
    arrive(bias), arrive(skip);
    ScanRows<T, TB, W, true, true> rows;
    ScanStreams<T, TB> k;
    k.flags = scan_flags(a.s);
    k.template open<false>(unit / a.blocks, c.group);
    if (k.begin < k.end) rows.read(k, channel, shared.o, shared.c, lane);
    float* saved = nullptr;
    while (k.item < items) {
        // an item: what enters it, its rows, what leaves it
        const int item = k.item, b = k.b, begin = k.begin, end = k.end;
        Stream<T> out;
        {
            const ArgsPtr p = arguments_again();
            const int64_t state = static_cast<int64_t>(p->s.states) * p->s.channels;
            load_state<V>(p->parts > 1 ? p->part_state + item * state : p->s.state ? p->s.state + b * state : nullptr, p->s.states, p->s.channels, channel4, h);
            out.set(p->s.out, b * p->s.out_batch, begin, p->s.out_time);
            saved = p->s.saved ? p->s.saved + (b * p->saved_blocks + begin / ILX_SCAN_BLOCK) * state : nullptr;
        }
        for (int t0 = begin; t0 < end; t0 += kScanRows) {
            const int count = end - t0 < kScanRows ? end - t0 : kScanRows;
            float x[kScanRows], dt[kScanRows], z[kScanRows], B[W], C[kScanRows][W];
#pragma unroll
            for (int i = 0; i < kScanRows; ++i) {
                x[i] = to_f32(rows.x[i]);
                dt[i] = to_f32(rows.delta[i]) + bias;
                z[i] = to_f32(rows.gate[i]);
#pragma unroll
                for (int j = 0; j < W; ++j) C[i][j] = masked(to_f32(rows.c[i][j]), shared.c_mask[j]);
            }
#pragma unroll
            for (int j = 0; j < W; ++j) B[j] = masked(to_f32(rows.o[j]), shared.o_mask[j]);
            const uint32_t starts = rows.starts();
            if (t0 + kScanRows < end) {
                k.template step<false>();
                rows.read(k, channel, shared.o, shared.c, lane);
            }
            if (saved && t0 % ILX_SCAN_BLOCK == 0) {
                const ArgsPtr p = arguments_again();
                if (c.active) store_state<V>(saved, p->s.states, p->s.channels, channel4, h);
                saved += static_cast<int64_t>(p->s.states) * p->s.channels;
            }
            if (k.flags & kSoftplus) {
#pragma unroll
                for (int i = 0; i < kScanRows; ++i) dt[i] = softplus_f(dt[i]);
            }
            float y[kScanRows];
            static_for<kScanRows>([&](auto r) {
                constexpr int i = r;
                if (i < count) {
                    forget_if(starts >> i & 1, h);
                    advance<i>(h, A2, B, dt[i], dt[i] * x[i]);
                    y[i] = dot<V>(C[i], h, skip * x[i]);
                }
            });
            if (k.flags & kHasGate) {
#pragma unroll
                for (int i = 0; i < kScanRows; ++i) y[i] *= z[i] * sigmoid_fast(z[i]);
            }
            rows.arrived();
            if (c.active) {
#pragma unroll
                for (int i = 0; i < kScanRows; ++i)
                    if (i < count) lane_store<T>(out.buffer(), channel, i * out.time, from_f32<T>(y[i]));
            }
            out.step(kScanRows);
        }
        // the next item's first rows are on their way while this one is finished
        const int next = item + slots;
        k.item = next;
        if (next < items) {
            k.template open<false>(next, c.group);
            if (k.begin < k.end) rows.read(k, channel, shared.o, shared.c, lane);
        }
        {
            const ArgsPtr p = arguments_again();
            const int length = static_cast<int>(p->s.length), part_rows = static_cast<int>(p->part_rows), limit = begin + part_rows < length ? begin + part_rows : length;
            const int first = end > begin ? end : begin;
            if (c.active && (first < limit || p->s.last)) {
                out.set(p->s.out, b * p->s.out_batch, first, p->s.out_time);
                for (int t = first; t < limit; ++t, out.step(1)) lane_store<T>(out.buffer(), channel, 0, from_f32<T>(0.0f));
                if (p->s.last) {   // the part that ends the sequence
                    const int len = p->s.lengths ? static_cast<int>(scan_length(a.s, b)) : length;
                    if ((begin < len && len <= limit) || (len == 0 && begin == 0))
                        store_state<V>(p->s.last + static_cast<int64_t>(b) * p->s.states * p->s.channels, p->s.states, p->s.channels, channel4, h);
                }
            }
        }
    }
}

// What a part of a sequence adds to the state, from zeros: forward the state behind it, backward (REVERSE) the gradient of the
// state ahead of it, r <- a (r + dy C) from its last row to its first.
template <typename T, typename TB, int S, bool REVERSE>
__global__ void __launch_bounds__(64 * kScanWaves) scan_part_kernel(StateSpaceArgs a) {
    constexpr int V = S / 4, W = (S + 15) / 16;
    const int lane = threadIdx.x & 63, unit = wave_unit();
    if (unit >= a.units) return;
    const ChannelLane c = channel_lane(a, unit % a.blocks, lane);
    const uint32_t channel = c.d * sizeof(T), channel4 = c.d * 4;
    const SharedStates<TB, W> shared(lane, a.s.states);
    f32x4 A2[V], h[V];
    load_decays<V>(a, c.d, A2);
#pragma unroll
    for (int m = 0; m < V; ++m) h[m] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    float sum = 0.0f;
    bool any = false;
    const float bias = a.s.delta_bias ? a.s.delta_bias[c.d] : 0.0f;
    ScanRows<T, TB, W, REVERSE, false> rows;
    ScanStreams<T, TB> k;
    k.flags = scan_flags(a.s);
    k.template open<REVERSE>(unit / a.blocks, c.group);
    if (k.begin < k.end) {
        rows.read(k, channel, shared.o, shared.c, lane);
        for (;;) {
            const int count = k.count();
            float x[kScanRows], dt[kScanRows], M[W];
#pragma unroll
            for (int i = 0; i < kScanRows; ++i) {
                x[i] = to_f32(rows.x[i]);
                dt[i] = to_f32(rows.delta[i]) + bias;
            }
            if (REVERSE && (k.flags & kHasGate)) {
#pragma unroll
                for (int i = 0; i < kScanRows; ++i) {
                    const float z = to_f32(rows.gate[i]);
                    x[i] *= z * sigmoid_fast(z);
                }
            }
#pragma unroll
            for (int j = 0; j < W; ++j) M[j] = masked(to_f32(rows.o[j]), shared.o_mask[j]);
            const uint32_t starts = rows.starts();
            any = any || starts != 0;
            const bool more = REVERSE ? k.t0 > k.begin : k.t0 + kScanRows < k.end;
            if (more) {
                k.template step<REVERSE>();
                rows.read(k, channel, shared.o, shared.c, lane);
            }
            if (k.flags & kSoftplus) {
#pragma unroll
                for (int i = 0; i < kScanRows; ++i) dt[i] = softplus_f(dt[i]);
            }
            static_for<kScanRows>([&](auto r) {
                constexpr int i = REVERSE ? kScanRows - 1 - r : r;
                if (i < count) {
                    sum += dt[i];
                    if constexpr (REVERSE) {
                        static_for<V>([&](auto q) {
                            constexpr int m = q;
                            h[m] = outer<4 * (m & 3) + i>(M[m >> 2], x[i], h[m]);
#pragma unroll
                            for (int j = 0; j < 4; ++j) h[m][j] *= __builtin_amdgcn_exp2f(dt[i] * A2[m][j]);
                        });
                    }
                    forget_if(starts >> i & 1, h);
                    if constexpr (!REVERSE) advance<i>(h, A2, M, dt[i], dt[i] * x[i]);
                }
            });
            if (!more) break;
        }
    }
    if (!c.active) return;
    const ArgsPtr p = arguments_again();
    store_state<V>(p->part_state + static_cast<int64_t>(k.item) * p->s.states * p->s.channels, p->s.states, p->s.channels, channel4, h);
    p->part_decay[static_cast<int64_t>(k.item) * p->s.channels + c.d] = any ? __builtin_inff() : sum;
}

// What a part makes of a state: nothing if an episode starts in it, and nothing of a zero state, however far a part of a growing
// recurrence multiplies it.  (A decay of exactly 0 still hands on a NaN, as every row does.)
constexpr float kCut = -1.0f;
__device__ __forceinline__ float pass_on(float decay, float h, float added) {
    return decay == kCut || h == 0.0f ? added : __builtin_fmaf(decay, h, added);
}

// Passes the states through the parts: part_state becomes what enters each part (backward: the gradient that enters it from
// the part behind).  64 states of a sequence to a workgroup, up to 16 parts to each of its waves: a wave joins its own parts, the
// waves' joins meet in LDS, and each wave passes what enters it through its parts again, out of registers.
__global__ void __launch_bounds__(1024) scan_join_kernel(StateSpaceArgs a, int backward, const float* first) {
    __shared__ float s_decay[kMostParts / kJoinParts][64], s_state[kMostParts / kJoinParts][64];
    const ilx_state_space& s = a.s;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int columns = s.states * s.channels, column_blocks = (columns + 63) / 64;
    const int64_t b = blockIdx.x / column_blocks;
    const int column = static_cast<int>(blockIdx.x % column_blocks) * 64 + lane;
    const bool active = column < columns;
    const int at = active ? column : columns - 1, n = at / s.channels, d = at - n * s.channels;
    const int parts = static_cast<int>(a.parts), waves = blockDim.x >> 6, per = (parts + waves - 1) / waves, p0 = w * per;
    const float A2 = s.A[static_cast<int64_t>(d) * s.states + n] * kLog2e;
    float decay[kJoinParts], state[kJoinParts];
#pragma unroll
    for (int j = 0; j < kJoinParts; ++j) {
        const bool in = j < per && p0 + j < parts;
        const int64_t p = b * parts + (backward ? parts - 1 - (p0 + j) : p0 + j);
        decay[j] = in ? a.part_decay[p * s.channels + d] : 0.0f;
        state[j] = in ? a.part_state[p * columns + at] : 0.0f;
    }
    float total = 0.0f, H = 0.0f;
    bool cut = false;
#pragma unroll
    for (int j = 0; j < kJoinParts; ++j) {
        const bool start = decay[j] == __builtin_inff();
        cut = cut || start;
        total += start ? 0.0f : decay[j];
        decay[j] = start ? kCut : __builtin_amdgcn_exp2f(decay[j] * A2);
        H = pass_on(decay[j], H, state[j]);
    }
    s_decay[w][lane] = cut ? kCut : __builtin_amdgcn_exp2f(total * A2);   // (not the product: factors of it may leave the range)
    s_state[w][lane] = H;
    __syncthreads();
    float h = first ? first[b * columns + at] : 0.0f;
    for (int k = 0; k < w; ++k) h = pass_on(s_decay[k][lane], h, s_state[k][lane]);
    if (!active) return;
#pragma unroll
    for (int j = 0; j < kJoinParts; ++j) {
        if (j < per && p0 + j < parts) {
            const int64_t p = b * parts + (backward ? parts - 1 - (p0 + j) : p0 + j);
            a.part_state[p * columns + at] = h;
            h = pass_on(decay[j], h, state[j]);
        }
    }
}

// One row per sequence: the recurrence above with sequences in the place of rows, so that A stays in registers.  Bound by
// the state, read and written once.
template <typename T, typename TB, int S>
__global__ void __launch_bounds__(64 * kScanWaves) scan_step_kernel(StateSpaceArgs a) {
    constexpr int V = S / 4, W = (S + 15) / 16;
    const int lane = threadIdx.x & 63, unit = wave_unit();
    if (unit >= a.units) return;
    const ChannelLane c = channel_lane(a, unit % a.blocks, lane);
    const uint32_t channel = c.d * sizeof(T), channel4 = c.d * 4;
    const SharedStates<TB, W> shared(lane, a.s.states);
    const ilx_state_space& s = a.s;
    f32x4 A2[V], h[V];
    load_decays<V>(a, c.d, A2);
    const float bias = s.delta_bias ? s.delta_bias[c.d] : 0.0f, skip = s.D ? s.D[c.d] : 0.0f;
    const int64_t state_size = static_cast<int64_t>(s.states) * s.channels;
    for (int64_t b = unit / a.blocks; b < s.batch; b += a.slots) {
        float* state = s.last + b * state_size;
        load_state<V>(state, s.states, s.channels, channel4, h);
        float x = to_f32(lane_load<T>(row_buffer(static_cast<const T*>(s.x) + b * s.x_batch), channel, 0));
        float dt = to_f32(lane_load<T>(row_buffer(static_cast<const T*>(s.delta) + b * s.delta_batch), channel, 0)) + bias, z = 0.0f;
        if (s.gate) z = to_f32(lane_load<T>(row_buffer(static_cast<const T*>(s.gate) + b * s.gate_batch), channel, 0));
        const TB* pB = static_cast<const TB*>(s.B) + b * s.B_batch + c.group * s.states;
        const TB* pC = static_cast<const TB*>(s.C) + b * s.C_batch + c.group * s.states;
        float B[W], C[W];
#pragma unroll
        for (int j = 0; j < W; ++j) {
            B[j] = masked(to_f32(lane_load<TB>(row_buffer(pB), shared.o[j], 0)), shared.o_mask[j]);
            C[j] = masked(to_f32(lane_load<TB>(row_buffer(pC), shared.c[j], 0)), shared.c_mask[j]);
        }
        const bool start = s.starts && uni(static_cast<int>(s.starts[b * s.starts_batch]));
        if (s.softplus) dt = softplus_f(dt);
        forget_if(start, h);
        advance<0>(h, A2, B, dt, dt * x);
        float y = dot<V>(C, h, skip * x);
        if (s.gate) y *= z * sigmoid_fast(z);
        if (!c.active) continue;
        store_state<V>(state, s.states, s.channels, channel4, h);
        lane_store<T>(row_buffer(static_cast<T*>(s.out) + b * s.out_batch), channel, 0, from_f32<T>(y));
    }
}

// The kernels count rows in 32 bits, up to the end of the last part, which may lie behind the sequence's: parts are rounded up to
// ILX_SCAN_BLOCK rows and there are at most kMostParts.
constexpr int64_t kMostRows = INT32_MAX - 4096;
static_assert(kMostParts * ILX_SCAN_BLOCK + 64 <= 4096, "rows behind a sequence's end");

int scan_check(const ilx_state_space& s, const char* name) {
    ILX_REQUIRE(s.batch >= 0 && s.length >= 0 && s.channels > 0 && s.groups > 0, ILX_EINVAL, "%s: bad shape (%lld, %lld, %d), %d groups", name,
                (long long)s.batch, (long long)s.length, s.channels, s.groups);
    ILX_REQUIRE(s.channels % s.groups == 0, ILX_ESHAPE, "%s: %d channels do not split into %d groups", name, s.channels, s.groups);
    ILX_REQUIRE(s.states >= 1 && s.states <= ILX_SCAN_MAX_STATES, ILX_ESHAPE, "%s: %d states (1..%d supported)", name, s.states,
                ILX_SCAN_MAX_STATES);
    ILX_REQUIRE(s.channels <= kMostChannels, ILX_ESHAPE, "%s: %d channels", name, s.channels);
    ILX_REQUIRE(s.dtype >= ILX_F32 && s.dtype <= ILX_F16, ILX_EINVAL, "%s: unknown type %d", name, s.dtype);
    ILX_REQUIRE(s.bc_dtype == ILX_F32 || s.bc_dtype == s.dtype, ILX_EINVAL, "%s: B and C of type %d beside activations of type %d", name,
                s.bc_dtype, s.dtype);
    ILX_REQUIRE(s.batch <= INT32_MAX && s.length <= kMostRows && s.batch * (s.length + 1) < (int64_t{1} << 40), ILX_ESHAPE,
                "%s: shape (%lld, %lld) too large", name, (long long)s.batch, (long long)s.length);
    if (s.length > 1)
        for (const int64_t stride : {s.x_time, s.delta_time, s.gate_time, s.B_time, s.C_time, s.out_time, s.grad_out_time, s.grad_time, s.starts_time})
            ILX_REQUIRE(stride >= 0 && stride < (int64_t{1} << 27), ILX_ESHAPE, "%s: a time stride of %lld elements", name, (long long)stride);
    return ILX_OK;
}

// Workgroups per block of channels: enough for four waves a SIMD, each with as many items as the next.
void share_items(StateSpaceArgs& a, int64_t items) {
    const int64_t waves = 16 * device_cu_count(), most = waves / a.blocks > 0 ? waves / a.blocks : 1, each = (items + most - 1) / most;
    a.slots = each > 0 ? (items + each - 1) / each : 0;
}

StateSpaceArgs scan_args(const ilx_state_space& s) {
    StateSpaceArgs a{};
    a.s = s;
    a.group_channels = s.channels / s.groups;
    a.group_blocks = (a.group_channels + 63) / 64;
    a.blocks = s.groups * a.group_blocks;
    a.saved_blocks = (s.length + ILX_SCAN_BLOCK - 1) / ILX_SCAN_BLOCK;
    a.parts = 1, a.part_rows = s.length;
    a.decays_aligned = aligned_to(s.A, 16);
    share_items(a, s.batch);
    return a;
}

// With a wave on every SIMD a sequence is not divided: a wave alone on a SIMD takes 420 ns for a row of 16 states, two together 650 for
// two, four 1190 for four, and the second pass costs as much again (400 x 100 rows x 256 channels: 65 us, in two parts 128; 256 x 500 x
// 256: 211 against 258).  Below that it is divided towards four waves a SIMD (128 x 500 x 256: 136 us, undivided 260), short ones only
// where the chip would be three quarters empty (128 x 64 x 256 with gradients: 78 us, divided 105; 1 x 64 x 256: 27 us, divided 15).  A
// part has at least 16 rows, or 8 while parts of 16 leave half of the SIMDs without a wave (1 x 512 x 512: 18 us with 8, 23 with 16, 33
// with 32; 4 x 215 x 1150: 30, 27 and 35).  More than 256 parts gain nothing and take 31 us for the join in the place of 11.
int64_t divide_scan(StateSpaceArgs& a, float* workspace) {
    const ilx_state_space& s = a.s;
    const int64_t waves = s.batch * a.blocks, full = 4 * device_cu_count();   // one per SIMD
    if (waves == 0 || waves >= full || s.length < (waves > full / 4 ? 128 : 64)) return 0;
    int64_t parts = 4 * full / waves;
    if (parts > kMostParts) parts = kMostParts;
    const int64_t least = waves * ((s.length + 15) / 16) > full / 2 ? 16 : ILX_SCAN_BLOCK;
    int64_t rows = (s.length + parts - 1) / parts;
    if (rows < least) rows = least;
    rows = (rows + ILX_SCAN_BLOCK - 1) / ILX_SCAN_BLOCK * ILX_SCAN_BLOCK;
    a.part_rows = rows, a.parts = (s.length + rows - 1) / rows;
    if (a.parts == 1) return 0;
    const int64_t states = s.batch * a.parts * s.states * s.channels, decays = s.batch * a.parts * s.channels;
    a.part_state = workspace, a.part_decay = workspace + states;
    share_items(a, s.batch * a.parts);
    return states + decays;
}

}  // namespace ilx

using namespace ilx;

namespace {

enum ScanKind { kForward, kStep, kParts, kPartsBackward };

template <typename T, typename TB, int S> void scan_launch(ScanKind kind, StateSpaceArgs a, hipStream_t s) {
    a.units = static_cast<int>((kind == kStep || kind == kForward ? a.slots : a.s.batch * a.parts) * a.blocks);
    const dim3 grid(blocks_for(a.units, kScanWaves)), threads(64 * kScanWaves);
    switch (kind) {
        case kStep: ILX_LAUNCH((scan_step_kernel<T, TB, S>), grid, threads, 0, s, a); break;
        case kParts: ILX_LAUNCH((scan_part_kernel<T, TB, S, false>), grid, threads, 0, s, a); break;
        case kPartsBackward: ILX_LAUNCH((scan_part_kernel<T, TB, S, true>), grid, threads, 0, s, a); break;
        default: ILX_LAUNCH((scan_forward_kernel<T, TB, S>), grid, threads, 0, s, a); break;
    }
}

template <typename T, typename TB> void scan_states(ScanKind kind, const StateSpaceArgs& a, hipStream_t s) {
    const int n = a.s.states;
    if (n <= 4) return scan_launch<T, TB, 4>(kind, a, s);
    if (n <= 8) return scan_launch<T, TB, 8>(kind, a, s);
    if (n <= 16) return scan_launch<T, TB, 16>(kind, a, s);
    scan_launch<T, TB, 32>(kind, a, s);
}

void scan_dispatch(ScanKind kind, const StateSpaceArgs& a, hipStream_t s) {
    const bool wide = a.s.bc_dtype == ILX_F32;
    switch (a.s.dtype) {
        case ILX_F32: return scan_states<float, float>(kind, a, s);
        case ILX_BF16: return wide ? scan_states<bf16_t, float>(kind, a, s) : scan_states<bf16_t, bf16_t>(kind, a, s);
        default: return wide ? scan_states<f16_t, float>(kind, a, s) : scan_states<f16_t, f16_t>(kind, a, s);
    }
}

}  // namespace

void ilx::launch_part_states(const StateSpaceArgs& a, bool backward, hipStream_t s) {
    scan_dispatch(backward ? kPartsBackward : kParts, a, s);
    const int64_t column_blocks = (static_cast<int64_t>(a.s.states) * a.s.channels + 63) / 64;
    ILX_LAUNCH(scan_join_kernel, dim3(static_cast<unsigned>(a.s.batch * column_blocks)), dim3(blocks_for(a.parts, kJoinParts) * 64), 0, s, a, backward ? 1 : 0,
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
    StateSpaceArgs a = scan_args(s);
    const int64_t needed = divide_scan(a, s.workspace);
    ILX_REQUIRE(needed == 0 || (s.workspace && s.workspace_floats >= needed), ILX_EINVAL,
                "ilx_state_space_forward: workspace of %lld floats, %lld needed", (long long)s.workspace_floats, (long long)needed);
    ILX_REQUIRE(s.batch * a.parts * a.blocks <= INT32_MAX - 65536, ILX_ESHAPE, "ilx_state_space_forward: shape too large for one launch");
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
    const StateSpaceArgs a = scan_args(s);
    ILX_REQUIRE(s.batch * a.blocks <= INT32_MAX - 65536, ILX_ESHAPE, "ilx_state_space_step: shape too large for one launch");
    scan_dispatch(kStep, a, as_stream(stream));
    ILX_LAUNCH_CHECK("ilx_state_space_step");
    return ILX_OK;
}
