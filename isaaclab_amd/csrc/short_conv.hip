// Short causal convolution over time, depthwise (one filter per channel), with a carried state and episode starts:
//   p_t = bias + sum_j w[W-1-j] x_{t-j},  out = p or p sigmoid(p);   rows t < 0 are the carried state.
// All three kernels move each input once and have 2 W + 6 flops per element, so they are bound by memory.  A thread owns V
// neighbouring channels (one access of 16 bytes per row, or 8 where the backward pass has 16-bit elements) of a segment of rows
// and keeps the last W - 1 rows in registers; a segment re-reads the W - 1 rows ahead of it, which the thread beside it has just
// brought into the cache.  An episode start clears the registers, so no row looks past it.  Where V does not divide the
// channels, the last thread's V channels end with the row's and overlap its neighbour's: both come to the same values and store
// them, but for the step, which writes what its neighbour reads and stores its own only.
// Measured, W = 4, against a large copy's 4.97 TB/s on the same card:
//   forward, 24 x 4096 x 256 f32: 41 us, 201 MB, 4.9 TB/s
//   forward, 3 x 8190 x 1536 bf16: 37 us (32 to 40), 151 MB, 4.1 TB/s
//   backward, 24 x 4096 x 256 f32: 70 us, 302 MB, 4.3 TB/s, and 7 us for the sums of 1024 workgroups' parts of dw and dbias
//   step, 16384 x 512 f32: 41 us in a loop on one state, 52 on states that are not cached (268 MB, 5.1 TB/s)
#include "sequence_dev.h"

namespace ilx {

constexpr int kConvThreads = 256;
constexpr int kConvRows = 2;   // read ahead; 4: a recording of 16384 x 1024 in bfloat16 takes 42 us for 36, 8 (V = 4): 38, and spills in the backward pass (89 us for 66)

struct ConvArgs {
    ilx_short_conv c;
    int groups;        // of V channels, the last one's shifted to end with the row
    int cx_log2;       // lanes side by side over channel groups; 256 >> cx_log2 rows of threads over segments
    int channel_blocks;
    int segment;       // rows per segment
    int64_t segments;  // per sequence
    int64_t items;     // batch * segments
    int64_t slots;     // rows of threads in the grid / rows per block (backward: partial sums)
};

template <int V> __device__ __forceinline__ int first_channel(const ConvArgs& a, int group) {
    return group * V + V <= a.c.channels ? group * V : a.c.channels - V;
}

__device__ __forceinline__ int64_t sequence_length(const int32_t* lengths, int64_t b, int64_t length) {
    if (!lengths) return length;
    const int64_t n = lengths[b];
    return n < 0 ? 0 : (n > length ? length : n);
}

template <int W, int V>
__device__ __forceinline__ void load_weights(const ConvArgs& a, int d0, float (&w)[W][V], float (&bias)[V]) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
        bias[v] = a.c.bias ? a.c.bias[d0 + v] : 0.0f;
#pragma unroll
        for (int k = 0; k < W; ++k) w[k][v] = a.c.weight[static_cast<int64_t>(d0 + v) * W + k];
    }
}

// The W - 1 rows ahead of row t0, oldest first, those from before an episode start as zeros.
template <typename T, int W, int V>
__device__ __forceinline__ void load_window(const ConvArgs& a, int d0, int64_t b, int64_t t0, float (&win)[W][V]) {
    const T* x = static_cast<const T*>(a.c.x) + b * a.c.x_batch;
#pragma unroll
    for (int i = 0; i < W - 1; ++i) {
        const int64_t t = t0 - (W - 1) + i;
#pragma unroll
        for (int v = 0; v < V; ++v) win[i][v] = 0.0f;
        if (t >= 0) {
            if (a.c.starts && a.c.starts[b * a.c.starts_batch + t * a.c.starts_time]) {
#pragma unroll
                for (int k = 0; k < i; ++k)
#pragma unroll
                    for (int v = 0; v < V; ++v) win[k][v] = 0.0f;
            }
            load_channels<V>(x + t * a.c.x_time + d0, win[i]);
        } else if (a.c.state) {
            load_channels<V>(a.c.state + (b * (W - 1) + (W - 1 + t)) * a.c.channels + d0, win[i]);
        }
    }
}

template <int W, int V>
__device__ __forceinline__ void filter(const float (&w)[W][V], const float (&bias)[V], const float (&win)[W][V], float (&p)[V]) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
        p[v] = bias[v];
#pragma unroll
        for (int k = 0; k < W; ++k) p[v] = __builtin_fmaf(w[k][v], win[k][v], p[v]);
    }
}

template <int W, int V> __device__ __forceinline__ void shift(float (&win)[W][V]) {
#pragma unroll
    for (int k = 0; k + 1 < W; ++k)
#pragma unroll
        for (int v = 0; v < V; ++v) win[k][v] = win[k + 1][v];
}
template <int W, int V> __device__ __forceinline__ void forget(float (&win)[W][V]) {
#pragma unroll
    for (int k = 0; k + 1 < W; ++k)
#pragma unroll
        for (int v = 0; v < V; ++v) win[k][v] = 0.0f;
}

// The next kConvRows rows of x (and of the output's gradient) and their start flags, read while the rows ahead are worked on.
template <typename T, int V, bool GRAD> struct ConvRows {
    Channels<T, V> x[kConvRows], g[kConvRows];
    uint8_t start[kConvRows];

    __device__ __forceinline__ void read(const ConvArgs& a, int d0, int64_t b, int64_t t, int64_t end) {
        const T* px = static_cast<const T*>(a.c.x) + b * a.c.x_batch + d0;
        const T* pg = static_cast<const T*>(a.c.grad_out) + b * a.c.grad_out_batch + d0;
        const uint8_t* ps = a.c.starts + b * a.c.starts_batch;
#pragma unroll
        for (int i = 0; i < kConvRows; ++i) {
            const int64_t r = t + i < end ? t + i : end - 1;
            x[i] = *reinterpret_cast<const Channels<T, V>*>(px + r * a.c.x_time);
            if (GRAD) g[i] = *reinterpret_cast<const Channels<T, V>*>(pg + r * a.c.grad_out_time);
            start[i] = 0;
            if (a.c.starts) start[i] = ps[r * a.c.starts_time];
        }
    }
};
template <int V, typename T> __device__ __forceinline__ void unpack(const Channels<T, V>& p, float (&v)[V]) {
#pragma unroll
    for (int k = 0; k < V; ++k) v[k] = to_f32(p.v[k]);
}

template <typename T, int W, int V>
__global__ void __launch_bounds__(kConvThreads) short_conv_forward_kernel(ConvArgs a) {
    const int cx = threadIdx.x & ((1 << a.cx_log2) - 1), row = threadIdx.x >> a.cx_log2;
    const int group = static_cast<int>(blockIdx.x % a.channel_blocks) * (1 << a.cx_log2) + cx;
    const int64_t item = static_cast<int64_t>(blockIdx.x / a.channel_blocks) * (kConvThreads >> a.cx_log2) + row;
    if (group >= a.groups || item >= a.items) return;
    const int d0 = first_channel<V>(a, group);
    const int64_t b = item / a.segments, t0 = (item - b * a.segments) * a.segment;
    const int64_t t1 = t0 + a.segment < a.c.length ? t0 + a.segment : a.c.length;
    const int64_t len = sequence_length(a.c.lengths, b, a.c.length), te = t1 < len ? t1 : len;
    T* out = static_cast<T*>(a.c.out) + b * a.c.out_batch + d0;
    if (t0 < len || t0 == 0) {
        float w[W][V], bias[V], win[W][V];
        ConvRows<T, V, false> rows;
        if (t0 < te) rows.read(a, d0, b, t0, te);
        load_weights<W, V>(a, d0, w, bias);
        load_window<T, W, V>(a, d0, b, t0, win);
        for (int64_t t = t0; t < te; t += kConvRows) {
            const ConvRows<T, V, false> now = rows;
            if (t + kConvRows < te) rows.read(a, d0, b, t + kConvRows, te);
#pragma unroll
            for (int i = 0; i < kConvRows; ++i) {
                if (t + i < te) {
                    if (now.start[i]) forget<W, V>(win);
                    unpack<V>(now.x[i], win[W - 1]);
                    float p[V];
                    filter<W, V>(w, bias, win, p);
                    if (a.c.silu) {
#pragma unroll
                        for (int v = 0; v < V; ++v) p[v] *= sigmoid_fast(p[v]);
                    }
                    store_channels<V>(out + (t + i) * a.c.out_time, p);
                    shift<W, V>(win);
                }
            }
        }
        if (a.c.last && (len == 0 || (te == len && t0 < len))) {   // the segment that ends the sequence
#pragma unroll
            for (int k = 0; k < W - 1; ++k) store_channels<V>(a.c.last + (b * (W - 1) + k) * a.c.channels + d0, win[k]);
        }
    }
    float zero[V];
#pragma unroll
    for (int v = 0; v < V; ++v) zero[v] = 0.0f;
    for (int64_t t = te > t0 ? te : t0; t < t1; ++t) store_channels<V>(out + t * a.c.out_time, zero);
}

// Backward.  With dp_t = dout_t act'(p_t):  dx_t = sum_j w[W-1-j] dp_{t+j} over the rows t + j that no start parts from t.
// A thread walks its segment and the W - 1 rows behind it, recomputing p; acc[j] gathers dx of row t - j and is stored
// when the walk has passed its last reader.  open[j] says whether row t still reaches row t - j.
template <typename T, int W, int V>
__global__ void __launch_bounds__(kConvThreads) short_conv_backward_kernel(ConvArgs a) {
    extern __shared__ float sums[];   // [rows of threads][lanes][(W + 1) * V]
    const int cx = threadIdx.x & ((1 << a.cx_log2) - 1), row = threadIdx.x >> a.cx_log2, rows = kConvThreads >> a.cx_log2;
    const int group = static_cast<int>(blockIdx.x % a.channel_blocks) * (1 << a.cx_log2) + cx;
    const int64_t slot = blockIdx.x / a.channel_blocks;
    const bool active = group < a.groups;
    const int d0 = first_channel<V>(a, active ? group : a.groups - 1);
    float w[W][V], bias[V], dw[W][V], db[V];
    load_weights<W, V>(a, d0, w, bias);
#pragma unroll
    for (int v = 0; v < V; ++v) {
        db[v] = 0.0f;
#pragma unroll
        for (int k = 0; k < W; ++k) dw[k][v] = 0.0f;
    }
    for (int64_t item = active ? slot * rows + row : a.items; item < a.items; item += a.slots * rows) {
        const int64_t b = item / a.segments, t0 = (item - b * a.segments) * a.segment;
        const int64_t t1 = t0 + a.segment < a.c.length ? t0 + a.segment : a.c.length;
        const int64_t len = sequence_length(a.c.lengths, b, a.c.length);
        T* dx = static_cast<T*>(a.c.grad_x) + b * a.c.grad_x_batch + d0;
        auto emit = [&](int64_t t, const float (&g)[V]) {
            if (t >= t0) {
                if (t < t1) store_channels<V>(dx + t * a.c.grad_x_time, g);
            } else if (t < 0 && t0 == 0 && a.c.grad_state) {
                store_channels<V>(a.c.grad_state + (b * (W - 1) + (W - 1 + t)) * a.c.channels + d0, g);
            }
        };
        if (t0 < len || t0 == 0) {
            float win[W][V], acc[W][V];
            bool open[W];
            load_window<T, W, V>(a, d0, b, t0, win);
#pragma unroll
            for (int j = 0; j < W; ++j) {
                open[j] = true;
#pragma unroll
                for (int v = 0; v < V; ++v) acc[j][v] = 0.0f;
            }
            const int64_t te = t1 + W - 1 < len ? t1 + W - 1 : len;
            ConvRows<T, V, true> rows;
            if (t0 < te) rows.read(a, d0, b, t0, te);
            for (int64_t first = t0; first < te; first += kConvRows) {
                const ConvRows<T, V, true> now = rows;
                if (first + kConvRows < te) rows.read(a, d0, b, first + kConvRows, te);
#pragma unroll
                for (int r = 0; r < kConvRows; ++r) {
                    const int64_t t = first + r;
                    if (t >= te) break;
                    if (now.start[r]) {
                        forget<W, V>(win);
#pragma unroll
                        for (int j = 1; j < W; ++j) open[j] = false;
                    }
                    unpack<V>(now.x[r], win[W - 1]);
                    float g[V], p[V];
                    unpack<V>(now.g[r], g);
                    filter<W, V>(w, bias, win, p);
                    if (a.c.silu) {
#pragma unroll
                        for (int v = 0; v < V; ++v) {
                            const float s = sigmoid_fast(p[v]);
                            g[v] *= s * __builtin_fmaf(p[v], 1.0f - s, 1.0f);
                        }
                    }
#pragma unroll
                    for (int j = 0; j < W; ++j)
                        if (open[j]) {
#pragma unroll
                            for (int v = 0; v < V; ++v) acc[j][v] = __builtin_fmaf(w[W - 1 - j][v], g[v], acc[j][v]);
                        }
                    if (t < t1) {
#pragma unroll
                        for (int v = 0; v < V; ++v) {
                            db[v] += g[v];
#pragma unroll
                            for (int k = 0; k < W; ++k) dw[k][v] = __builtin_fmaf(g[v], win[k][v], dw[k][v]);
                        }
                    }
                    emit(t - (W - 1), acc[W - 1]);
                    shift<W, V>(win);
#pragma unroll
                    for (int j = W - 1; j > 0; --j) {
                        open[j] = open[j - 1];
#pragma unroll
                        for (int v = 0; v < V; ++v) acc[j][v] = acc[j - 1][v];
                    }
                    open[0] = true;
#pragma unroll
                    for (int v = 0; v < V; ++v) acc[0][v] = 0.0f;
                }
            }
            if (te == len) {   // rows whose last readers are the carried-out state
#pragma unroll
                for (int j = W - 1; j > 0; --j) {
                    if (a.c.grad_last && open[j]) {
                        float g[V];
                        load_channels<V>(a.c.grad_last + (b * (W - 1) + (W - 1 - j)) * a.c.channels + d0, g);
#pragma unroll
                        for (int v = 0; v < V; ++v) acc[j][v] += g[v];
                    }
                    emit(len - j, acc[j]);
                }
            }
        }
        float zero[V];
#pragma unroll
        for (int v = 0; v < V; ++v) zero[v] = 0.0f;
        for (int64_t t = len > t0 ? len : t0; t < t1; ++t) store_channels<V>(dx + t * a.c.grad_x_time, zero);
    }
    // the workgroup's part of dw and db: one row of partial sums, added over the rows of threads in order and in 64 bits
    constexpr int P = (W + 1) * V;
    float* mine = sums + threadIdx.x * P;
#pragma unroll
    for (int v = 0; v < V; ++v) {
#pragma unroll
        for (int k = 0; k < W; ++k) mine[k * V + v] = dw[k][v];
        mine[W * V + v] = db[v];
    }
    __syncthreads();
    const int lanes = 1 << a.cx_log2;
    for (int i = threadIdx.x; i < lanes * P; i += kConvThreads) {
        const int lane = i / P, kv = i - lane * P, k = kv / V, v = kv - k * V;
        const int g = static_cast<int>(blockIdx.x % a.channel_blocks) * lanes + lane;
        if (g >= a.groups) continue;
        double s = 0.0;
        for (int r = 0; r < rows; ++r) s += static_cast<double>(sums[(r * lanes + lane) * P + kv]);
        a.c.workspace[(slot * (W + 1) + k) * a.c.channels + first_channel<V>(a, g) + v] = static_cast<float>(s);
    }
}

// One row per sequence; the state moves up by one row in place.
template <typename T, int W, int V>
__global__ void __launch_bounds__(kConvThreads) short_conv_step_kernel(ConvArgs a) {
    const int64_t i = static_cast<int64_t>(blockIdx.x) * kConvThreads + threadIdx.x;
    if (i >= a.items) return;
    const int64_t b = i / a.groups;
    const int group = static_cast<int>(i - b * a.groups), d0 = first_channel<V>(a, group), shared = group * V - d0;   // the neighbour's channels
    float w[W][V], bias[V], win[W][V], p[V];
    const bool start = a.c.starts && a.c.starts[b * a.c.starts_batch];
    float* last = a.c.last + b * (W - 1) * a.c.channels + d0;
#pragma unroll
    for (int k = 0; k < W - 1; ++k) load_channels<V>(last + k * static_cast<int64_t>(a.c.channels), win[k]);
    load_channels<V>(static_cast<const T*>(a.c.x) + b * a.c.x_batch + d0, win[W - 1]);
    load_weights<W, V>(a, d0, w, bias);
    if (start) forget<W, V>(win);
    filter<W, V>(w, bias, win, p);
    if (a.c.silu) {
#pragma unroll
        for (int v = 0; v < V; ++v) p[v] *= sigmoid_fast(p[v]);
    }
    T* out = static_cast<T*>(a.c.out) + b * a.c.out_batch + d0;
    if (shared == 0) {
        store_channels<V>(out, p);
#pragma unroll
        for (int k = 0; k < W - 1; ++k) store_channels<V>(last + k * static_cast<int64_t>(a.c.channels), win[k + 1]);
    } else {
#pragma unroll
        for (int v = 0; v < V; ++v) {
            if (v < shared) continue;
            out[v] = from_f32<T>(p[v]);
#pragma unroll
            for (int k = 0; k < W - 1; ++k) last[k * static_cast<int64_t>(a.c.channels) + v] = win[k + 1][v];
        }
    }
}

// out0[d, k] = sum over the partial rows of value (k, d): kSumColumns columns to a workgroup, kSumParts threads to a column, eight rows of
// a thread in flight.  1024 rows of 1280 columns take 8 us with 16 columns, 11 with 32 (40 workgroups), 10 with 8 (reads of 32 bytes).
constexpr int kSumColumns = 16, kSumParts = 1024 / kSumColumns;

__global__ void __launch_bounds__(1024) parameter_sums_kernel(const float* partial, int64_t count, int channels, int n0, int columns,
                                                              float* out0, float* out1, float* out2) {
    __shared__ double sums[kSumParts][kSumColumns + 1];
    const int lane = threadIdx.x % kSumColumns, part = threadIdx.x / kSumColumns;
    const int col = static_cast<int>(blockIdx.x) * kSumColumns + lane;
    double s = 0.0;
    if (col < columns)
        for (int64_t r = part; r < count; r += 8 * kSumParts) {
            float v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = r + kSumParts * k < count ? partial[(r + kSumParts * k) * columns + col] : 0.0f;
#pragma unroll
            for (int k = 0; k < 8; ++k) s += static_cast<double>(v[k]);
        }
    sums[part][lane] = s;
    __syncthreads();
    if (part != 0 || col >= columns) return;
    s = 0.0;
#pragma unroll
    for (int k = 0; k < kSumParts; ++k) s += sums[k][lane];
    const int k = col / channels, d = col - k * channels;
    if (k < n0)
        out0[static_cast<int64_t>(d) * n0 + k] = static_cast<float>(s);
    else if (k == n0) {
        if (out1) out1[d] = static_cast<float>(s);
    } else if (out2)
        out2[d] = static_cast<float>(s);
}

void launch_parameter_sums(const float* partial, int64_t count, int32_t channels, int32_t n0, int32_t extra, float* out0, float* out1, float* out2,
                           hipStream_t stream) {
    const int columns = channels * (n0 + extra);
    ILX_LAUNCH(parameter_sums_kernel, dim3(blocks_for(columns, kSumColumns)), dim3(1024), 0, stream, partial, count, static_cast<int>(channels),
               static_cast<int>(n0), columns, out0, out1, out2);
}

}  // namespace ilx

using namespace ilx;

namespace {

constexpr int kMostSegment = 64, kLeastSegment = 8;   // rows

size_t conv_item_bytes(int dtype) { return dtype == ILX_F32 ? 4 : 2; }

// Channels of a thread: 16 bytes of them (four in the backward pass, which keeps five rows of values a channel), fewer where that
// would leave less than two waves a SIMD with the shortest segments.  Measured in bf16, forward: 3 x 8190 x 1535 channels 38 us with 8,
// 55 with one; 1000 x 24 x 256 9 us with 4, 13 with 8; 1 x 2048 x 256 4 us with one, 8 with 8.
int conv_vector(const ilx_short_conv& c, bool backward) {
    for (const int v : {8, 4}) {
        if (c.channels < v || (v == 8 && (backward || conv_item_bytes(c.dtype) == 4))) continue;
        if (c.batch * ((c.length + kLeastSegment - 1) / kLeastSegment) * ((c.channels + v - 1) / v) >= 512 * device_cu_count()) return v;
    }
    return 1;
}

ConvArgs conv_args(const ilx_short_conv& c, int v, bool backward) {
    ConvArgs a{};
    a.c = c;
    a.groups = (c.channels + v - 1) / v;
    a.cx_log2 = 0;
    while (a.cx_log2 < 6 && (1 << a.cx_log2) < a.groups) ++a.cx_log2;
    a.channel_blocks = (a.groups + (1 << a.cx_log2) - 1) >> a.cx_log2;
    // A long segment reads few rows twice; it is halved while there are too few threads for two waves a SIMD.
    a.segment = kMostSegment;
    while (a.segment > kLeastSegment && c.batch * ((c.length + a.segment - 1) / a.segment) * a.groups < 512 * device_cu_count()) a.segment /= 2;
    a.segments = c.length > 0 ? (c.length + a.segment - 1) / a.segment : 1;
    a.items = c.batch * a.segments;
    const int rows = kConvThreads >> a.cx_log2;
    a.slots = (a.items + rows - 1) / rows;
    if (backward) {
        // a thousand workgroups, and more where a thread's segments would hold more than kChainRows rows
        const int64_t most = 1024 / a.channel_blocks > 0 ? 1024 / a.channel_blocks : 1;
        const int64_t chain = kChainRows / (c.length < 1 ? 1 : c.length < a.segment ? c.length : a.segment) * rows, least = (a.items + chain - 1) / chain;
        const int64_t wanted = most > least ? most : least;
        if (a.slots > wanted) a.slots = wanted;
    }
    return a;
}

int conv_check(const ilx_short_conv& c, const char* name) {
    ILX_REQUIRE(c.batch >= 0 && c.length >= 0 && c.channels > 0, ILX_EINVAL, "%s: bad shape (%lld, %lld, %d)", name, (long long)c.batch,
                (long long)c.length, c.channels);
    ILX_REQUIRE(c.width >= 1 && c.width <= ILX_CONV_MAX_WIDTH, ILX_ESHAPE, "%s: width %d (1..%d supported)", name, c.width,
                ILX_CONV_MAX_WIDTH);
    ILX_REQUIRE(c.channels <= kMostChannels, ILX_ESHAPE, "%s: %d channels", name, c.channels);
    ILX_REQUIRE(c.dtype >= ILX_F32 && c.dtype <= ILX_F16, ILX_EINVAL, "%s: unknown type %d", name, c.dtype);
    ILX_REQUIRE(c.batch <= INT32_MAX && c.length <= INT32_MAX && c.batch * (c.length + 1) < (int64_t{1} << 40), ILX_ESHAPE,
                "%s: shape (%lld, %lld) too large", name, (long long)c.batch, (long long)c.length);
    return ILX_OK;
}

enum ConvKind { kForward, kBackward, kStep };

template <typename T, int W, int V> void conv_launch(ConvKind kind, const ConvArgs& a, hipStream_t s) {
    const unsigned threads = kConvThreads;
    if (kind == kStep) {
        ILX_LAUNCH((short_conv_step_kernel<T, W, V>), dim3(blocks_for(a.items, kConvThreads)), dim3(threads), 0, s, a);
    } else if (kind == kForward) {
        ILX_LAUNCH((short_conv_forward_kernel<T, W, V>), dim3(static_cast<unsigned>(a.slots * a.channel_blocks)), dim3(threads), 0, s, a);
    } else if constexpr (V <= 4) {
        ILX_LAUNCH((short_conv_backward_kernel<T, W, V>), dim3(static_cast<unsigned>(a.slots * a.channel_blocks)), dim3(threads),
                   static_cast<unsigned>(kConvThreads * (W + 1) * V * sizeof(float)), s, a);
    }
}

template <typename T, int V> void conv_width(ConvKind kind, const ConvArgs& a, hipStream_t s) {
    switch (a.c.width) {
        case 1: return conv_launch<T, 1, V>(kind, a, s);
        case 2: return conv_launch<T, 2, V>(kind, a, s);
        case 3: return conv_launch<T, 3, V>(kind, a, s);
        case 4: return conv_launch<T, 4, V>(kind, a, s);
        case 5: return conv_launch<T, 5, V>(kind, a, s);
        case 6: return conv_launch<T, 6, V>(kind, a, s);
        case 7: return conv_launch<T, 7, V>(kind, a, s);
        default: return conv_launch<T, 8, V>(kind, a, s);
    }
}

template <typename T> void conv_vector_width(ConvKind kind, const ConvArgs& a, int v, hipStream_t s) {
    if constexpr (sizeof(T) == 2) {
        if (v == 8) return conv_width<T, 8>(kind, a, s);
    }
    if (v == 4)
        conv_width<T, 4>(kind, a, s);
    else
        conv_width<T, 1>(kind, a, s);
}

void conv_dispatch(ConvKind kind, const ConvArgs& a, int v, hipStream_t s) {
    switch (a.c.dtype) {
        case ILX_F32: return conv_vector_width<float>(kind, a, v, s);
        case ILX_BF16: return conv_vector_width<bf16_t>(kind, a, v, s);
        default: return conv_vector_width<f16_t>(kind, a, v, s);
    }
}

}  // namespace

extern "C" int ilx_short_conv_forward(const ilx_short_conv* conv, void* stream) {
    ILX_REQUIRE(conv, ILX_EINVAL, "ilx_short_conv_forward: descriptor is NULL");
    const ilx_short_conv& c = *conv;
    const int rc = conv_check(c, "ilx_short_conv_forward");
    if (rc != ILX_OK) return rc;
    if (c.batch == 0) return ILX_OK;
    ILX_REQUIRE(c.weight && (c.length == 0 || (c.x && c.out)), ILX_EINVAL, "ilx_short_conv_forward: NULL operand");
    ILX_REQUIRE(!c.last || c.last != c.state, ILX_EINVAL, "ilx_short_conv_forward: last and state are the same buffer");
    const int v = conv_vector(c, false);
    const ConvArgs a = conv_args(c, v, false);
    ILX_REQUIRE(a.slots * a.channel_blocks * kConvThreads <= kMostThreads, ILX_ESHAPE, "ilx_short_conv_forward: shape too large for one launch");
    conv_dispatch(kForward, a, v, as_stream(stream));
    ILX_LAUNCH_CHECK("ilx_short_conv_forward");
    return ILX_OK;
}

extern "C" int ilx_short_conv_workspace(const ilx_short_conv* conv, int64_t* floats) {
    ILX_REQUIRE(conv && floats, ILX_EINVAL, "ilx_short_conv_workspace: NULL argument");
    const int rc = conv_check(*conv, "ilx_short_conv_workspace");
    if (rc != ILX_OK) return rc;
    const ConvArgs a = conv_args(*conv, conv_vector(*conv, true), true);
    *floats = a.slots * (conv->width + 1) * conv->channels;
    return ILX_OK;
}

extern "C" int ilx_short_conv_backward(const ilx_short_conv* conv, void* stream) {
    ILX_REQUIRE(conv, ILX_EINVAL, "ilx_short_conv_backward: descriptor is NULL");
    const ilx_short_conv& c = *conv;
    const int rc = conv_check(c, "ilx_short_conv_backward");
    if (rc != ILX_OK) return rc;
    ILX_REQUIRE(c.weight && c.grad_weight && (c.batch == 0 || c.length == 0 || (c.x && c.grad_out && c.grad_x)), ILX_EINVAL,
                "ilx_short_conv_backward: NULL operand");
    const int v = conv_vector(c, true);
    const ConvArgs a = conv_args(c, v, true);
    ILX_REQUIRE(a.slots * a.channel_blocks * kConvThreads <= kMostThreads, ILX_ESHAPE, "ilx_short_conv_backward: shape too large for one launch");
    ILX_REQUIRE(c.workspace_floats >= a.slots * (c.width + 1) * c.channels && (c.workspace || a.slots == 0), ILX_EINVAL,
                "ilx_short_conv_backward: workspace of %lld floats, %lld needed", (long long)c.workspace_floats,
                (long long)(a.slots * (c.width + 1) * c.channels));
    hipStream_t s = as_stream(stream);
    if (c.batch > 0) conv_dispatch(kBackward, a, v, s);
    launch_parameter_sums(c.workspace, a.slots, c.channels, c.width, 1, c.grad_weight, c.grad_bias, nullptr, s);
    ILX_LAUNCH_CHECK("ilx_short_conv_backward");
    return ILX_OK;
}

extern "C" int ilx_short_conv_step(const ilx_short_conv* conv, void* stream) {
    ILX_REQUIRE(conv, ILX_EINVAL, "ilx_short_conv_step: descriptor is NULL");
    ilx_short_conv c = *conv;
    c.length = 1;
    const int rc = conv_check(c, "ilx_short_conv_step");
    if (rc != ILX_OK) return rc;
    if (c.batch == 0) return ILX_OK;
    ILX_REQUIRE(c.x && c.weight && c.out && (c.width == 1 || (c.state && c.last)), ILX_EINVAL, "ilx_short_conv_step: NULL operand");
    ILX_REQUIRE(c.state == c.last, ILX_EINVAL, "ilx_short_conv_step: the state is updated in place, last must be state");
    ILX_REQUIRE(!c.lengths, ILX_EINVAL, "ilx_short_conv_step: lengths must be NULL");
    const int v = conv_vector(c, false);
    ConvArgs a = conv_args(c, v, false);
    a.items = c.batch * a.groups;
    ILX_REQUIRE(a.items <= kMostThreads, ILX_ESHAPE, "ilx_short_conv_step: shape too large for one launch");
    conv_dispatch(kStep, a, v, as_stream(stream));
    ILX_LAUNCH_CHECK("ilx_short_conv_step");
    return ILX_OK;
}
