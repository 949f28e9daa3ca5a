// Global norm of many gradient tensors, and their scaling in place.
// Two launches: every workgroup reduces its share of the elements to one number, then every workgroup of the second launch
// adds all these numbers in the same order (there are at most 1 024) and scales its share.  Bound by memory: two reads and one
// write of every element, the second read left out where nothing is to scale.  Squares are added in 64 bits, so a gradient
// of 1e30 has a norm and small gradients beside large ones count; the adds hide behind the loads.
// The tensors' pointers and sizes travel as kernel arguments, kTensors of them to a launch: no table in device memory that
// would have to be copied or kept for a replay.
#include "sequence_dev.h"

#include <algorithm>
#include <new>

namespace ilx {

constexpr int kTensors = 96;              // per launch
constexpr int64_t kChunk = 16384;         // elements: one share of a tensor
constexpr int kMostPartials = 1024;

struct TensorTable {
    void* data[kTensors];
    int64_t size[kTensors];
    int32_t first_chunk[kTensors + 1];    // chunks ahead of tensor i
    int32_t dtype[kTensors];
    int32_t count;
};

struct NormArgs {
    TensorTable t;
    double* partials;
    int32_t partial0, partials_here, partials_all;
    int32_t maximum;
    float max_norm;
    float* norm;
};

__device__ __forceinline__ int find_tensor(const TensorTable& t, int chunk) {
    int lo = 0, hi = t.count - 1;   // the last tensor whose first chunk is not past `chunk`
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (t.first_chunk[mid] <= chunk)
            lo = mid;
        else
            hi = mid - 1;
    }
    return lo;
}

// Calls f(value) for the elements of a chunk that fall to this thread, and with STORE writes back what it returns.
template <bool STORE, typename T, typename F> __device__ __forceinline__ void each_element(T* p, int64_t n, F f) {
    constexpr int V = 16 / sizeof(T);
    int64_t head = 0;   // elements ahead of the first 16-byte boundary
    const unsigned off = static_cast<unsigned>(reinterpret_cast<uintptr_t>(p) & 15) / sizeof(T);
    if (off) head = V - off < n ? V - off : n;
    const int64_t packs = (n - head) / V, tail = head + packs * V;
    if (static_cast<int64_t>(threadIdx.x) < head) {
        const float y = f(to_f32(p[threadIdx.x]));
        if (STORE) p[threadIdx.x] = from_f32<T>(y);
    }
    for (int64_t i = threadIdx.x; i < packs; i += blockDim.x) {
        float v[V];
        load_channels<V>(p + head + i * V, v);
#pragma unroll
        for (int k = 0; k < V; ++k) v[k] = f(v[k]);
        if (STORE) store_channels<V>(p + head + i * V, v);
    }
    const int64_t at = tail + threadIdx.x;
    if (at < n) {
        const float y = f(to_f32(p[at]));
        if (STORE) p[at] = from_f32<T>(y);
    }
}

template <bool STORE, typename F> __device__ __forceinline__ void each_in_chunk(const TensorTable& t, int chunk, F f) {
    const int i = find_tensor(t, chunk);
    const int64_t at = static_cast<int64_t>(chunk - t.first_chunk[i]) * kChunk;
    const int64_t n = t.size[i] - at < kChunk ? t.size[i] - at : kChunk;
    switch (t.dtype[i]) {
        case ILX_F32: each_element<STORE>(static_cast<float*>(t.data[i]) + at, n, f); break;
        case ILX_BF16: each_element<STORE>(static_cast<bf16_t*>(t.data[i]) + at, n, f); break;
        default: each_element<STORE>(static_cast<f16_t*>(t.data[i]) + at, n, f); break;
    }
}

// max that keeps a NaN
__device__ __forceinline__ double larger(double a, double b) { return a != a || a > b ? a : b; }

__device__ __forceinline__ double reduce_block(double v, bool maximum) {
    __shared__ double sums[16];
    for (int k = 32; k > 0; k >>= 1) {
        const double o = __shfl_xor(v, k);
        v = maximum ? larger(v, o) : v + o;
    }
    if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = v;
    __syncthreads();
    v = sums[0];
    for (unsigned k = 1; k < blockDim.x >> 6; ++k) v = maximum ? larger(v, sums[k]) : v + sums[k];
    return v;
}

__global__ void __launch_bounds__(256) gradient_partials_kernel(NormArgs a) {
    double s = 0.0;
    const int chunks = a.t.first_chunk[a.t.count];
    const bool maximum = a.maximum;
    for (int chunk = blockIdx.x; chunk < chunks; chunk += a.partials_here)
        each_in_chunk<false>(a.t, chunk, [&](float v) {
            const double d = v;
            s = maximum ? larger(__builtin_fabs(d), s) : __builtin_fma(d, d, s);
            return v;
        });
    s = reduce_block(s, maximum);
    if (threadIdx.x == 0) a.partials[a.partial0 + blockIdx.x] = s;
}

__global__ void __launch_bounds__(256) gradient_scale_kernel(NormArgs a) {
    const bool maximum = a.maximum;
    double s = 0.0;
    for (int i = threadIdx.x; i < a.partials_all; i += 256) s = maximum ? larger(a.partials[i], s) : s + a.partials[i];
    s = reduce_block(s, maximum);
    const float norm = static_cast<float>(maximum ? s : __builtin_sqrt(s));
    if (a.norm && blockIdx.x == 0 && threadIdx.x == 0) *a.norm = norm;
    const float ratio = a.max_norm / (norm + 1e-6f);
    const float scale = ratio > 1.0f ? 1.0f : ratio;   // NaN stays NaN
    if (scale == 1.0f) return;
    const int chunks = a.t.first_chunk[a.t.count];
    for (int chunk = blockIdx.x; chunk < chunks; chunk += gridDim.x) each_in_chunk<true>(a.t, chunk, [&](float v) { return v * scale; });
}

}  // namespace ilx

using namespace ilx;

namespace {

constexpr int kMostTables = kMostPartials / 4;

size_t element_size(int dtype) { return dtype == ILX_F32 ? 4 : 2; }
int64_t chunks_of(int64_t n) { return (n + kChunk - 1) / kChunk; }

// The tensors from number `next` on that fit one table, empty ones left out; returns the number behind the last.
int fill_table(TensorTable& t, void* const* data, const int64_t* sizes, const int32_t* dtypes, int count, int next) {
    t.count = 0, t.first_chunk[0] = 0;
    for (; next < count && t.count < kTensors; ++next) {
        if (sizes[next] == 0) continue;
        t.data[t.count] = data[next], t.size[t.count] = sizes[next], t.dtype[t.count] = dtypes[next];
        t.first_chunk[t.count + 1] = t.first_chunk[t.count] + static_cast<int32_t>(chunks_of(sizes[next]));
        ++t.count;
    }
    return next;
}

// Two tensors that share memory would be scaled twice, in no order.
int check_apart(void* const* data, const int64_t* sizes, const int32_t* dtypes, int count, int used) {
    struct Range {
        uintptr_t begin, end;
        int which;
    };
    Range* r = new (std::nothrow) Range[used > 0 ? used : 1];
    if (!r) return fail(ILX_EINVAL, "ilx_gradient_norm: out of host memory");
    int n = 0;
    for (int i = 0; i < count; ++i)
        if (sizes[i] > 0) {
            const uintptr_t p = reinterpret_cast<uintptr_t>(data[i]);
            r[n++] = {p, p + static_cast<uintptr_t>(sizes[i]) * element_size(dtypes[i]), i};
        }
    std::sort(r, r + n, [](const Range& x, const Range& y) { return x.begin < y.begin; });
    int rc = ILX_OK;
    for (int i = 1; i < n && rc == ILX_OK; ++i)
        if (r[i].begin < r[i - 1].end)
            rc = fail(ILX_EINVAL, "ilx_gradient_norm: tensors %d and %d share memory", r[i - 1].which, r[i].which);
    delete[] r;
    return rc;
}

}  // namespace

extern "C" int ilx_gradient_norm_workspace(const int64_t* sizes_host, int32_t count, int64_t* floats) {
    ILX_REQUIRE(floats && count >= 0 && (sizes_host || count == 0), ILX_EINVAL, "ilx_gradient_norm_workspace: bad argument");
    *floats = 2 * kMostPartials;
    return ILX_OK;
}

extern "C" int ilx_gradient_norm(void* const* tensors_host, const int64_t* sizes_host, const int32_t* dtypes_host, int32_t count,
                                 int32_t norm_kind, int32_t clip, float max_norm, float* norm, float* workspace, int64_t workspace_floats,
                                 void* stream) {
    ILX_REQUIRE(count >= 0 && (count == 0 || (tensors_host && sizes_host && dtypes_host)), ILX_EINVAL, "ilx_gradient_norm: bad tensor list");
    ILX_REQUIRE(norm_kind == 0 || norm_kind == 1, ILX_EINVAL, "ilx_gradient_norm: unknown norm %d", norm_kind);
    ILX_REQUIRE(norm, ILX_EINVAL, "ilx_gradient_norm: norm is NULL");
    ILX_REQUIRE(!clip || max_norm >= 0.0f, ILX_EINVAL, "ilx_gradient_norm: max_norm %g is negative or not a number", static_cast<double>(max_norm));
    ILX_REQUIRE(workspace && workspace_floats >= 2 * kMostPartials && aligned_to(workspace, 8), ILX_EINVAL,
                "ilx_gradient_norm: workspace of %lld floats, %d needed, 8-byte aligned", (long long)workspace_floats, 2 * kMostPartials);
    int64_t chunks_all = 0;
    int used = 0;   // tensors with elements
    for (int i = 0; i < count; ++i) {
        ILX_REQUIRE(sizes_host[i] >= 0 && (tensors_host[i] || sizes_host[i] == 0), ILX_EINVAL, "ilx_gradient_norm: tensor %d is NULL or of negative size", i);
        ILX_REQUIRE(dtypes_host[i] >= ILX_F32 && dtypes_host[i] <= ILX_F16, ILX_EINVAL, "ilx_gradient_norm: tensor %d has unknown type %d", i,
                    dtypes_host[i]);
        ILX_REQUIRE(aligned_to(tensors_host[i], element_size(dtypes_host[i])), ILX_EINVAL, "ilx_gradient_norm: tensor %d is not aligned to its type", i);
        chunks_all += chunks_of(sizes_host[i]);
        used += sizes_host[i] > 0;
    }
    ILX_REQUIRE(chunks_all < INT32_MAX, ILX_ESHAPE, "ilx_gradient_norm: too many elements");
    const int tables = used > 0 ? (used + kTensors - 1) / kTensors : 1;
    ILX_REQUIRE(tables <= kMostTables, ILX_ESHAPE, "ilx_gradient_norm: %d tensors (at most %d)", used, kTensors * kMostTables);
    if (clip) {
        const int rc = check_apart(tensors_host, sizes_host, dtypes_host, count, used);
        if (rc != ILX_OK) return rc;
    }
    // Both passes walk the tensors kTensors at a time; a table's workgroups of the first pass, and so its partial sums, are at
    // most its share of kMostPartials.
    const int most = kMostPartials / tables;
    NormArgs a{};
    a.partials = reinterpret_cast<double*>(workspace);
    a.maximum = norm_kind, a.max_norm = clip ? max_norm : 3.402823466e+38f;
    hipStream_t s = as_stream(stream);
    int at = 0;
    for (int k = 0, next = 0; k < tables; ++k) {
        next = fill_table(a.t, tensors_host, sizes_host, dtypes_host, count, next);
        const int chunks = a.t.first_chunk[a.t.count];
        a.partial0 = at, a.partials_here = chunks < 1 ? 1 : (chunks < most ? chunks : most);
        at += a.partials_here;
        ILX_LAUNCH(gradient_partials_kernel, dim3(a.partials_here), dim3(256), 0, s, a);
    }
    a.partials_all = at, a.norm = norm;
    if (!clip) {
        a.t.count = 0, a.t.first_chunk[0] = 0;
        ILX_LAUNCH(gradient_scale_kernel, dim3(1), dim3(256), 0, s, a);
    } else {
        for (int k = 0, next = 0; k < tables; ++k) {
            next = fill_table(a.t, tensors_host, sizes_host, dtypes_host, count, next);
            const int chunks = a.t.first_chunk[a.t.count];
            ILX_LAUNCH(gradient_scale_kernel, dim3(chunks < 1 ? 1 : (chunks < 2048 ? chunks : 2048)), dim3(256), 0, s, a);
            a.norm = nullptr;
        }
    }
    ILX_LAUNCH_CHECK("ilx_gradient_norm");
    return ILX_OK;
}
