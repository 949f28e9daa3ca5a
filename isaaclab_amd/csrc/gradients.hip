// Global norm of many gradient tensors, and their scaling in place.
// Two launches: every workgroup reduces its share of the elements to one number, then every workgroup of the second launch
// adds all these numbers in the same order (there are at most 2 048) and scales its share.  Bound by memory: two reads and one
// write of every element, the second read left out where nothing is to scale.  Squares are added in 64 bits, so a gradient
// of 1e30 has a norm and small gradients beside large ones count; the adds hide behind the loads.
// The tensors' pointers and sizes travel as kernel arguments, kTensors of them to a launch: no table in device memory that
// would have to be copied or kept for a replay.
// Measured, 200 tensors of 200 M bf16 elements together: 121 us for the sums (400 MB, 3.3 TB/s; 94 where the last-level cache holds part of
// them) and 126 to scale (800 MB; part of what it reads is still in that cache), against 4.97 TB/s of a large copy.  16 tensors of a
// policy (572 K f32): 6.2 and 5.6 us in 46 shares: most of the chip has none.
#include "sequence_dev.h"

#include <algorithm>
#include <new>

namespace ilx {

constexpr size_t kArgumentBytes = 4096 - 256;   // of a kernel: 4 KB with the runtime's own
constexpr int kTensors = 223;             // per launch: as many as fit the arguments
constexpr uint32_t kChunk = 16384;        // elements: one share of a tensor
constexpr int64_t kMostElements = int64_t{1} << 30;   // of an entry; a larger tensor takes several
constexpr int kMostPartials = 2048;
constexpr int kPacks = 8;                 // 16-byte reads that a thread has in flight

struct TensorTable {
    void* data[kTensors];
    uint32_t size[kTensors];
    int32_t first_chunk[kTensors + 1];    // chunks ahead of entry i
    uint8_t dtype[kTensors];
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
static_assert(sizeof(NormArgs) <= kArgumentBytes && sizeof(NormArgs) + 8 + 4 + 4 + 1 > kArgumentBytes, "kernel arguments");

// The entry of a chunk: the last one whose first chunk is not past it.  A wave holds all first chunks, read together (a search of the
// table would wait for one read of the arguments after the other), and counts.
struct ChunkFinder {
    int32_t first[(kTensors + 63) / 64];
    __device__ __forceinline__ explicit ChunkFinder(const TensorTable& t) {
        const int lane = threadIdx.x & 63;
#pragma unroll
        for (int k = 0; k < (kTensors + 63) / 64; ++k) first[k] = 64 * k + lane < t.count ? t.first_chunk[64 * k + lane] : INT32_MAX;
    }
    __device__ __forceinline__ int operator()(int chunk) const {
        int n = 0;
#pragma unroll
        for (int k = 0; k < (kTensors + 63) / 64; ++k) n += __popcll(__ballot(first[k] <= chunk));
        return n - 1;
    }
};

// Calls f(value) for the elements of a chunk that fall to this thread, and with STORE writes back what it returns.
template <bool STORE, typename T, typename F> __device__ __forceinline__ void each_element(T* p, uint32_t n, F f) {
    constexpr uint32_t V = 16 / sizeof(T);
    const uint32_t off = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(p) & 15) / sizeof(T);
    const uint32_t head = off == 0 ? 0 : (V - off < n ? V - off : n);   // elements ahead of the first 16-byte boundary
    const uint32_t packs = (n - head) / V, tail = head + packs * V;
    if (threadIdx.x < head) {
        const float y = f(to_f32(p[threadIdx.x]));
        if (STORE) p[threadIdx.x] = from_f32<T>(y);
    }
    Pack<T, V>* q = reinterpret_cast<Pack<T, V>*>(p + head);
    for (uint32_t i = threadIdx.x; i < packs; i += kPacks * 256) {
        Pack<T, V> v[kPacks];
#pragma unroll
        for (int k = 0; k < kPacks; ++k) v[k] = q[i + k * 256 < packs ? i + k * 256 : i];
#pragma unroll
        for (int k = 0; k < kPacks; ++k) {
            if (i + k * 256 < packs) {
#pragma unroll
                for (uint32_t e = 0; e < V; ++e) {
                    const float y = f(to_f32(v[k].v[e]));
                    if (STORE) v[k].v[e] = from_f32<T>(y);
                }
                if (STORE) q[i + k * 256] = v[k];
            }
        }
    }
    const uint32_t at = tail + threadIdx.x;
    if (at < n) {
        const float y = f(to_f32(p[at]));
        if (STORE) p[at] = from_f32<T>(y);
    }
}

template <bool STORE, typename F> __device__ __forceinline__ void each_in_chunk(const TensorTable& t, const ChunkFinder& entry_of, int chunk, F f) {
    const int i = entry_of(chunk);
    const uint32_t at = static_cast<uint32_t>(chunk - t.first_chunk[i]) * kChunk, left = t.size[i] - at;
    const uint32_t n = left < kChunk ? left : kChunk;
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
    const ChunkFinder entry_of(a.t);
    for (int chunk = blockIdx.x; chunk < chunks; chunk += a.partials_here)
        each_in_chunk<false>(a.t, entry_of, chunk, [&](float v) {
            const double d = v;
            s = maximum ? larger(__builtin_fabs(d), s) : __builtin_fma(d, d, s);
            return v;
        });
    s = reduce_block(s, maximum);
    if (threadIdx.x == 0) a.partials[a.partial0 + blockIdx.x] = s;
}

__global__ void __launch_bounds__(256) gradient_scale_kernel(NormArgs a) {
    const bool maximum = a.maximum;
    const ChunkFinder entry_of(a.t);
    double s = 0.0;
    for (int i = threadIdx.x; i < a.partials_all; i += 256) s = maximum ? larger(a.partials[i], s) : s + a.partials[i];
    s = reduce_block(s, maximum);
    const float norm = static_cast<float>(maximum ? s : __builtin_sqrt(s));
    if (a.norm && blockIdx.x == 0 && threadIdx.x == 0) *a.norm = norm;
    // The reciprocal is rounded ahead of the product, as torch rounds a number over a tensor: one last bit of the scale moves
    // every 16-bit gradient whose product lies halfway, one in 128 of them, and a run that changes over keeps its results.
    const float ratio = a.max_norm * (1.0f / (norm + 1e-6f));
    const float scale = ratio > 1.0f ? 1.0f : ratio;   // NaN stays NaN
    if (scale == 1.0f) return;
    const int chunks = a.t.first_chunk[a.t.count];
    for (int chunk = blockIdx.x; chunk < chunks; chunk += gridDim.x) each_in_chunk<true>(a.t, entry_of, chunk, [&](float v) { return v * scale; });
}

}  // namespace ilx

using namespace ilx;

namespace {

constexpr int kMostTables = kMostPartials / 16;

size_t element_size(int dtype) { return dtype == ILX_F32 ? 4 : 2; }
int64_t chunks_of(int64_t n) { return (n + kChunk - 1) / kChunk; }
int64_t entries_of(int64_t n) { return (n + kMostElements - 1) / kMostElements; }

// Where a walk over the tensors' entries is: entry `part` of tensor `which`.
struct Walk {
    int which = 0;
    int64_t part = 0;
};

// The next entries that fit one table, empty tensors left out.
void fill_table(TensorTable& t, void* const* data, const int64_t* sizes, const int32_t* dtypes, int count, Walk& w) {
    t.count = 0, t.first_chunk[0] = 0;
    while (w.which < count && t.count < kTensors) {
        const int64_t begin = w.part * kMostElements, left = sizes[w.which] - begin;
        if (left <= 0) {
            ++w.which, w.part = 0;
            continue;
        }
        const int64_t n = left < kMostElements ? left : kMostElements;
        t.data[t.count] = static_cast<char*>(data[w.which]) + begin * element_size(dtypes[w.which]);
        t.size[t.count] = static_cast<uint32_t>(n), t.dtype[t.count] = static_cast<uint8_t>(dtypes[w.which]);
        t.first_chunk[t.count + 1] = t.first_chunk[t.count] + static_cast<int32_t>(chunks_of(n));
        ++t.count, ++w.part;
    }
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
    int64_t entries = 0;
    int used = 0;   // tensors with elements
    for (int i = 0; i < count; ++i) {
        ILX_REQUIRE(sizes_host[i] >= 0 && (tensors_host[i] || sizes_host[i] == 0), ILX_EINVAL, "ilx_gradient_norm: tensor %d is NULL or of negative size", i);
        ILX_REQUIRE(dtypes_host[i] >= ILX_F32 && dtypes_host[i] <= ILX_F16, ILX_EINVAL, "ilx_gradient_norm: tensor %d has unknown type %d", i,
                    dtypes_host[i]);
        ILX_REQUIRE(aligned_to(tensors_host[i], element_size(dtypes_host[i])), ILX_EINVAL, "ilx_gradient_norm: tensor %d is not aligned to its type", i);
        entries += entries_of(sizes_host[i]);
        used += sizes_host[i] > 0;
    }
    ILX_REQUIRE(entries <= kTensors * kMostTables, ILX_ESHAPE, "ilx_gradient_norm: %d tensors, %lld pieces of 2^30 elements (at most %d)", used,
                (long long)entries, kTensors * kMostTables);
    const int tables = entries > 0 ? static_cast<int>((entries + kTensors - 1) / kTensors) : 1;
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
    Walk walk;
    for (int k = 0; k < tables; ++k) {
        fill_table(a.t, tensors_host, sizes_host, dtypes_host, count, walk);
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
        walk = Walk();
        for (int k = 0; k < tables; ++k) {
            if (tables > 1) fill_table(a.t, tensors_host, sizes_host, dtypes_host, count, walk);   // (else it is filled)
            const int chunks = a.t.first_chunk[a.t.count];
            ILX_LAUNCH(gradient_scale_kernel, dim3(chunks < 1 ? 1 : (chunks < 4096 ? chunks : 4096)), dim3(256), 0, s, a);
            a.norm = nullptr;
        }
    }
    ILX_LAUNCH_CHECK("ilx_gradient_norm");
    return ILX_OK;
}
