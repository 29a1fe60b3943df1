// Global gradient norm over a list of tensors, and clipping in place (device half of nfe_grad_norm / nfe_grad_clip).  Part of
// nfe_planes.hip's code object: its callers optimise tri-planes.
//
//   t = sqrt(sum_i sum_j g_ij^2)   (or max |g_ij|),   f = min(1, max_norm / (t + 1e-6)),   g_ij <- round(f g_ij)
//
// Two launches for up to TABLE tensors (for more, two for each TABLE, of which each scaling one adds the partials of all): grad_reduce_kernel leaves one fp64 partial per workgroup, grad_clip_kernel adds the
// partials in their order in every workgroup (no atomics: the same call gives the same bits) and scales.  Nothing is read or written a
// second time when f = 1.  Both are bound by memory: 50.3 million fp32 values (201 MB) take 48.6 + 65.9 us, three passes at the 5.3 TB/s of a
// large copy; 6.3 million that need no clipping 6.8 + 4.5 us.  (Clipping from the last chunk back, to find it in the last-level cache, changed
// nothing.)  The table of tensors travels by value in the kernel's arguments, so a captured
// call replays without a host copy.
#pragma once
#include <algorithm>
#include <exception>
#include <utility>
#include <vector>

#include "nfe_dense.h"
#include "nfe_wave.h"

NFE_NO_PACKED_FP32_BEGIN

namespace nfe {
namespace grad {

constexpr int TABLE = 256;             // tensors per launch: 14 bytes each keep the kernel's arguments under 4 KB
constexpr int CHUNK = 4096;            // elements a workgroup takes at a time: 16 KB chunks share 2048 workgroups evenly (64 KB ones left a tail)
constexpr int MAX_BLOCKS = 2048;       // 8 workgroups of 256 threads per CU; also the partials of one launch
constexpr int THREADS = 256;
constexpr int SMALL = 4;               // chunks that one workgroup takes alone
constexpr long long MAX_ELEMENTS = 1ll << 34;      // of one tensor (32 GB at least): TABLE of them stay below 2^31 chunks
static_assert(TABLE * (MAX_ELEMENTS / CHUNK) < 0x7fffffffll, "chunk numbers are 32-bit");

struct Table {
    unsigned long long where[TABLE];   // address, type << 62
    int first[TABLE + 1];              // chunks before tensor i
    unsigned short last[TABLE];        // elements of its last chunk
    int count;
};
static_assert(sizeof(Table) <= 3840, "kernel arguments stay under 4 KB");

template <typename T> struct alignas(16) Vec { static constexpr int N = 16 / (int)sizeof(T); T e[N]; };

// |x| as bits, so that a NaN is larger than everything and survives the maximum
__device__ __forceinline__ unsigned abs_bits(float v) { return bits_of(v) & 0x7fffffffu; }

struct Sum {        // fp64: squares of any fp32 value stay in range, and 2^31 values lose nothing that fp32 shows
    double s;
    __device__ __forceinline__ void clear() { s = 0.0; }
    __device__ __forceinline__ void add(float v) { const double d = (double)v; s = fma(d, d, s); }
    __device__ __forceinline__ void join(const Sum& o) { s += o.s; }
    __device__ __forceinline__ Sum shuffled(int off) const { Sum r; r.s = wave_xor(s, off); return r; }
    __device__ __forceinline__ double partial() const { return s; }
    __device__ __forceinline__ void from(double p) { s = p; }
    __device__ __forceinline__ double norm() const { return sqrt(s); }
};
struct Max {
    unsigned m;
    __device__ __forceinline__ void clear() { m = 0; }
    __device__ __forceinline__ void add(float v) { const unsigned b = abs_bits(v); m = m > b ? m : b; }
    __device__ __forceinline__ void join(const Max& o) { m = m > o.m ? m : o.m; }
    __device__ __forceinline__ Max shuffled(int off) const { Max r; r.m = wave_xor(m, off); return r; }
    __device__ __forceinline__ double partial() const { return (double)float_of(m); }
    __device__ __forceinline__ void from(double p) { m = abs_bits((float)p); }
    __device__ __forceinline__ double norm() const { return (double)float_of(m); }
};

template <typename ACC>
__device__ __forceinline__ ACC block_reduce(ACC a, ACC* lds) {          // every thread gets the result; fixed order
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) a.join(a.shuffled(off));
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = a;
    block_sync();
    ACC r = lds[0];
#pragma unroll
    for (int w = 1; w < THREADS / 64; ++w) r.join(lds[w]);
    return r;
}

__device__ __forceinline__ int find_tensor(const Table& t, int chunk) {  // uniform: last i with first[i] <= chunk
    int a = 0, b = t.count;
    while (b - a > 1) { const int m = (a + b) >> 1; if (t.first[m] <= chunk) a = m; else b = m; }
    return a;
}

// A chunk as [head][16-byte vectors][tail]: views may start anywhere
template <typename T> struct Span {
    T* p; int head, vecs, tail;
    __device__ __forceinline__ Span(void* data, int len) {
        p = (T*)data;
        const int lead = (int)((16u - ((unsigned)(unsigned long long)p & 15u)) & 15u) / (int)sizeof(T);
        head = lead < len ? lead : len;
        vecs = (len - head) / Vec<T>::N;
        tail = len - head - vecs * Vec<T>::N;
    }
};

template <typename T, typename ACC>
__device__ __forceinline__ void reduce_chunk(ACC& acc, void* data, int len) {
    constexpr int V = Vec<T>::N, U = CHUNK / (V * THREADS);
    const Span<T> s(data, len);
    const int tid = threadIdx.x;
    if (tid < s.head) acc.add((float)s.p[tid]);
    if (tid < s.tail) acc.add((float)s.p[s.head + s.vecs * V + tid]);
    const Vec<T>* v = (const Vec<T>*)(s.p + s.head);
    int i = tid;
    for (; i + (U - 1) * THREADS < s.vecs; i += U * THREADS) {
        Vec<T> q[U];
#pragma unroll
        for (int u = 0; u < U; ++u) q[u] = v[i + u * THREADS];
#pragma unroll
        for (int u = 0; u < U; ++u) {
#pragma unroll
            for (int k = 0; k < V; ++k) acc.add((float)q[u].e[k]);
        }
    }
    for (; i < s.vecs; i += THREADS) {
        const Vec<T> q = v[i];
#pragma unroll
        for (int k = 0; k < V; ++k) acc.add((float)q.e[k]);
    }
}

template <typename T>
__device__ __forceinline__ void scale_chunk(float f, void* data, int len) {
    constexpr int V = Vec<T>::N, U = CHUNK / (V * THREADS);
    const Span<T> s(data, len);
    const int tid = threadIdx.x;
    if (tid < s.head) s.p[tid] = (T)((float)s.p[tid] * f);
    if (tid < s.tail) { T* e = s.p + s.head + s.vecs * V + tid; *e = (T)((float)*e * f); }
    Vec<T>* v = (Vec<T>*)(s.p + s.head);
    int i = tid;
    for (; i + (U - 1) * THREADS < s.vecs; i += U * THREADS) {
        Vec<T> q[U];
#pragma unroll
        for (int u = 0; u < U; ++u) q[u] = v[i + u * THREADS];
#pragma unroll
        for (int u = 0; u < U; ++u) {
#pragma unroll
            for (int k = 0; k < V; ++k) q[u].e[k] = (T)((float)q[u].e[k] * f);
            v[i + u * THREADS] = q[u];
        }
    }
    for (; i < s.vecs; i += THREADS) {
        Vec<T> q = v[i];
#pragma unroll
        for (int k = 0; k < V; ++k) q.e[k] = (T)((float)q.e[k] * f);
        v[i] = q;
    }
}

// body(type, address, elements) for every chunk of this workgroup.  Chunk numbers rise, so the tensor is looked up only when one is left.
template <typename F>
__device__ __forceinline__ void each_chunk(const Table& t, F body) {
    const int chunks = t.first[t.count];
    int i = 0, from = 0, to = 0;
    for (int c = blockIdx.x; c < chunks; c += gridDim.x) {
        if (c >= to) { i = find_tensor(t, c); from = t.first[i]; to = t.first[i + 1]; }
        const unsigned long long where = t.where[i];
        const int type = (int)(where >> 62);
        const long long at = (long long)(c - from) * CHUNK;
        body(type, (char*)(where & ((1ull << 62) - 1)) + at * (type == NFE_F32 ? 4 : 2), c + 1 == to ? (int)t.last[i] : CHUNK);
    }
}

template <typename ACC>
__device__ __forceinline__ ACC reduce_all(const Table& t, ACC* lds) {
    ACC acc; acc.clear();
    each_chunk(t, [&](int type, void* p, int len) {
        if (type == NFE_F32) reduce_chunk<float>(acc, p, len);
        else if (type == NFE_BF16) reduce_chunk<__bf16>(acc, p, len);
        else reduce_chunk<_Float16>(acc, p, len);
    });
    return block_reduce(acc, lds);
}
__device__ __forceinline__ void scale_all(const Table& t, float f) {
    each_chunk(t, [&](int type, void* p, int len) {
        if (type == NFE_F32) scale_chunk<float>(f, p, len);
        else if (type == NFE_BF16) scale_chunk<__bf16>(f, p, len);
        else scale_chunk<_Float16>(f, p, len);
    });
}
__device__ __forceinline__ float factor(double max_norm, double total) { return (float)(max_norm / (total + 1e-6)); }

template <typename ACC>
__global__ __launch_bounds__(THREADS) void grad_reduce_kernel(Table t, double* __restrict__ partial) {
    __shared__ ACC lds[THREADS / 64];
    const ACC acc = reduce_all(t, lds);
    if (threadIdx.x == 0) partial[blockIdx.x] = acc.partial();
}

// A handful of chunks: one workgroup does all of it in one launch (2 x 96 values: 13.4 -> 10.4 us a call, of which 3.6 us are a launch)
template <typename ACC>
__global__ __launch_bounds__(THREADS) void grad_small_kernel(Table t, int clip, float max_norm, float* __restrict__ norm) {
    __shared__ ACC lds[THREADS / 64];
    const double total = reduce_all<ACC>(t, lds).norm();
    if (threadIdx.x == 0) *norm = (float)total;
    if (!clip) return;
    const float f = factor(max_norm, total);
    if (f >= 1.0f) return;             // every value has been read: block_reduce has a barrier
    scale_all(t, f);
}

// clip = 0: the norm alone (one workgroup, an empty table)
template <typename ACC>
__global__ __launch_bounds__(THREADS) void grad_clip_kernel(Table t, const double* __restrict__ partial, int n_partial, int clip, float max_norm,
                                                            float* __restrict__ norm) {
    __shared__ ACC lds[THREADS / 64];
    ACC acc; acc.clear();
    for (int i = threadIdx.x; i < n_partial; i += THREADS) { ACC p; p.from(partial[i]); acc.join(p); }
    const double total = block_reduce(acc, lds).norm();
    if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)total;
    if (!clip) return;
    const float f = factor(max_norm, total);
    if (f >= 1.0f) return;             // a NaN goes on and makes every gradient NaN
    scale_all(t, f);
}

// ---- host ------------------------------------------------------------------------------------
static int check_list(const char* who, const uint64_t* data, const int64_t* n, const int32_t* dtype, int count, bool writes) {
    NFE_REQUIRE(data && n && dtype, "%s: null pointer", who);
    NFE_REQUIRE(count > 0, "%s: count=%d must be positive", who, count);
    for (int i = 0; i < count; ++i) {
        NFE_REQUIRE(n[i] >= 0 && n[i] <= MAX_ELEMENTS, "%s: tensor %d has %lld elements", who, i, (long long)n[i]);
        NFE_REQUIRE(dtype[i] == NFE_F32 || dtype[i] == NFE_BF16 || dtype[i] == NFE_F16, "%s: tensor %d has unknown dtype %d", who, i, (int)dtype[i]);
        const int size = dtype[i] == NFE_F32 ? 4 : 2;
        NFE_REQUIRE(n[i] == 0 || (data[i] && data[i] % size == 0 && data[i] >> 62 == 0), "%s: tensor %d: null or misaligned pointer", who, i);
    }
    if (!writes) return NFE_OK;
    // two entries that share memory would be scaled by two workgroups at once
    try {
        std::vector<std::pair<uint64_t, uint64_t>> span;
        span.reserve(count);
        for (int i = 0; i < count; ++i)
            if (n[i]) span.emplace_back(data[i], data[i] + (uint64_t)n[i] * (dtype[i] == NFE_F32 ? 4 : 2));
        std::sort(span.begin(), span.end());
        for (size_t i = 1; i < span.size(); ++i) NFE_REQUIRE(span[i].first >= span[i - 1].second, "%s: two tensors of the list share memory", who);
    } catch (const std::exception& e) {
        return fail(NFE_EINVAL, "%s: %s", who, e.what());
    }
    return NFE_OK;
}
// tables of up to TABLE non-empty tensors; returns the blocks of each
struct Launch { Table t; int blocks; };
static void fill(Launch& l, const uint64_t* data, const int64_t* n, const int32_t* dtype, int count, int& at) {
    Table& t = l.t;
    t.count = 0;
    long long chunks = 0;
    for (; at < count && t.count < TABLE; ++at) {
        if (!n[at]) continue;
        const long long c = (n[at] + CHUNK - 1) / CHUNK;
        const int i = t.count++;
        t.where[i] = data[at] | (unsigned long long)dtype[at] << 62;
        t.last[i] = (unsigned short)(n[at] - (c - 1) * CHUNK);
        t.first[i] = (int)chunks;
        chunks += c;
    }
    t.first[t.count] = (int)chunks;
    l.blocks = (int)(chunks < MAX_BLOCKS ? chunks : MAX_BLOCKS);
}

template <typename ACC>
static int run(const char* who, const uint64_t* data, const int64_t* n, const int32_t* dtype, int count, int clip, float max_norm, float* norm, double* partial,
               hipStream_t st) {
    int n_partial = 0;
    Launch l;
    int end = 0;
    fill(l, data, n, dtype, count, end);
    if (end == count && l.blocks <= SMALL) {
        hipLaunchKernelGGL((grad_small_kernel<ACC>), dim3(1), dim3(THREADS), 0, st, l.t, clip, max_norm, norm);
        NFE_CHECK_LAUNCH(who);
        return NFE_OK;
    }
    for (int at = 0; at < count;) {
        fill(l, data, n, dtype, count, at);
        if (!l.blocks) break;
        hipLaunchKernelGGL((grad_reduce_kernel<ACC>), dim3((unsigned)l.blocks), dim3(THREADS), 0, st, l.t, partial + n_partial);
        NFE_CHECK_LAUNCH(who);
        n_partial += l.blocks;
    }
    bool wrote = false;
    if (clip)
        for (int at = 0; at < count;) {
            fill(l, data, n, dtype, count, at);
            if (!l.blocks) break;
            hipLaunchKernelGGL((grad_clip_kernel<ACC>), dim3((unsigned)l.blocks), dim3(THREADS), 0, st, l.t, (const double*)partial, n_partial, 1, max_norm,
                               wrote ? (float*)nullptr : norm);
            NFE_CHECK_LAUNCH(who);
            wrote = true;
        }
    if (!wrote) {
        l.t.count = 0; l.t.first[0] = 0;
        hipLaunchKernelGGL((grad_clip_kernel<ACC>), dim3(1), dim3(THREADS), 0, st, l.t, (const double*)partial, n_partial, 0, 0.0f, norm);
        NFE_CHECK_LAUNCH(who);
    }
    return NFE_OK;
}
static int entry(const char* who, const uint64_t* data, const int64_t* n, const int32_t* dtype, int count, int norm_type, int clip, float max_norm, float* norm,
                 void* workspace, uint64_t workspace_bytes, nfe_stream_t stream) {
    if (int rc = check_list(who, data, n, dtype, count, clip != 0)) return rc;
    NFE_REQUIRE(norm_type == NFE_NORM_2 || norm_type == NFE_NORM_MAX, "%s: unknown norm_type %d", who, norm_type);
    NFE_REQUIRE(norm && workspace && (uintptr_t)workspace % 8 == 0, "%s: null or misaligned norm / workspace", who);
    NFE_REQUIRE(!clip || max_norm >= 0.0f, "%s: max_norm must be >= 0", who);
    if (workspace_bytes < nfe_grad_workspace_bytes(count)) return fail(NFE_EWORKSPACE, "%s: workspace too small", who);
    return (norm_type == NFE_NORM_2 ? run<Sum> : run<Max>)(who, data, n, dtype, count, clip, max_norm, norm, (double*)workspace, (hipStream_t)stream);
}

}  // namespace grad
}  // namespace nfe

NFE_NO_PACKED_FP32_END

extern "C" uint64_t nfe_grad_workspace_bytes(int count) {
    using namespace nfe::grad;
    return count > 0 ? ((uint64_t)count + TABLE - 1) / TABLE * MAX_BLOCKS * sizeof(double) : 0;
}
extern "C" int nfe_grad_norm(const uint64_t* data, const int64_t* n, const int32_t* dtype, int count, int norm_type, float* norm, void* workspace,
                             uint64_t workspace_bytes, nfe_stream_t stream) {
    return nfe::grad::entry("nfe_grad_norm", data, n, dtype, count, norm_type, 0, 0.0f, norm, workspace, workspace_bytes, stream);
}
extern "C" int nfe_grad_clip(const uint64_t* data, const int64_t* n, const int32_t* dtype, int count, int norm_type, float max_norm, float* norm,
                             void* workspace, uint64_t workspace_bytes, nfe_stream_t stream) {
    return nfe::grad::entry("nfe_grad_clip", data, n, dtype, count, norm_type, 1, max_norm, norm, workspace, workspace_bytes, stream);
}
