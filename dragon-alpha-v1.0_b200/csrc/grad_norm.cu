// The 2-norm of all gradients of a step, and the gradients scaled down to a largest norm.
//
// Two passes at HBM speed, each one launch for every 128 tensors: sums of squares, a partial sum per CTA; then every CTA adds the
// partial sums (the same few thousand bytes from L2, in the same order) and scales its share.  The second pass walks backwards, so that it begins with what the
// first one left in L2.  A tensor is cut into chunks of 8192 elements, counted from the 16-byte boundary at or before its start, so that whole
// words are aligned wherever it begins; a CTA takes every gridDim.x-th chunk of the launch.
//
// A word of 4 or 8 elements is summed in fp32 and added to a thread's sum in fp64: one fp64 addition a word keeps the conversions, 16 a clock of
// an SM, out of the way, and rounds a word's squares by 2^-24 each way, 1e-8 of a norm.  Where that sum is not between 2^-110 and 2^120 its
// squares may have left fp32's range, and the word is summed in fp64 throughout.
#include "../../include/alpha_conv_b200.h"
#include "dependent_launch.cuh"
#include "fc_act.cuh"
#include "host_common.h"

#include <algorithm>
#include <exception>
#include <vector>

namespace alpha {
namespace {

constexpr int kGradTensors = 128, kGradThreads = 256;
constexpr long long kGradChunk = 8192;

struct GradTensor {
    const void* grad;
    void* out;
    long long count;
    int lead;                       // elements from the 16-byte boundary to the first
    unsigned char type, out_type, in_place, out_words;   // out_words: the words of `out` start at 16-byte boundaries too
};
struct GradTable {
    GradTensor t[kGradTensors];
    unsigned first[kGradTensors + 1];   // first chunk of each tensor; the last: chunks in all
    int n;
};

// Chunk -> tensor and the chunk's number within it.
__device__ __forceinline__ const GradTensor& find_tensor(const GradTable& g, unsigned chunk, long long& begin)
{
    int lo = 0, hi = g.n;               // first[lo] <= chunk < first[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (g.first[mid] <= chunk) lo = mid;
        else hi = mid;
    }
    begin = static_cast<long long>(chunk - g.first[lo]) * kGradChunk;
    return g.t[lo];
}

template <class T> __device__ __forceinline__ float element(const T* p);
template <> __device__ __forceinline__ float element<float>(const float* p) { return *p; }
template <> __device__ __forceinline__ float element<__nv_bfloat16>(const __nv_bfloat16* p) { return __bfloat162float(*p); }
template <> __device__ __forceinline__ float element<__half>(const __half* p) { return __half2float(*p); }
__device__ __forceinline__ void put_element(float* p, float x) { *p = x; }
__device__ __forceinline__ void put_element(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }
__device__ __forceinline__ void put_element(__half* p, float x) { *p = __float2half_rn(x); }

template <class F> __device__ __forceinline__ void with_type(int type, F&& f)
{
    if (type == ALPHA_F32) f(float{});
    else if (type == ALPHA_BF16) f(__nv_bfloat16{});
    else f(__half{});
}

// (a gradient may be its own output: not by the read-only path)
__device__ __forceinline__ uint4 load_once(const uint4* p)
{
    uint4 v;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
    return v;
}

template <int N> __device__ __forceinline__ double word_squares(const float (&f)[N])
{
    float s = f[0] * f[0];
#pragma unroll
    for (int i = 1; i < N; ++i) s = fmaf(f[i], f[i], s);
    if (s > 0x1p-110f && s < 0x1p120f) return s;
    double d = 0.0;
#pragma unroll
    for (int i = 0; i < N; ++i) d = fma(static_cast<double>(f[i]), static_cast<double>(f[i]), d);
    return d;
}

// Sum over the threads of a CTA, in every thread, in a fixed order.
__device__ __forceinline__ double cta_sum(double s, double* shared)
{
#pragma unroll
    for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
    if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = s;
    __syncthreads();
    s = 0.0;
#pragma unroll
    for (int w = 0; w < kGradThreads / 32; ++w) s += shared[w];
    return s;
}

// Elements of a chunk: word(w, number) for whole words, single(v) for the elements of words at the ends of the tensor (v counts from the boundary).
// A chunk of whole words is loaded at once, so that all loads of a thread are in flight together.
template <int N, class Word, class Single>
__device__ __forceinline__ void walk_chunk(const GradTensor& t, const uint4* base, long long begin, Word&& word, Single&& single)
{
    const long long end = t.lead + t.count;                          // in elements from the boundary
    constexpr int kWords = kGradChunk / N / kGradThreads;
    if (begin >= t.lead && begin + kGradChunk <= end) {
        const long long first = begin / N + threadIdx.x;
        uint4 w[kWords];
#pragma unroll
        for (int i = 0; i < kWords; ++i) w[i] = load_once(base + first + i * kGradThreads);
#pragma unroll
        for (int i = 0; i < kWords; ++i) word(w[i], first + i * kGradThreads);
        return;
    }
    const long long stop = begin + kGradChunk < end ? begin + kGradChunk : end;
    for (long long v = begin + static_cast<long long>(threadIdx.x) * N; v < stop; v += static_cast<long long>(kGradThreads) * N) {
        if (v >= t.lead && v + N <= stop) word(load_once(base + v / N), v / N);
        else
            for (long long e = v < t.lead ? t.lead : v; e < v + N && e < stop; ++e) single(e);
    }
}

__global__ void __launch_bounds__(kGradThreads) grad_squares_kernel(const __grid_constant__ GradTable g, double* part)
{
    __shared__ double shared[kGradThreads / 32];
    grid_dependency_wait();
    grid_dependency_trigger();
    double sum = 0.0;
    for (unsigned chunk = blockIdx.x; chunk < g.first[g.n]; chunk += gridDim.x) {
        long long begin;
        const GradTensor& t = find_tensor(g, chunk, begin);
        with_type(t.type, [&](auto type) {
            using T = decltype(type);
            constexpr int N = Word16<T>::N;
            const T* base = static_cast<const T*>(t.grad) - t.lead;
            walk_chunk<N>(t, reinterpret_cast<const uint4*>(base), begin,
                [&](const uint4& v, long long) {
                    float f[N];
                    Word16<T>::load(v, f);
                    sum += word_squares(f);
                },
                [&](long long e) { const double x = element(base + e); sum = fma(x, x, sum); });
        });
    }
    sum = cta_sum(sum, shared);
    if (threadIdx.x == 0) part[blockIdx.x] = sum;
}

__device__ __forceinline__ double norm_of(const double* part, int parts, double* shared)
{
    double s = 0.0;
    for (int i = threadIdx.x; i < parts; i += kGradThreads) s += part[i];
    return sqrt(cta_sum(s, shared));
}

__global__ void __launch_bounds__(kGradThreads) grad_norm_kernel(const double* part, int parts, float* norm)
{
    __shared__ double shared[kGradThreads / 32];
    grid_dependency_wait();
    grid_dependency_trigger();
    const double n = norm_of(part, parts, shared);
    if (threadIdx.x == 0) *norm = static_cast<float>(n);
}

// (norm: written by CTA 0 where it is not nullptr)
__global__ void __launch_bounds__(kGradThreads) grad_scale_kernel(const __grid_constant__ GradTable g, const double* part, int parts, double max_norm, float* norm)
{
    __shared__ double shared[kGradThreads / 32];
    grid_dependency_wait();
    grid_dependency_trigger();
    const double n = norm_of(part, parts, shared), ratio = max_norm / (n + 1e-6);
    if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = static_cast<float>(n);
    const bool one = ratio >= 1.0;                                   // (a NaN is not)
    // two factors where a single one would be near or among the denormals
    const double scaled = one ? 1.0 : ratio < 0x1p-60 ? ratio * 0x1p60 : ratio;
    const float tail = ratio < 0x1p-60 ? 0x1p-60f : 1.f;
    // c in two floats for fp32 outputs, so that a product is rounded once: with max_norm and c as floats they erred by 9.6e-8, not 3e-8.  (For 16-bit
    // ones it changes nothing but the time, 0.8 billion elements 815 -> 875 us.)
    const float c = static_cast<float>(scaled), c_low = static_cast<float>(scaled - static_cast<double>(c));
    auto times = [&](float f, auto out) { return (sizeof(out) == 4 ? fmaf(f, c, f * c_low) : f * c) * tail; };
    const unsigned chunks = g.first[g.n];
    for (unsigned q = blockIdx.x; q < chunks; q += gridDim.x) {
        long long begin;
        const GradTensor& t = find_tensor(g, chunks - 1 - q, begin);
        if (one && t.in_place) continue;
        with_type(t.type, [&](auto type) {
            using T = decltype(type);
            constexpr int N = Word16<T>::N;
            const T* base = static_cast<const T*>(t.grad) - t.lead;
            with_type(t.out_type, [&](auto out_type) {
                using O = decltype(out_type);
                O* out = static_cast<O*>(t.out) - t.lead;
                walk_chunk<N>(t, reinterpret_cast<const uint4*>(base), begin,
                    [&](const uint4& v, long long w) {
                        float f[N];
                        Word16<T>::load(v, f);
#pragma unroll
                        for (int i = 0; i < N; ++i) f[i] = times(f[i], O{});
                        if constexpr (sizeof(O) <= sizeof(T) && N < Word16<O>::N) {      // half a word of a narrower type
                            if (t.out_words) { *reinterpret_cast<uint2*>(out + w * N) = make_uint2(pack16<O>(f[0], f[1]), pack16<O>(f[2], f[3])); return; }
                        } else {
                            if (t.out_words) {
#pragma unroll
                                for (int i = 0; i < N; i += Word16<O>::N) *reinterpret_cast<uint4*>(out + w * N + i) = Word16<O>::store(f + i);
                                return;
                            }
                        }
#pragma unroll
                        for (int i = 0; i < N; ++i) put_element(out + w * N + i, f[i]);
                    },
                    [&](long long e) { put_element(out + e, times(element(base + e), O{})); });
            });
        });
    }
}

int launched(const char* what)
{
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? ALPHA_OK : fail(ALPHA_E_CUDA, "%s launch failed: %s", what, cudaGetErrorString(e));
}
int type_size(int dtype) { return dtype == ALPHA_F32 ? 4 : 2; }

int check_grads(const char* what, int n, const AlphaGrad* grads, const float* norm, bool scale)
{
    if (n < 0 || (n && !grads)) return fail(ALPHA_E_ARG, "%s: no tensors", what);
    if (!norm || (reinterpret_cast<uintptr_t>(norm) & 3)) return fail(ALPHA_E_ARG, "%s: norm must be a device pointer to a float", what);
    struct Range { uintptr_t from, to; bool write; };
    std::vector<Range> ranges;
    try {
        ranges.reserve(2 * static_cast<size_t>(n) + 1);
    } catch (const std::exception&) {
        return fail(ALPHA_E_NOSCRATCH, "%s: no host memory to check %d tensors", what, n);
    }
    auto add = [&](const void* p, size_t bytes, bool write) { ranges.push_back(Range{reinterpret_cast<uintptr_t>(p), reinterpret_cast<uintptr_t>(p) + bytes, write}); };
    add(norm, sizeof(float), true);
    for (int i = 0; i < n; ++i) {
        const AlphaGrad& g = grads[i];
        auto known = [](int t) { return t == ALPHA_F32 || t == ALPHA_BF16 || t == ALPHA_F16; };
        if (!known(g.dtype) || (scale && !known(g.out_dtype))) return fail(ALPHA_E_ARG, "%s: unknown element type of tensor %d", what, i);
        if (g.count < 0 || g.count >= 1LL << 43) return fail(ALPHA_E_ARG, "%s: tensor %d has %lld elements", what, i, static_cast<long long>(g.count));
        if (g.count == 0) continue;
        if (!g.grad || (scale && !g.out)) return fail(ALPHA_E_ARG, "%s: null pointer of tensor %d", what, i);
        const size_t size = type_size(g.dtype), out_size = type_size(g.out_dtype);
        if (reinterpret_cast<uintptr_t>(g.grad) % size || (scale && reinterpret_cast<uintptr_t>(g.out) % out_size))
            return fail(ALPHA_E_ARG, "%s: tensor %d is not aligned to its elements", what, i);
        const bool in_place = scale && g.grad == g.out && g.dtype == g.out_dtype;
        add(g.grad, g.count * size, in_place);
        if (scale && !in_place) add(g.out, g.count * out_size, true);
    }
    std::sort(ranges.begin(), ranges.end(), [](const Range& a, const Range& b) { return a.from < b.from; });
    uintptr_t read = 0, written = 0;          // ends of the ranges so far
    for (const Range& r : ranges) {
        if (r.from < written || (r.write && r.from < read)) return fail(ALPHA_E_ARG, "%s: an output overlaps another tensor", what);
        (r.write ? written : read) = std::max(r.write ? written : read, r.to);
    }
    return ALPHA_OK;
}

// Tables of up to kGradTensors tensors with elements; f(table, chunks) for each.
template <class F> int for_tables(int n, const AlphaGrad* grads, bool scale, F&& f)
{
    GradTable g;
    g.n = 0;
    long long chunks = 0;
    for (int i = 0; i <= n; ++i) {
        long long more = 0;
        int lead = 0;
        if (i < n) {
            if (grads[i].count == 0) continue;
            lead = static_cast<int>((reinterpret_cast<uintptr_t>(grads[i].grad) & 15) / type_size(grads[i].dtype));
            more = (grads[i].count + lead + kGradChunk - 1) / kGradChunk;
        }
        if (g.n && (i == n || g.n == kGradTensors || chunks + more > 2147483647LL)) {
            g.first[g.n] = static_cast<unsigned>(chunks);
            const int rc = f(g, chunks);
            if (rc) return rc;
            g.n = 0;
            chunks = 0;
        }
        if (i == n) break;
        GradTensor& t = g.t[g.n];
        t.grad = grads[i].grad; t.count = grads[i].count; t.lead = lead; t.type = static_cast<unsigned char>(grads[i].dtype);
        t.out = nullptr; t.out_type = t.type; t.in_place = t.out_words = 0;
        if (scale) {
            t.out = grads[i].out; t.out_type = static_cast<unsigned char>(grads[i].out_dtype);
            t.in_place = t.out == t.grad && t.out_type == t.type;
            // words of 4 or 8 elements: 8 bytes of a 16-bit output of fp32, else 16 or 32
            const uintptr_t start = reinterpret_cast<uintptr_t>(t.out) - static_cast<uintptr_t>(lead) * type_size(grads[i].out_dtype);
            t.out_words = start % (type_size(grads[i].dtype) > type_size(grads[i].out_dtype) ? 8 : 16) == 0;
        }
        g.first[g.n++] = static_cast<unsigned>(chunks);
        chunks += more;
    }
    return ALPHA_OK;
}

int run(const char* what, int n, const AlphaGrad* grads, bool scale, double max_norm, float* norm, cudaStream_t stream)
{
    int rc = check_grads(what, n, grads, norm, scale);
    if (!rc) rc = call_begin(stream);
    int sms = 0;
    if (!rc) rc = device_sms(&sms);
    if (rc) return rc;
    const int most = 6 * sms;
    auto ctas = [&](long long chunks) { return static_cast<unsigned>(chunks < most ? chunks : most); };
    size_t parts = 0;
    for_tables(n, grads, scale, [&](const GradTable&, long long chunks) { parts += ctas(chunks); return ALPHA_OK; });
    void* ws = nullptr;
    rc = call_scratch(stream, (parts ? parts : 1) * sizeof(double), &ws);
    if (rc || dry_run()) return rc;
    double* part = static_cast<double*>(ws);
    size_t at = 0;
    rc = for_tables(n, grads, scale, [&](const GradTable& g, long long chunks) {
        launch_after(grad_squares_kernel, ctas(chunks), kGradThreads, 0, stream, g, part + at);
        note_launch("grad_norm");
        at += ctas(chunks);
        return launched("grad_squares_kernel");
    });
    if (rc) return rc;
    if (!scale || !parts) {
        launch_after(grad_norm_kernel, 1, kGradThreads, 0, stream, part, static_cast<int>(parts), norm);
        note_launch("grad_norm");
        return launched("grad_norm_kernel");
    }
    float* out = norm;
    return for_tables(n, grads, scale, [&](const GradTable& g, long long chunks) {
        launch_after(grad_scale_kernel, ctas(chunks), kGradThreads, 0, stream, g, part, static_cast<int>(parts), max_norm, out);
        note_launch("grad_norm");
        out = nullptr;
        return launched("grad_scale_kernel");
    });
}

}  // namespace
}  // namespace alpha

using namespace alpha;

extern "C" {

int alpha_grad_norm(int n, const AlphaGrad* grads, float* norm, alpha_stream_t stream)
{
    OpRange range("alpha_grad_norm");
    return run("grad_norm", n, grads, false, 0.0, norm, static_cast<cudaStream_t>(stream));
}

int alpha_clip_grad_norm(int n, const AlphaGrad* grads, double max_norm, float* norm, alpha_stream_t stream)
{
    OpRange range("alpha_clip_grad_norm");
    if (!(max_norm >= 0.0)) return fail(ALPHA_E_ARG, "clip_grad_norm: max_norm must not be negative or NaN");
    return run("clip_grad_norm", n, grads, true, max_norm, norm, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
