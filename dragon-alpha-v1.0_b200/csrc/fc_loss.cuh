// The passes over rows that surround the products of a softmax cross entropy.
#pragma once
#include "dependent_launch.cuh"
#include "fc_act.cuh"

namespace alpha {

// A row's label, or -1 where it does not count.
__device__ __forceinline__ int label_of(const void* label, int bytes, int row, int classes)
{
    const long long l = bytes == 8 ? static_cast<const long long*>(label)[row] : static_cast<const int*>(label)[row];
    return l >= 0 && l < classes ? static_cast<int>(l) : -1;
}

// The larger of two maxima, and the sum of exponentials about it (-Inf: nothing yet, or nothing but -Inf).
__device__ __forceinline__ void join_stats(float& m, float& s, float m2, float s2)
{
    const float most = fmaxf(m, m2), about = most > -__int_as_float(0x7f800000) ? most : 0.f;
    s = s * expf(m - about) + s2 * expf(m2 - about);
    m = most;
}

// lse and loss of rows from the parts of the tiles' columns, [slots][rows].  A CTA has `across` rows (a power of two up to 32, neighbouring lanes) and shares their
// slots among its other threads.
constexpr int kJoinThreads = 1024;
__global__ void __launch_bounds__(kJoinThreads) loss_join_kernel(const float2* __restrict__ part, int slots, int rows, int across, const void* label, int label_bytes, int classes,
                                                                  const float* __restrict__ at_label, float* loss, float* lse)
{
    __shared__ float2 shared[kJoinThreads];
    grid_dependency_wait();
    grid_dependency_trigger();
    const int x = threadIdx.x % across, y = threadIdx.x / across, ways = kJoinThreads / across, row = blockIdx.x * across + x;
    float m = -__int_as_float(0x7f800000), s = 0.f;
    if (row < rows) {
        const float2* at = part + row;
        int i = y;
        for (; i + 7 * ways < slots; i += 8 * ways) {
            float2 v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = at[static_cast<size_t>(i + j * ways) * rows];
            // (about one maximum, so that no exponential waits for another)
            float most = m;
#pragma unroll
            for (int j = 0; j < 8; ++j) most = fmaxf(most, v[j].x);
            const float about = most > -__int_as_float(0x7f800000) ? most : 0.f;
            s *= expf(m - about);
#pragma unroll
            for (int j = 0; j < 8; ++j) s = fmaf(v[j].y, expf(v[j].x - about), s);
            m = most;
        }
        for (; i < slots; i += ways) {
            const float2 v = at[static_cast<size_t>(i) * rows];
            join_stats(m, s, v.x, v.y);
        }
    }
    shared[threadIdx.x] = make_float2(m, s);
    // (halves of the threads, in a fixed order)
    for (int d = kJoinThreads / 2; d >= across; d >>= 1) {
        __syncthreads();
        if (static_cast<int>(threadIdx.x) < d) {
            const float2 v = shared[threadIdx.x + d];
            join_stats(m, s, v.x, v.y);
            shared[threadIdx.x] = make_float2(m, s);
        }
    }
    if (static_cast<int>(threadIdx.x) >= across || row >= rows) return;
    const float l = m + logf(s);
    if (lse) lse[row] = l;
    if (loss) loss[row] = label_of(label, label_bytes, row, classes) >= 0 ? l - at_label[row] : 0.f;
}

// scale[0]: the power of two that brings the largest of |grad|, of the rows that count, to 2^14 .. 2^15 (1 where it is 0, Inf or NaN), scale[1]: its inverse.
__global__ void __launch_bounds__(1024) loss_scale_kernel(const float* __restrict__ grad, int n, const void* label, int label_bytes, int classes, float* scale)
{
    __shared__ float shared[32];
    grid_dependency_wait();
    grid_dependency_trigger();
    float m = 0.f;
    for (int i = threadIdx.x; i < n; i += 1024)
        if (label_of(label, label_bytes, i, classes) >= 0) m = fmaxf(m, fabsf(grad[i]));
#pragma unroll
    for (int d = 16; d; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
    if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = m;
    __syncthreads();
    if (threadIdx.x) return;
    for (int w = 1; w < 32; ++w) m = fmaxf(m, shared[w]);
    const int e = static_cast<int>(__float_as_uint(m) >> 23);         // (of denormals 0, of Inf 255)
    int k = m > 0.f && e < 255 ? 127 + 14 - e : 0;
    k = k > 126 ? 126 : k < -126 ? -126 : k;
    scale[0] = __uint_as_float(static_cast<uint32_t>(127 + k) << 23);
    scale[1] = __uint_as_float(static_cast<uint32_t>(127 - k) << 23);
}

// Column sums of a matrix, partial sums of every gridDim.y-th block of 8 rows: a thread has a word of 16 bytes; then of the partial sums.
template <class T>
__global__ void __launch_bounds__(256) loss_columns_kernel(const T* __restrict__ a, int rows, int pitch, float* part)
{
    constexpr int N = Word16<T>::N;
    __shared__ float red[8][32 * N + 1];
    grid_dependency_wait();
    grid_dependency_trigger();
    const int x = threadIdx.x & 31, y = threadIdx.x >> 5, words = pitch / N, word = blockIdx.x * 32 + x;
    float s[N];
#pragma unroll
    for (int j = 0; j < N; ++j) s[j] = 0.f;
    if (word < words)
#pragma unroll 4
        for (long long r = blockIdx.y * 8 + y; r < rows; r += gridDim.y * 8) {
            float f[N];
            Word16<T>::load(__ldg(reinterpret_cast<const uint4*>(a + r * pitch) + word), f);
#pragma unroll
            for (int j = 0; j < N; ++j) s[j] += f[j];
        }
#pragma unroll
    for (int j = 0; j < N; ++j) red[y][x * N + j] = s[j];
    __syncthreads();
    for (int c = threadIdx.x; c < 32 * N; c += 256) {
        float sum = 0.f;
#pragma unroll
        for (int r = 0; r < 8; ++r) sum += red[r][c];
        const int col = blockIdx.x * 32 * N + c;
        if (col < pitch) part[static_cast<size_t>(blockIdx.y) * pitch + col] = sum;
    }
}
template <class T>
__global__ void __launch_bounds__(256) loss_bias_kernel(const float* __restrict__ part, int parts, int pitch, const float* by, float factor, T* out)
{
    grid_dependency_wait();
    grid_dependency_trigger();
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c >= pitch) return;
    float s = 0.f;
#pragma unroll 8
    for (int i = 0; i < parts; ++i) s += part[static_cast<size_t>(i) * pitch + c];
    out[c] = static_cast<T>(s * ((by ? *by : 1.f) * factor));
}

// The same of few rows at once: a warp's 32 columns, 32 warps.
template <class T>
__global__ void __launch_bounds__(1024) loss_few_columns_kernel(const T* __restrict__ a, int rows, int pitch, const float* by, float factor, T* out)
{
    __shared__ float red[32][33];
    grid_dependency_wait();
    grid_dependency_trigger();
    const int x = threadIdx.x & 31, y = threadIdx.x >> 5, c = blockIdx.x * 32 + x;
    float s = 0.f;
    if (c < pitch)
#pragma unroll 8
        for (int r = y; r < rows; r += 32) s += static_cast<float>(a[static_cast<size_t>(r) * pitch + c]);
    red[y][x] = s;
    __syncthreads();
    if (y || c >= pitch) return;
#pragma unroll
    for (int r = 1; r < 32; ++r) s += red[r][x];
    out[c] = static_cast<T>(s * ((by ? *by : 1.f) * factor));
}

// ---- fp32: logits of a piece of the classes lie in memory ---------------------------------------------------------

constexpr int kRowThreads = 256;
__device__ __forceinline__ float cta_most(float x, float* shared)
{
#pragma unroll
    for (int d = 16; d; d >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
    __syncthreads();
    if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = x;
    __syncthreads();
    x = shared[0];
#pragma unroll
    for (int w = 1; w < kRowThreads / 32; ++w) x = fmaxf(x, shared[w]);
    return x;
}
__device__ __forceinline__ float cta_total(float x, float* shared)
{
#pragma unroll
    for (int d = 16; d; d >>= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = x;
    __syncthreads();
    x = 0.f;
#pragma unroll
    for (int w = 0; w < kRowThreads / 32; ++w) x += shared[w];
    return x;
}
// gridDim.y CTAs to a row: the largest logit of a CTA's share of the piece, then the sum about it, a slot of the row's parts, and from the first the label's logit if it lies in the piece.
// Of a share that is all the classes (part NULL) lse and loss.
__global__ void __launch_bounds__(kRowThreads) loss_rows_kernel(const float* __restrict__ z, int pitch, int cols, int base, int classes, int rows, const void* label, int label_bytes,
                                                                float2* part, float* at_label, float* loss, float* lse)
{
    __shared__ float shared[kRowThreads / 32];
    grid_dependency_wait();
    grid_dependency_trigger();
    const int row = blockIdx.x, first = blockIdx.y * kRowThreads + threadIdx.x, step = gridDim.y * kRowThreads;
    const float* at = z + static_cast<size_t>(row) * pitch;
    float m = -__int_as_float(0x7f800000);
    for (int c = first; c < cols; c += step) m = fmaxf(m, at[c]);
    m = cta_most(m, shared);
    const float about = m > -__int_as_float(0x7f800000) ? m : 0.f;
    float s = 0.f;
    for (int c = first; c < cols; c += step) s += expf(at[c] - about);
    s = cta_total(s, shared);
    if (threadIdx.x) return;
    const int l = label_of(label, label_bytes, row, classes) - base;
    if (!part) {
        const float log_sum = m + logf(s);
        if (lse) lse[row] = log_sum;
        if (loss) loss[row] = l >= 0 ? log_sum - at[l] : 0.f;
        return;
    }
    part[static_cast<size_t>(blockIdx.y) * rows + row] = make_float2(m, s);
    if (l >= 0 && l < cols && blockIdx.y == 0) at_label[row] = at[l];
}
// Logits become their gradients, in place; the padding of a row 0.  Logits that were formed in parts are added first, with the bias.
__global__ void __launch_bounds__(kRowThreads) loss_delta_kernel(float* z, const float* __restrict__ part, int parts, const float* __restrict__ bias, int rows, int pitch, int cols, int base, int classes, const void* label, int label_bytes, const float* __restrict__ lse,
                                                                 const float* __restrict__ grad, int grad_step)
{
    grid_dependency_wait();
    grid_dependency_trigger();
    const int row = blockIdx.x, l = label_of(label, label_bytes, row, classes);
    const float log_sum = lse[row], g = grad[static_cast<size_t>(row) * grad_step];
    float* at = z + static_cast<size_t>(row) * pitch;
    for (int c = blockIdx.y * kRowThreads + threadIdx.x; c < pitch; c += gridDim.y * kRowThreads) {
        float logit = part ? 0.f : at[c];
        if (part)
            for (int i = 0; i < parts; ++i) logit += part[(static_cast<size_t>(i) * rows + row) * pitch + c];
        if (bias) logit += bias[c];
        const float p = expf(logit - log_sum);
        at[c] = l >= 0 && c < cols ? g * (c == l - base ? p - 1.f : p) : 0.f;
    }
}
// The parts of deltaX's reduction, four outputs a thread: added in order to what the classes before gave, and rounded with the last.
template <class T>
__global__ void __launch_bounds__(256) loss_parts_kernel(const float4* __restrict__ part, int parts, size_t words, float4* total, int first, int last, const float* by, float factor, uint2* out)
{
    grid_dependency_wait();
    grid_dependency_trigger();
    const float scale = (by ? *by : 1.f) * factor;
    for (size_t i = static_cast<size_t>(blockIdx.x) * 256 + threadIdx.x; i < words; i += static_cast<size_t>(gridDim.x) * 256) {
        float4 s = first ? make_float4(0.f, 0.f, 0.f, 0.f) : total[i];
#pragma unroll 4
        for (int r = 0; r < parts; ++r) {
            const float4 v = __ldcs(part + r * words + i);
            s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
        }
        if (last) out[i] = make_uint2(pack16<T>(s.x * scale, s.y * scale), pack16<T>(s.z * scale, s.w * scale));
        else total[i] = s;
    }
}
__global__ void __launch_bounds__(256) loss_add_kernel(float4* to, const float4* __restrict__ more, size_t words)
{
    grid_dependency_wait();
    grid_dependency_trigger();
    for (size_t i = static_cast<size_t>(blockIdx.x) * 256 + threadIdx.x; i < words; i += static_cast<size_t>(gridDim.x) * 256) {
        const float4 a = to[i], b = more[i];
        to[i] = make_float4(a.x + b.x, a.y + b.y, a.z + b.z, a.w + b.w);
    }
}

}  // namespace alpha
