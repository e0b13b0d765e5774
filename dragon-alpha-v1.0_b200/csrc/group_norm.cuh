// Group normalisation of channels-last tensors with the activation that follows it, and its gradients.
//
//   xh = (x - mean) rstd,  z = xh gamma + beta,  y = act(z)        mean, rstd over the positions and the C / G channels of (sample, group)
//   dz = dy act'(z),  deltaGamma_c = sum dz xh,  deltaBeta_c = sum dz
//   deltaX = rstd (dz gamma - s1 - xh s2)                          s1, s2: means of dz gamma and dz gamma xh over (sample, group)
//
// Bound by HBM: the tensors are to be read once although nothing can be written before the last element of a group is known.
//
// Resident: a sample is cut into slabs of whole groups whose words of 16 bytes lie side by side; a CTA, or a cluster of up to eight that share the positions, brings its part of
// a slab into shared memory by asynchronous copies, forms the sums there, adds those of its cluster, and writes the outputs from shared memory: each
// tensor crosses HBM once.  Two or more CTAs to an SM, so that one copies while another computes or stores.  A thread keeps one word of the row (its channels) and walks the
// positions, so that the words of neighbouring threads are neighbours in memory and a thread reads only what it copied itself.
//
// Streamed: what does not fit (and widths that are no multiple of 16 bytes, a thread to an element): partial sums of runs of positions, their sum, and a second pass over
// the tensors, from their end, so that it begins with what the first left in L2.
//
// Variances come from differences to a mean: within a CTA's part (or eight positions of a thread), and parts are joined by their means; nothing is a
// difference of large sums.  Sums are fp32, joined in a fixed order.
#pragma once
#include "dependent_launch.cuh"
#include "fc_act.cuh"
#include "sm100_ptx.cuh"

namespace alpha {

constexpr int kNormThreads = 256;

struct Norm {
    const void *X, *dY;
    void* out;                      // Y, or deltaX
    const void *gamma, *beta;       // (or NULL: 1 and 0)
    int affine_f32;                 // gamma and beta are floats
    float *mean, *rstd;             // [N][G]: written by a forward call (may be NULL), read by a backward one
    float2* sums;                   // [N][C] sums of dz and dz xh
    int N, R, C, G, D;
    float eps, k;
    int act;
    // resident: words of a slab, slabs of a row, CTAs that share a slab, positions of each, rows of threads
    int words, slabs, cluster, part, rows;
    // streamed: column blocks of `words` words, runs of `part` positions
    int blocks, runs;
    float2* partial;                // [N][runs][C] mean and sum of squared differences, or sums of dz and dz xh
    float2* group;                  // [N][G] mean and rstd, or s1 and s2
};

// A word of V elements as floats and back.
template <class T, int V> struct NormWord {
    using Raw = uint4;
    static __device__ void load(const Raw& r, float* f) { Word16<T>::load(r, f); }
    static __device__ Raw store(const float* f) { return Word16<T>::store(f); }
};
template <class T> struct NormWord<T, 1> {
    using Raw = T;
    static __device__ void load(const Raw& r, float* f) { f[0] = static_cast<float>(r); }
    static __device__ Raw store(const float* f) { return static_cast<T>(f[0]); }
};

template <class T> __device__ __forceinline__ float affine_at(const void* p, int c, int f32, float none)
{
    return !p ? none : f32 ? static_cast<const float*>(p)[c] : static_cast<float>(static_cast<const T*>(p)[c]);
}

__device__ __forceinline__ void copy_async16(uint32_t to, const void* from) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory"); }
__device__ __forceinline__ void copies_done() { asm volatile("cp.async.wait_all;" ::: "memory"); }
__device__ __forceinline__ float warp_sum(float x)
{
#pragma unroll
    for (int d = 16; d; d >>= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
    return x;
}

// Sums over (group): a thread's V sums of its channels lie in red[j][thread]; warp w adds those of groups w, w + 8, ...  f(group, sum) in every lane.
template <int V, class F> __device__ __forceinline__ void group_sums(const float* red, const Norm& p, int groups, F&& f)
{
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, count = p.rows * p.D;
    for (int g = warp; g < groups; g += kNormThreads / 32) {
        float s = 0.f;
        for (int i = lane; i < count; i += 32) {
            const int row = i / p.D, c = g * p.D + i - row * p.D;
            s += red[(c % V) * kNormThreads + row * p.words + c / V];
        }
        f(g, warp_sum(s));
    }
}

// Shared memory of a resident CTA: its words of X (and deltaY), V sums (backward: twice) of each thread, and the groups'.
__host__ __device__ inline size_t norm_smem(bool back, int V, int part, int words, int groups)
{
    return static_cast<size_t>(part) * words * 16 * (back ? 2 : 1) + static_cast<size_t>(V) * kNormThreads * 4 * (back ? 2 : 1) + static_cast<size_t>(groups) * 16;
}

template <class T, bool BACK>
__global__ void __launch_bounds__(kNormThreads, 2) norm_resident_kernel(const __grid_constant__ Norm p)
{
    constexpr int V = Word16<T>::N;
    extern __shared__ __align__(128) uint8_t smem[];
    const int cl = p.cluster, rank = cl > 1 ? static_cast<int>(cluster_ctarank()) : 0, item = blockIdx.x / cl, n = item / p.slabs, slab = item - n * p.slabs;
    const int r0 = rank * p.part, mine = min(p.part, p.R - r0);             // (positive: no part is empty)
    const int ty = threadIdx.x / p.words, tx = threadIdx.x - ty * p.words, c0 = slab * p.words * V, groups = p.words * V / p.D, g0 = c0 / p.D;
    const bool busy = ty < p.rows;
    uint4* xs = reinterpret_cast<uint4*>(smem);
    uint4* ys = xs + static_cast<size_t>(p.part) * p.words;
    float* red = reinterpret_cast<float*>(ys + (BACK ? static_cast<size_t>(p.part) * p.words : 0));
    float2* own = reinterpret_cast<float2*>(red + V * kNormThreads * (BACK ? 2 : 1));      // this CTA's sums of each group
    float2* all = own + groups;                                                            // the cluster's
    const size_t from = (static_cast<size_t>(n) * p.R + r0) * p.C + c0 + tx * V;
    grid_dependency_wait();
    grid_dependency_trigger();
    if (busy) {
        const T *x = static_cast<const T*>(p.X) + from, *y = BACK ? static_cast<const T*>(p.dY) + from : nullptr;
        const uint32_t to = smem_u32(xs), to_y = smem_u32(ys);
        for (int r = ty; r < mine; r += p.rows) {
            copy_async16(to + (r * p.words + tx) * 16, x + static_cast<size_t>(r) * p.C);
            if (BACK) copy_async16(to_y + (r * p.words + tx) * 16, y + static_cast<size_t>(r) * p.C);
        }
    }
    float gamma[V], beta[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        gamma[j] = affine_at<T>(p.gamma, c0 + tx * V + j, p.affine_f32, 1.f);
        beta[j] = affine_at<T>(p.beta, c0 + tx * V + j, p.affine_f32, 0.f);
    }
    float mean[V], rstd[V];
    if (BACK) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const size_t g = static_cast<size_t>(n) * p.G + (c0 + tx * V + j) / p.D;
            mean[j] = busy ? p.mean[g] : 0.f;
            rstd[j] = busy ? p.rstd[g] : 0.f;
        }
    }
    copies_done();
    const float count = static_cast<float>(p.R) * static_cast<float>(p.D);
    T* out = static_cast<T*>(p.out) + from;
    if constexpr (!BACK) {
        const float own_count = static_cast<float>(mine) * static_cast<float>(p.D);
        float s[V];
#pragma unroll
        for (int j = 0; j < V; ++j) s[j] = 0.f;
        if (busy)
            for (int r = ty; r < mine; r += p.rows) {
                float f[V];
                Word16<T>::load(xs[r * p.words + tx], f);
#pragma unroll
                for (int j = 0; j < V; ++j) s[j] += f[j];
            }
#pragma unroll
        for (int j = 0; j < V; ++j) red[j * kNormThreads + threadIdx.x] = s[j];
        __syncthreads();
        group_sums<V>(red, p, groups, [&](int g, float sum) { if ((threadIdx.x & 31) == 0) own[g].x = sum / own_count; });
        __syncthreads();
        if (busy) {
#pragma unroll
            for (int j = 0; j < V; ++j) { mean[j] = own[(tx * V + j) / p.D].x; s[j] = 0.f; }
            for (int r = ty; r < mine; r += p.rows) {
                float f[V];
                Word16<T>::load(xs[r * p.words + tx], f);
#pragma unroll
                for (int j = 0; j < V; ++j) { const float d = f[j] - mean[j]; s[j] = fmaf(d, d, s[j]); }
            }
#pragma unroll
            for (int j = 0; j < V; ++j) red[j * kNormThreads + threadIdx.x] = s[j];
        }
        __syncthreads();
        group_sums<V>(red, p, groups, [&](int g, float sum) { if ((threadIdx.x & 31) == 0) own[g].y = sum; });
        if (cl > 1) cluster_sync_all();
        else __syncthreads();
        // mean and rstd of a group from its parts
        for (int g = threadIdx.x; g < groups; g += kNormThreads) {
            float m = own[g].x, squares = own[g].y;
            if (cl > 1) {
                const uint32_t at = smem_u32(own + g);
                float sum = 0.f;
                for (int q = 0; q < cl; ++q) sum = fmaf(ld_shared_cluster(mapa_u32(at, q)), static_cast<float>(min(p.part, p.R - q * p.part)), sum);
                m = sum / static_cast<float>(p.R);
                squares = 0.f;
                for (int q = 0; q < cl; ++q) {
                    const uint32_t peer = mapa_u32(at, q);
                    const float d = ld_shared_cluster(peer) - m;
                    squares += ld_shared_cluster(peer + 4) + d * d * (static_cast<float>(min(p.part, p.R - q * p.part)) * static_cast<float>(p.D));
                }
            }
            const float r = 1.f / sqrtf(squares / count + p.eps);
            all[g] = make_float2(m, r);
            if (rank == 0 && p.mean) {
                p.mean[static_cast<size_t>(n) * p.G + g0 + g] = m;
                p.rstd[static_cast<size_t>(n) * p.G + g0 + g] = r;
            }
        }
        if (cl > 1) cluster_sync_all();          // (and no CTA leaves while another may still read its sums)
        else __syncthreads();
        if (!busy) return;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const float2 m = all[(tx * V + j) / p.D];
            mean[j] = m.x;
            gamma[j] *= m.y;
        }
        with_act(p.act, [&](auto a) {
            for (int r = ty; r < mine; r += p.rows) {
                float f[V];
                Word16<T>::load(xs[r * p.words + tx], f);
#pragma unroll
                for (int j = 0; j < V; ++j) f[j] = act_value<decltype(a)::value, Word16<T>::kFast>(fmaf(f[j] - mean[j], gamma[j], beta[j]), p.k);
                *reinterpret_cast<uint4*>(out + static_cast<size_t>(r) * p.C) = Word16<T>::store(f);
            }
        });
    } else {
        float a[V], b[V];
#pragma unroll
        for (int j = 0; j < V; ++j) { a[j] = b[j] = 0.f; }
        if (busy)
            with_act(p.act, [&](auto act) {
                for (int r = ty; r < mine; r += p.rows) {
                    float x[V], y[V];
                    Word16<T>::load(xs[r * p.words + tx], x);
                    Word16<T>::load(ys[r * p.words + tx], y);
#pragma unroll
                    for (int j = 0; j < V; ++j) {
                        const float xh = (x[j] - mean[j]) * rstd[j];
                        float value, slope;
                        act_both<decltype(act)::value, Word16<T>::kFast>(fmaf(xh, gamma[j], beta[j]), p.k, value, slope);
                        const float dz = y[j] * slope;
                        a[j] += dz;
                        b[j] = fmaf(dz, xh, b[j]);
                    }
                }
            });
#pragma unroll
        for (int j = 0; j < V; ++j) {
            red[j * kNormThreads + threadIdx.x] = a[j];
            red[(V + j) * kNormThreads + threadIdx.x] = b[j];
        }
        __syncthreads();
        // channels: the threads' sums into the first row of threads
        const int wide = p.words * V;
        for (int c = threadIdx.x; c < 2 * wide; c += kNormThreads) {
            const int second = c >= wide, ch = c - second * wide;
            float* at = red + (ch % V + second * V) * kNormThreads + ch / V;
            float s = 0.f;
            for (int r = 0; r < p.rows; ++r) s += at[r * p.words];
            at[0] = s;
        }
        if (cl > 1) cluster_sync_all();
        else __syncthreads();
        // over the cluster: every CTA adds all parts in the same order
        float keep[2 * V];
#pragma unroll
        for (int j = 0; j < 2 * V; ++j) keep[j] = 0.f;
        if (threadIdx.x < p.words) {
#pragma unroll
            for (int j = 0; j < 2 * V; ++j) {
                if (cl == 1) { keep[j] = red[j * kNormThreads + threadIdx.x]; continue; }
                const uint32_t at = smem_u32(red + j * kNormThreads + threadIdx.x);
                for (int q = 0; q < cl; ++q) keep[j] += ld_shared_cluster(mapa_u32(at, q));
            }
        }
        if (cl > 1) cluster_sync_all();          // (all parts have been read)
        if (threadIdx.x < p.words) {
            // channels' sums, weighted by gamma, for the groups'
#pragma unroll
            for (int j = 0; j < V; ++j) {
                if (rank == 0) p.sums[static_cast<size_t>(n) * p.C + c0 + tx * V + j] = make_float2(keep[j], keep[V + j]);
                red[j * kNormThreads + threadIdx.x] = keep[j] * gamma[j];
                red[(V + j) * kNormThreads + threadIdx.x] = keep[V + j] * gamma[j];
            }
        }
        __syncthreads();
        {
            const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
            for (int g = warp; g < groups; g += kNormThreads / 32) {
                float s1 = 0.f, s2 = 0.f;
                for (int i = lane; i < p.D; i += 32) {
                    const int c = g * p.D + i;
                    s1 += red[(c % V) * kNormThreads + c / V];
                    s2 += red[(V + c % V) * kNormThreads + c / V];
                }
                s1 = warp_sum(s1);
                s2 = warp_sum(s2);
                if (lane == 0) all[g] = make_float2(s1 / count, s2 / count);
            }
        }
        __syncthreads();
        if (!busy) return;
        float s1[V], s2[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const float2 s = all[(tx * V + j) / p.D];
            s1[j] = s.x; s2[j] = s.y;
        }
        with_act(p.act, [&](auto act) {
            for (int r = ty; r < mine; r += p.rows) {
                float x[V], y[V];
                Word16<T>::load(xs[r * p.words + tx], x);
                Word16<T>::load(ys[r * p.words + tx], y);
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float xh = (x[j] - mean[j]) * rstd[j];
                    float value, slope;
                    act_both<decltype(act)::value, Word16<T>::kFast>(fmaf(xh, gamma[j], beta[j]), p.k, value, slope);
                    x[j] = rstd[j] * (fmaf(y[j] * slope, gamma[j], -s1[j]) - xh * s2[j]);
                }
                *reinterpret_cast<uint4*>(out + static_cast<size_t>(r) * p.C) = Word16<T>::store(x);
            }
        });
    }
}

// ---- streamed ---------------------------------------------------------------------------------------------------

// Where a CTA of the streamed passes is: a block of columns, a run of positions, a sample.
struct NormAt { int n, run, r0, count, ty, word; bool busy; size_t from; };
template <int V> __device__ __forceinline__ NormAt norm_at(const Norm& p, unsigned block)
{
    NormAt a;
    const unsigned col = block % p.blocks, rest = block / p.blocks;
    a.run = rest % p.runs; a.n = rest / p.runs;
    a.r0 = a.run * p.part;
    a.count = min(p.part, p.R - a.r0);
    a.ty = threadIdx.x / p.words;
    a.word = col * p.words + threadIdx.x - a.ty * p.words;
    a.busy = a.ty < p.rows && a.word < p.C / V;
    a.from = (static_cast<size_t>(a.n) * p.R + a.r0) * p.C + static_cast<size_t>(a.word) * V;
    return a;
}
// Mean and squared differences of a run, or its sums of dz and dz xh, for every channel.
template <class T, int V, bool BACK>
__global__ void __launch_bounds__(kNormThreads) norm_sums_kernel(const __grid_constant__ Norm p)
{
    using W = NormWord<T, V>;
    using Raw = typename W::Raw;
    constexpr int U = V == 1 ? 8 : BACK ? 4 : 8;
    __shared__ float red[2 * V * kNormThreads];
    grid_dependency_wait();
    grid_dependency_trigger();
    const NormAt a = norm_at<V>(p, blockIdx.x);
    float s[V], q[V];
#pragma unroll
    for (int j = 0; j < V; ++j) s[j] = q[j] = 0.f;
    if (a.busy) {
        const T *x = static_cast<const T*>(p.X) + a.from, *y = BACK ? static_cast<const T*>(p.dY) + a.from : nullptr;
        const size_t step = static_cast<size_t>(p.rows) * p.C;
        if constexpr (!BACK) {
            float seen = 0.f;                     // s: mean of what has been seen, q: its squared differences
            for (int r = a.ty; r < a.count; r += U * p.rows) {
                Raw raw[U];
                int have = (a.count - r + p.rows - 1) / p.rows;
                if (have > U) have = U;
                const T* at = x + static_cast<size_t>(r) * p.C;
#pragma unroll
                for (int i = 0; i < U; ++i) raw[i] = *reinterpret_cast<const Raw*>(at + (i < have ? i : 0) * step);
                const float each = static_cast<float>(have), total = seen + each, weight = each / total, inverse = 1.f / each;
                float m[V], d2[V];
#pragma unroll
                for (int j = 0; j < V; ++j) m[j] = d2[j] = 0.f;
#pragma unroll
                for (int i = 0; i < U; ++i) {
                    float f[V];
                    W::load(raw[i], f);
#pragma unroll
                    for (int j = 0; j < V; ++j) m[j] += i < have ? f[j] : 0.f;
                }
#pragma unroll
                for (int j = 0; j < V; ++j) m[j] *= inverse;
#pragma unroll
                for (int i = 0; i < U; ++i) {
                    float f[V];
                    W::load(raw[i], f);
#pragma unroll
                    for (int j = 0; j < V; ++j) { const float d = i < have ? f[j] - m[j] : 0.f; d2[j] = fmaf(d, d, d2[j]); }
                }
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float d = m[j] - s[j];
                    s[j] = fmaf(d, weight, s[j]);
                    q[j] += fmaf(d * d, seen * weight, d2[j]);
                }
                seen = total;
            }
        } else {
            float mean[V], rstd[V], gamma[V], beta[V];
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const int c = a.word * V + j;
                const size_t g = static_cast<size_t>(a.n) * p.G + c / p.D;
                mean[j] = p.mean[g]; rstd[j] = p.rstd[g];
                gamma[j] = affine_at<T>(p.gamma, c, p.affine_f32, 1.f);
                beta[j] = affine_at<T>(p.beta, c, p.affine_f32, 0.f);
            }
            with_act(p.act, [&](auto act) {
                for (int r = a.ty; r < a.count; r += U * p.rows) {
                    Raw rx[U], ry[U];
                    const size_t at = static_cast<size_t>(r) * p.C;
#pragma unroll
                    for (int i = 0; i < U; ++i) {
                        const size_t o = at + (r + i * p.rows < a.count ? i : 0) * step;
                        rx[i] = *reinterpret_cast<const Raw*>(x + o);
                        ry[i] = *reinterpret_cast<const Raw*>(y + o);
                    }
#pragma unroll
                    for (int i = 0; i < U; ++i) {
                        if (r + i * p.rows >= a.count) break;
                        float fx[V], fy[V];
                        W::load(rx[i], fx);
                        W::load(ry[i], fy);
#pragma unroll
                        for (int j = 0; j < V; ++j) {
                            const float xh = (fx[j] - mean[j]) * rstd[j];
                            float value, slope;
                            act_both<decltype(act)::value, Word16<T>::kFast>(fmaf(xh, gamma[j], beta[j]), p.k, value, slope);
                            const float dz = fy[j] * slope;
                            s[j] += dz;
                            q[j] = fmaf(dz, xh, q[j]);
                        }
                    }
                }
            });
        }
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
        red[j * kNormThreads + threadIdx.x] = s[j];
        red[(V + j) * kNormThreads + threadIdx.x] = q[j];
    }
    __syncthreads();
    float2* to = p.partial + (static_cast<size_t>(a.n) * p.runs + a.run) * p.C;
    const int first = (a.word - (static_cast<int>(threadIdx.x) - a.ty * p.words)) * V, wide = min(p.words * V, p.C - first);
    const int rows = min(p.rows, a.count);
    for (int c = threadIdx.x; c < wide; c += kNormThreads) {
        const float *ms = red + (c % V) * kNormThreads + c / V, *qs = ms + V * kNormThreads;
        float sum = 0.f, squares = 0.f;
        if constexpr (BACK) {
            for (int r = 0; r < rows; ++r) { sum += ms[r * p.words]; squares += qs[r * p.words]; }
        } else {
            const int each = a.count / p.rows, left = a.count - each * p.rows;
            auto had = [&](int r) { return static_cast<float>(each + (r < left ? 1 : 0)); };
            for (int r = 0; r < rows; ++r) sum = fmaf(ms[r * p.words], had(r), sum);
            sum /= static_cast<float>(a.count);
            for (int r = 0; r < rows; ++r) { const float d = ms[r * p.words] - sum; squares += fmaf(d * d, had(r), qs[r * p.words]); }
        }
        to[first + c] = make_float2(sum, squares);
    }
}

__device__ __forceinline__ float block_sum(float x, float* shared)
{
    x = warp_sum(x);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = x;
    __syncthreads();
    x = 0.f;
#pragma unroll
    for (int w = 0; w < kNormThreads / 32; ++w) x += shared[w];
    return x;
}
// A CTA to each (sample, group): its mean and rstd, or s1 and s2 and the channels' sums, from those of the runs.
template <class T, bool BACK>
__global__ void __launch_bounds__(kNormThreads) norm_join_kernel(const __grid_constant__ Norm p)
{
    __shared__ float shared[kNormThreads / 32];
    grid_dependency_wait();
    grid_dependency_trigger();
    const int n = blockIdx.x / p.G, g = blockIdx.x - n * p.G;
    const float2* from = p.partial + static_cast<size_t>(n) * p.runs * p.C + g * p.D;
    const float count = static_cast<float>(p.R) * static_cast<float>(p.D);
    if constexpr (!BACK) {
        const int entries = p.runs * p.D;
        float sum = 0.f, squares = 0.f;
        for (int i = threadIdx.x; i < entries; i += kNormThreads) {
            const int run = i / p.D;
            sum = fmaf(from[static_cast<size_t>(run) * p.C + i - run * p.D].x, static_cast<float>(min(p.part, p.R - run * p.part)), sum);
        }
        const float mean = block_sum(sum, shared) / count;
        for (int i = threadIdx.x; i < entries; i += kNormThreads) {
            const int run = i / p.D;
            const float2 e = from[static_cast<size_t>(run) * p.C + i - run * p.D];
            const float d = e.x - mean;
            squares += fmaf(d * d, static_cast<float>(min(p.part, p.R - run * p.part)), e.y);
        }
        const float rstd = 1.f / sqrtf(block_sum(squares, shared) / count + p.eps);
        if (threadIdx.x == 0) {
            p.group[blockIdx.x] = make_float2(mean, rstd);
            if (p.mean) { p.mean[blockIdx.x] = mean; p.rstd[blockIdx.x] = rstd; }
        }
    } else {
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
        float s1 = 0.f, s2 = 0.f;
        for (int d = warp; d < p.D; d += kNormThreads / 32) {
            float a = 0.f, b = 0.f;
            for (int run = lane; run < p.runs; run += 32) { const float2 e = from[static_cast<size_t>(run) * p.C + d]; a += e.x; b += e.y; }
            a = warp_sum(a);
            b = warp_sum(b);
            if (lane == 0) {
                const int c = g * p.D + d;
                const float gamma = affine_at<T>(p.gamma, c, p.affine_f32, 1.f);
                p.sums[static_cast<size_t>(n) * p.C + c] = make_float2(a, b);
                s1 = fmaf(a, gamma, s1);
                s2 = fmaf(b, gamma, s2);
            }
        }
        s1 = block_sum(s1, shared);
        s2 = block_sum(s2, shared);
        if (threadIdx.x == 0) p.group[blockIdx.x] = make_float2(s1 / count, s2 / count);
    }
}
// The outputs, from the end of the tensors.
template <class T, int V, bool BACK>
__global__ void __launch_bounds__(kNormThreads) norm_apply_kernel(const __grid_constant__ Norm p)
{
    using W = NormWord<T, V>;
    using Raw = typename W::Raw;
    constexpr int U = 4;
    grid_dependency_wait();
    grid_dependency_trigger();
    const NormAt a = norm_at<V>(p, gridDim.x - 1 - blockIdx.x);
    if (!a.busy) return;
    float mean[V], rstd[V], gamma[V], beta[V], s1[V], s2[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int c = a.word * V + j;
        const size_t g = static_cast<size_t>(a.n) * p.G + c / p.D;
        const float2 two = p.group[g];
        gamma[j] = affine_at<T>(p.gamma, c, p.affine_f32, 1.f);
        beta[j] = affine_at<T>(p.beta, c, p.affine_f32, 0.f);
        if (BACK) { mean[j] = p.mean[g]; rstd[j] = p.rstd[g]; s1[j] = two.x; s2[j] = two.y; }
        else { mean[j] = two.x; gamma[j] *= two.y; }
    }
    const T *x = static_cast<const T*>(p.X) + a.from, *y = BACK ? static_cast<const T*>(p.dY) + a.from : nullptr;
    T* out = static_cast<T*>(p.out) + a.from;
    const size_t step = static_cast<size_t>(p.rows) * p.C;
    with_act(p.act, [&](auto act) {
        for (int r = a.ty; r < a.count; r += U * p.rows) {
            Raw rx[U], ry[U];
            const size_t at = static_cast<size_t>(r) * p.C;
#pragma unroll
            for (int i = 0; i < U; ++i) {
                const size_t o = at + (r + i * p.rows < a.count ? i : 0) * step;
                rx[i] = *reinterpret_cast<const Raw*>(x + o);
                if (BACK) ry[i] = *reinterpret_cast<const Raw*>(y + o);
            }
#pragma unroll
            for (int i = 0; i < U; ++i) {
                if (r + i * p.rows >= a.count) break;
                float f[V], fy[V];
                W::load(rx[i], f);
                if (BACK) W::load(ry[i], fy);
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    if constexpr (BACK) {
                        const float xh = (f[j] - mean[j]) * rstd[j];
                        float value, slope;
                        act_both<decltype(act)::value, Word16<T>::kFast>(fmaf(xh, gamma[j], beta[j]), p.k, value, slope);
                        f[j] = rstd[j] * (fmaf(fy[j] * slope, gamma[j], -s1[j]) - xh * s2[j]);
                    } else {
                        f[j] = act_value<decltype(act)::value, Word16<T>::kFast>(fmaf(f[j] - mean[j], gamma[j], beta[j]), p.k);
                    }
                }
                *reinterpret_cast<Raw*>(out + at + i * step) = W::store(f);
            }
        }
    });
}

// deltaGamma and deltaBeta: the samples' sums of a channel, eight rows of 32 threads.
template <class T>
__global__ void __launch_bounds__(256) norm_affine_kernel(const float2* __restrict__ sums, int N, int C, void* dgamma, void* dbeta, int f32)
{
    __shared__ float2 red[8][33];
    grid_dependency_wait();
    grid_dependency_trigger();
    const int x = threadIdx.x & 31, y = threadIdx.x >> 5, c = blockIdx.x * 32 + x;
    float a = 0.f, b = 0.f;
    if (c < C)
        for (int n = y; n < N; n += 8) { const float2 s = sums[static_cast<size_t>(n) * C + c]; a += s.x; b += s.y; }
    red[y][x] = make_float2(a, b);
    __syncthreads();
    if (y || c >= C) return;
#pragma unroll
    for (int r = 1; r < 8; ++r) { a += red[r][x].x; b += red[r][x].y; }
    if (f32) { static_cast<float*>(dgamma)[c] = b; static_cast<float*>(dbeta)[c] = a; }
    else { static_cast<T*>(dgamma)[c] = static_cast<T>(b); static_cast<T*>(dbeta)[c] = static_cast<T>(a); }
}

}  // namespace alpha
