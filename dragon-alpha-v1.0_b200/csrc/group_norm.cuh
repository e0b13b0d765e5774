// Group normalisation of channels-last tensors with the activation that follows it, and its gradients.
//
//   xh = (x - mean) rstd,  z = xh gamma + beta,  y = act(z)        mean, rstd over the positions and the C / G channels of (sample, group)
//   dz = dy act'(z),  deltaGamma_c = sum dz xh,  deltaBeta_c = sum dz
//   deltaX = rstd (dz gamma - s1 - xh s2)                          s1, s2: means of dz gamma and dz gamma xh over (sample, group)
//
// Bound by HBM: the tensors are to be read once although nothing can be written before the last element of a group is known.
//
// Resident: a sample is cut into slabs of whole groups; a CTA, or a cluster of up to eight that share the positions, brings its part of a slab into shared
// memory by asynchronous copies, forms the sums there, adds those of its cluster, and writes the outputs from shared memory: each tensor crosses HBM once.  Several CTAs
// to an SM, so that one copies while another computes or stores.  A thread keeps one word of the row (four channels) and walks the positions, so that the words of
// neighbouring threads are neighbours in memory and a thread reads only what it copied itself.  Words of four elements, not of 16 bytes: what a thread holds of
// its channels fits 64 registers, for 32 warps on an SM.  Backward dz is kept in shared memory in fp32, so that a slope is formed once: arithmetic is the second bound.
//
// Streamed: what does not fit (and widths that are no multiple of four, a thread to an element): partial sums of runs of positions, their sum, and a second pass over
// the tensors, from their end, so that it begins with what the first left in L2.
//
// Variances come from differences to a mean: within a CTA's part (or eight positions of a thread), and parts are joined by their means; nothing is a
// difference of large sums.  Sums are fp32, joined in a fixed order.
#pragma once
#include "dependent_launch.cuh"
#include "fc_act.cuh"
#include "pairs.cuh"
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
template <class T, int V> struct NormWord;
template <class T> struct NormWord<T, 4> {
    using Raw = uint2;
    static __device__ void load(const Raw& r, float2 (&f)[2])
    {
        unpack16<T>(r.x, f[0].x, f[0].y);
        unpack16<T>(r.y, f[1].x, f[1].y);
    }
    static __device__ Raw store(const float2 (&f)[2]) { return make_uint2(pack16<T>(f[0].x, f[0].y), pack16<T>(f[1].x, f[1].y)); }
};
template <> struct NormWord<float, 4> {
    using Raw = float4;
    static __device__ void load(const Raw& r, float2 (&f)[2]) { f[0] = make_float2(r.x, r.y); f[1] = make_float2(r.z, r.w); }
    static __device__ Raw store(const float2 (&f)[2]) { return make_float4(f[0].x, f[0].y, f[1].x, f[1].y); }
};
// (one element: the second of the pair is 0 and goes nowhere)
template <class T> struct NormWord<T, 1> {
    using Raw = T;
    static __device__ void load(const Raw& r, float2 (&f)[1]) { f[0] = make_float2(static_cast<float>(r), 0.f); }
    static __device__ Raw store(const float2 (&f)[1]) { return static_cast<T>(f[0].x); }
};
template <class T> constexpr bool kNormFast = sizeof(T) == 2;

// Activations of 16-bit tensors by a sigmoid without the care that quotients and exponentials of denormal results take (good to 2^-21 of its value; below 1e-38 it is 0).
__device__ __forceinline__ Sigmoid sigmoid_lean(float z)
{
    float e, big;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(-1.44269504f * fabsf(z)));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(big) : "f"(1.f + e));
    const float small = e * big;
    return z >= 0.f ? Sigmoid{big, small} : Sigmoid{small, big};
}
template <int ACT, bool FAST> __device__ __forceinline__ float norm_value(float z, float k)
{
    if constexpr (FAST && ACT == ALPHA_ACT_SILU) return z * sigmoid_lean(z).pos;
    else if constexpr (FAST && ACT == ALPHA_ACT_GELU_TANH) return z * sigmoid_lean(1.59576912f * (z + 0.044715f * z * z * z)).pos;
    else if constexpr (FAST && ACT == ALPHA_ACT_SIGMOID) return sigmoid_lean(z).pos;
    else return act_value<ACT, FAST>(z, k);
}
template <int ACT, bool FAST> __device__ __forceinline__ float norm_slope(float z, float k)
{
    if constexpr (FAST && ACT == ALPHA_ACT_SILU) {
        const Sigmoid s = sigmoid_lean(z);
        return s.pos * fmaf(z, s.neg, 1.f);
    } else if constexpr (FAST && ACT == ALPHA_ACT_SIGMOID) {
        const Sigmoid s = sigmoid_lean(z);
        return s.pos * s.neg;
    } else {
        float value, slope;
        act_both<ACT, FAST>(z, k, value, slope);
        return slope;
    }
}

template <class T> __device__ __forceinline__ float affine_at(const void* p, int c, int f32, float none)
{
    return !p ? none : f32 ? static_cast<const float*>(p)[c] : static_cast<float>(static_cast<const T*>(p)[c]);
}
// gamma and beta of the V channels from c on.
template <class T, int V> __device__ __forceinline__ void load_affine(const Norm& p, int c, float2 (&gamma)[(V + 1) / 2], float2 (&beta)[(V + 1) / 2])
{
#pragma unroll
    for (int j = 0; j < (V + 1) / 2; ++j) {
        gamma[j] = make_float2(affine_at<T>(p.gamma, c + 2 * j, p.affine_f32, 1.f), V > 1 ? affine_at<T>(p.gamma, c + 2 * j + 1, p.affine_f32, 1.f) : 0.f);
        beta[j] = make_float2(affine_at<T>(p.beta, c + 2 * j, p.affine_f32, 0.f), V > 1 ? affine_at<T>(p.beta, c + 2 * j + 1, p.affine_f32, 0.f) : 0.f);
    }
}

template <int BYTES> __device__ __forceinline__ void copy_async(uint32_t to, const void* from)
{
    if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void copies_done() { asm volatile("cp.async.wait_all;" ::: "memory"); }
__device__ __forceinline__ float warp_sum(float x)
{
#pragma unroll
    for (int d = 16; d; d >>= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
    return x;
}
// A thread's four sums, as they lie in shared memory: red[j][thread].
__device__ __forceinline__ void put_sums(float* red, const float2 (&s)[2])
{
    red[threadIdx.x] = s[0].x;
    red[kNormThreads + threadIdx.x] = s[0].y;
    red[2 * kNormThreads + threadIdx.x] = s[1].x;
    red[3 * kNormThreads + threadIdx.x] = s[1].y;
}
// Channels' sums: over the rows of threads, into red[c % 4][c / 4].  `share` threads, neighbouring lanes, add a channel's (a power of two that divides 32).
__device__ __forceinline__ void channel_sums(float* red, const Norm& p, int arrays)
{
    const int wide = 4 * p.words, total = arrays * wide;
    int share = 1;
    while (share < 32 && total * share * 2 <= kNormThreads) share *= 2;
    __syncthreads();
    const int lane = threadIdx.x % share;
    for (int c0 = 0; c0 < total; c0 += kNormThreads / share) {
        const int c = c0 + static_cast<int>(threadIdx.x) / share, array = c / wide, ch = c - array * wide;
        float s = 0.f;
        const float* at = red + (array * 4 + ch % 4) * kNormThreads + ch / 4;
        if (c < total)
            for (int r = lane; r < p.rows; r += share) s += at[r * p.words];
        for (int d = share / 2; d; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
        __syncwarp();
        if (c < total && lane == 0) red[(array * 4 + ch % 4) * kNormThreads + ch / 4] = s;
    }
    __syncthreads();
}
// Groups' sums of channels' sums, a warp to a group: f(group, sum) in every lane.
template <class F> __device__ __forceinline__ void group_sums(const float* red, const Norm& p, int groups, F&& f)
{
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int g = warp; g < groups; g += kNormThreads / 32) {
        float s = 0.f;
        for (int i = lane; i < p.D; i += 32) {
            const int c = g * p.D + i;
            s += red[(c % 4) * kNormThreads + c / 4];
        }
        f(g, warp_sum(s));
    }
}

// Shared memory of a resident CTA: its words of X, backward 16 bytes for each of deltaY and dz, four (eight) sums of each thread, and the groups'.
__host__ __device__ inline size_t norm_smem(bool back, int size, int part, int words, int groups)
{
    return static_cast<size_t>(part) * words * (4 * size + (back ? 16 : 0)) + kNormThreads * 16 * (back ? 2 : 1) + static_cast<size_t>(groups) * 16;
}

template <class T, bool BACK>
__global__ void __launch_bounds__(kNormThreads, 4) norm_resident_kernel(const __grid_constant__ Norm p)
{
    using W = NormWord<T, 4>;
    using Raw = typename W::Raw;
    extern __shared__ __align__(128) uint8_t smem[];
    const int cl = p.cluster, rank = cl > 1 ? static_cast<int>(cluster_ctarank()) : 0, item = blockIdx.x / cl, n = item / p.slabs, slab = item - n * p.slabs;
    const int r0 = rank * p.part, mine = min(p.part, p.R - r0);             // (positive: no part is empty)
    const int ty = threadIdx.x / p.words, tx = threadIdx.x - ty * p.words, c0 = slab * p.words * 4, groups = p.words * 4 / p.D, g0 = c0 / p.D, c = c0 + tx * 4;
    const bool busy = ty < p.rows;
    const int first = busy ? ty * p.words + tx : 0, step = p.rows * p.words, last = busy ? mine * p.words : 0;      // its words: first, first + step, ... < last
    float4* ds = reinterpret_cast<float4*>(smem);                                                                    // deltaY, then dz
    Raw* xs = reinterpret_cast<Raw*>(smem + (BACK ? static_cast<size_t>(p.part) * p.words * 16 : 0));
    float* red = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(xs) + ((static_cast<size_t>(p.part) * p.words * sizeof(Raw) + 15) & ~static_cast<size_t>(15)));
    float2* own = reinterpret_cast<float2*>(red + 4 * kNormThreads * (BACK ? 2 : 1));      // this CTA's sums of each group
    float2* all = own + groups;                                                            // the cluster's
    const size_t from = (static_cast<size_t>(n) * p.R + r0 + ty) * p.C + c, jump = static_cast<size_t>(p.rows) * p.C;
    grid_dependency_wait();
    grid_dependency_trigger();
    {
        const T *x = static_cast<const T*>(p.X) + from, *y = BACK ? static_cast<const T*>(p.dY) + from : nullptr;
        const uint32_t to = smem_u32(xs), to_y = smem_u32(ds);
#pragma unroll 4
        for (int i = first; i < last; i += step) {
            copy_async<sizeof(Raw)>(to + i * sizeof(Raw), x);
            x += jump;
            if (BACK) { copy_async<sizeof(Raw)>(to_y + i * 16, y); y += jump; }
        }
    }
    float2 gamma[2], beta[2], mean[2], s[2], q[2];
    load_affine<T, 4>(p, c, gamma, beta);
    const int gi[4] = {c / p.D - g0, (c + 1) / p.D - g0, (c + 2) / p.D - g0, (c + 3) / p.D - g0};         // groups of its channels
    const float count = static_cast<float>(p.R) * static_cast<float>(p.D);
    T* out = static_cast<T*>(p.out) + from;
#pragma unroll
    for (int j = 0; j < 2; ++j) s[j] = q[j] = make_float2(0.f, 0.f);
    if constexpr (!BACK) {
        copies_done();
        const float own_count = static_cast<float>(mine) * static_cast<float>(p.D);
#pragma unroll 4
        for (int i = first; i < last; i += step) {
            float2 f[2];
            W::load(xs[i], f);
            s[0] = add2(s[0], f[0]);
            s[1] = add2(s[1], f[1]);
        }
        put_sums(red, s);
        channel_sums(red, p, 1);
        group_sums(red, p, groups, [&](int g, float sum) { if ((threadIdx.x & 31) == 0) own[g].x = sum / own_count; });
        __syncthreads();
        mean[0] = make_float2(own[gi[0]].x, own[gi[1]].x);
        mean[1] = make_float2(own[gi[2]].x, own[gi[3]].x);
#pragma unroll 4
        for (int i = first; i < last; i += step) {
            float2 f[2];
            W::load(xs[i], f);
#pragma unroll
            for (int j = 0; j < 2; ++j) { f[j] = add2(f[j], neg2(mean[j])); q[j] = fma2(f[j], f[j], q[j]); }
        }
        put_sums(red, q);
        channel_sums(red, p, 1);
        group_sums(red, p, groups, [&](int g, float sum) { if ((threadIdx.x & 31) == 0) own[g].y = sum; });
        if (cl > 1) cluster_sync_all();
        else __syncthreads();
        // mean and rstd of a group from its parts
        for (int g = threadIdx.x; g < groups; g += kNormThreads) {
            float m = own[g].x, squares = own[g].y;
            if (cl > 1) {
                const uint32_t at = smem_u32(own + g);
                float sum = 0.f;
                for (int r = 0; r < cl; ++r) sum = fmaf(ld_shared_cluster(mapa_u32(at, r)), static_cast<float>(min(p.part, p.R - r * p.part)), sum);
                m = sum / static_cast<float>(p.R);
                squares = 0.f;
                for (int r = 0; r < cl; ++r) {
                    const uint32_t peer = mapa_u32(at, r);
                    const float d = ld_shared_cluster(peer) - m;
                    squares += ld_shared_cluster(peer + 4) + d * d * (static_cast<float>(min(p.part, p.R - r * p.part)) * static_cast<float>(p.D));
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
        mean[0] = make_float2(all[gi[0]].x, all[gi[1]].x);
        mean[1] = make_float2(all[gi[2]].x, all[gi[3]].x);
        gamma[0] = mul2(gamma[0], make_float2(all[gi[0]].y, all[gi[1]].y));
        gamma[1] = mul2(gamma[1], make_float2(all[gi[2]].y, all[gi[3]].y));
        with_act(p.act, [&](auto a) {
            constexpr int ACT = decltype(a)::value;
#pragma unroll 2
            for (int i = first; i < last; i += step) {
                float2 f[2];
                W::load(xs[i], f);
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    f[j] = fma2(add2(f[j], neg2(mean[j])), gamma[j], beta[j]);
                    f[j] = make_float2(norm_value<ACT, kNormFast<T>>(f[j].x, p.k), norm_value<ACT, kNormFast<T>>(f[j].y, p.k));
                }
                *reinterpret_cast<Raw*>(out) = W::store(f);
                out += jump;
            }
        });
    } else {
        // s: sums of dz, q: of dz (x - mean)
        const size_t at_group = static_cast<size_t>(n) * p.G + g0;
        float2 rstd[2], scale[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            mean[j] = make_float2(p.mean[at_group + gi[2 * j]], p.mean[at_group + gi[2 * j + 1]]);
            rstd[j] = make_float2(p.rstd[at_group + gi[2 * j]], p.rstd[at_group + gi[2 * j + 1]]);
            scale[j] = mul2(rstd[j], gamma[j]);
        }
        copies_done();
        with_act(p.act, [&](auto a) {
            constexpr int ACT = decltype(a)::value;
#pragma unroll 2
            for (int i = first; i < last; i += step) {
                float2 x[2], y[2];
                W::load(xs[i], x);
                W::load(*reinterpret_cast<const Raw*>(ds + i), y);
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    x[j] = add2(x[j], neg2(mean[j]));
                    const float2 z = fma2(x[j], scale[j], beta[j]);
                    y[j] = mul2(y[j], make_float2(norm_slope<ACT, kNormFast<T>>(z.x, p.k), norm_slope<ACT, kNormFast<T>>(z.y, p.k)));
                    s[j] = add2(s[j], y[j]);
                    q[j] = fma2(y[j], x[j], q[j]);
                }
                ds[i] = make_float4(y[0].x, y[0].y, y[1].x, y[1].y);
            }
        });
#pragma unroll
        for (int j = 0; j < 2; ++j) q[j] = mul2(q[j], rstd[j]);
        put_sums(red, s);
        put_sums(red + 4 * kNormThreads, q);
        channel_sums(red, p, 2);
        // over the cluster: every CTA adds all parts in the same order
        float keep[8];
        if (cl > 1) cluster_sync_all();
        if (threadIdx.x < p.words) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                keep[j] = 0.f;
                if (cl == 1) { keep[j] = red[j * kNormThreads + threadIdx.x]; continue; }
                const uint32_t at = smem_u32(red + j * kNormThreads + threadIdx.x);
                for (int r = 0; r < cl; ++r) keep[j] += ld_shared_cluster(mapa_u32(at, r));
            }
        }
        if (cl > 1) cluster_sync_all();          // (all parts have been read)
        if (threadIdx.x < p.words) {
            const float by[4] = {gamma[0].x, gamma[0].y, gamma[1].x, gamma[1].y};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (rank == 0) p.sums[static_cast<size_t>(n) * p.C + c + j] = make_float2(keep[j], keep[4 + j]);
                red[j * kNormThreads + threadIdx.x] = keep[j] * by[j];
                red[(4 + j) * kNormThreads + threadIdx.x] = keep[4 + j] * by[j];
            }
        }
        __syncthreads();
        group_sums(red, p, groups, [&](int g, float sum) { if ((threadIdx.x & 31) == 0) all[g].x = sum / count; });
        group_sums(red + 4 * kNormThreads, p, groups, [&](int g, float sum) { if ((threadIdx.x & 31) == 0) all[g].y = sum / count; });
        __syncthreads();
        // deltaX = scale dz + more (x - mean) + base
        float2 more[2], base[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const float2 a = all[gi[2 * j]], b = all[gi[2 * j + 1]];
            base[j] = neg2(mul2(rstd[j], make_float2(a.x, b.x)));
            more[j] = neg2(mul2(mul2(rstd[j], rstd[j]), make_float2(a.y, b.y)));
        }
#pragma unroll 4
        for (int i = first; i < last; i += step) {
            float2 x[2];
            W::load(xs[i], x);
            const float4 d = ds[i];
            x[0] = fma2(make_float2(d.x, d.y), scale[0], fma2(add2(x[0], neg2(mean[0])), more[0], base[0]));
            x[1] = fma2(make_float2(d.z, d.w), scale[1], fma2(add2(x[1], neg2(mean[1])), more[1], base[1]));
            *reinterpret_cast<Raw*>(out) = W::store(x);
            out += jump;
        }
    }
}

// ---- streamed ---------------------------------------------------------------------------------------------------

// Where a CTA of the streamed passes is: a block of columns, a run of positions, a sample.
struct NormAt { int n, run, count, ty, word; bool busy; size_t from; };
template <int V> __device__ __forceinline__ NormAt norm_at(const Norm& p, unsigned block)
{
    NormAt a;
    const unsigned col = block % p.blocks, rest = block / p.blocks;
    a.run = rest % p.runs; a.n = rest / p.runs;
    const int r0 = a.run * p.part;
    a.count = min(p.part, p.R - r0);
    a.ty = threadIdx.x / p.words;
    a.word = col * p.words + threadIdx.x - a.ty * p.words;
    a.busy = a.ty < p.rows && a.word < p.C / V;
    a.from = (static_cast<size_t>(a.n) * p.R + r0) * p.C + static_cast<size_t>(a.word) * V;
    return a;
}
// Mean and squared differences of a run, or its sums of dz and dz xh, for every channel.
template <class T, int V, bool BACK>
__global__ void __launch_bounds__(kNormThreads, 4) norm_sums_kernel(const __grid_constant__ Norm p)
{
    using W = NormWord<T, V>;
    using Raw = typename W::Raw;
    constexpr int U = BACK ? 4 : 8, P = (V + 1) / 2;
    __shared__ float red[2 * V * kNormThreads];
    grid_dependency_wait();
    grid_dependency_trigger();
    const NormAt a = norm_at<V>(p, blockIdx.x);
    float2 s[P], q[P];
#pragma unroll
    for (int j = 0; j < P; ++j) s[j] = q[j] = make_float2(0.f, 0.f);
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
                float2 m[P], d2[P];
#pragma unroll
                for (int j = 0; j < P; ++j) m[j] = d2[j] = make_float2(0.f, 0.f);
#pragma unroll
                for (int i = 0; i < U; ++i) {
                    float2 f[P];
                    W::load(raw[i], f);
#pragma unroll
                    for (int j = 0; j < P; ++j) m[j] = i < have ? add2(m[j], f[j]) : m[j];
                }
#pragma unroll
                for (int j = 0; j < P; ++j) m[j] = mul2(m[j], make_float2(inverse, inverse));
#pragma unroll
                for (int i = 0; i < U; ++i) {
                    float2 f[P];
                    W::load(raw[i], f);
#pragma unroll
                    for (int j = 0; j < P; ++j) {
                        const float2 d = add2(f[j], neg2(m[j]));
                        d2[j] = i < have ? fma2(d, d, d2[j]) : d2[j];
                    }
                }
                const float cross = seen * weight;
#pragma unroll
                for (int j = 0; j < P; ++j) {
                    const float2 d = add2(m[j], neg2(s[j]));
                    s[j] = fma2(d, make_float2(weight, weight), s[j]);
                    q[j] = add2(q[j], fma2(mul2(d, d), make_float2(cross, cross), d2[j]));
                }
                seen = total;
            }
        } else {
            float2 mean[P], rstd[P], gamma[P], beta[P];
            load_affine<T, V>(p, a.word * V, gamma, beta);
#pragma unroll
            for (int j = 0; j < P; ++j) {
                const size_t g = static_cast<size_t>(a.n) * p.G + (a.word * V + 2 * j) / p.D, h = static_cast<size_t>(a.n) * p.G + (a.word * V + 2 * j + (V > 1)) / p.D;
                mean[j] = make_float2(p.mean[g], p.mean[h]);
                rstd[j] = make_float2(p.rstd[g], p.rstd[h]);
                gamma[j] = mul2(gamma[j], rstd[j]);
            }
            with_act(p.act, [&](auto act) {
                constexpr int ACT = decltype(act)::value;
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
                        float2 fx[P], fy[P];
                        W::load(rx[i], fx);
                        W::load(ry[i], fy);
#pragma unroll
                        for (int j = 0; j < P; ++j) {
                            fx[j] = add2(fx[j], neg2(mean[j]));
                            const float2 z = fma2(fx[j], gamma[j], beta[j]);
                            fy[j] = mul2(fy[j], make_float2(norm_slope<ACT, kNormFast<T>>(z.x, p.k), V > 1 ? norm_slope<ACT, kNormFast<T>>(z.y, p.k) : 0.f));
                            s[j] = add2(s[j], fy[j]);
                            q[j] = fma2(fy[j], fx[j], q[j]);
                        }
                    }
                }
            });
#pragma unroll
            for (int j = 0; j < P; ++j) q[j] = mul2(q[j], rstd[j]);
        }
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
        red[j * kNormThreads + threadIdx.x] = j % 2 ? s[j / 2].y : s[j / 2].x;
        red[(V + j) * kNormThreads + threadIdx.x] = j % 2 ? q[j / 2].y : q[j / 2].x;
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

constexpr int kJoinNormThreads = 512;
__device__ __forceinline__ float block_sum(float x, float* shared)
{
    x = warp_sum(x);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = x;
    __syncthreads();
    x = 0.f;
#pragma unroll
    for (int w = 0; w < kJoinNormThreads / 32; ++w) x += shared[w];
    return x;
}
// A CTA to each (sample, group): its mean and rstd, or s1 and s2 and the channels' sums, from those of the runs.
template <class T, bool BACK>
__global__ void __launch_bounds__(kJoinNormThreads) norm_join_kernel(const __grid_constant__ Norm p)
{
    __shared__ float shared[kJoinNormThreads / 32];
    grid_dependency_wait();
    grid_dependency_trigger();
    const int n = blockIdx.x / p.G, g = blockIdx.x - n * p.G;
    const float2* from = p.partial + static_cast<size_t>(n) * p.runs * p.C + g * p.D;
    const float count = static_cast<float>(p.R) * static_cast<float>(p.D);
    if constexpr (!BACK) {
        const int entries = p.runs * p.D;
        float sum = 0.f, squares = 0.f;
#pragma unroll 4
        for (int i = threadIdx.x; i < entries; i += kJoinNormThreads) {
            const int run = i / p.D;
            sum = fmaf(from[static_cast<size_t>(run) * p.C + i - run * p.D].x, static_cast<float>(min(p.part, p.R - run * p.part)), sum);
        }
        const float mean = block_sum(sum, shared) / count;
#pragma unroll 4
        for (int i = threadIdx.x; i < entries; i += kJoinNormThreads) {
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
        for (int d = warp; d < p.D; d += kJoinNormThreads / 32) {
            float a = 0.f, b = 0.f;
#pragma unroll 4
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
__global__ void __launch_bounds__(kNormThreads, 4) norm_apply_kernel(const __grid_constant__ Norm p)
{
    using W = NormWord<T, V>;
    using Raw = typename W::Raw;
    constexpr int U = 4, P = (V + 1) / 2;
    grid_dependency_wait();
    grid_dependency_trigger();
    const NormAt a = norm_at<V>(p, gridDim.x - 1 - blockIdx.x);
    if (!a.busy) return;
    float2 mean[P], gamma[P], beta[P], more[P], base[P];
    load_affine<T, V>(p, a.word * V, gamma, beta);
#pragma unroll
    for (int j = 0; j < P; ++j) {
        const size_t g = static_cast<size_t>(a.n) * p.G + (a.word * V + 2 * j) / p.D, h = static_cast<size_t>(a.n) * p.G + (a.word * V + 2 * j + (V > 1)) / p.D;
        const float2 t = p.group[g], u = p.group[h];
        if constexpr (BACK) {
            const float2 rstd = make_float2(p.rstd[g], p.rstd[h]);
            mean[j] = make_float2(p.mean[g], p.mean[h]);
            gamma[j] = mul2(gamma[j], rstd);
            base[j] = neg2(mul2(rstd, make_float2(t.x, u.x)));
            more[j] = neg2(mul2(mul2(rstd, rstd), make_float2(t.y, u.y)));
        } else {
            mean[j] = make_float2(t.x, u.x);
            gamma[j] = mul2(gamma[j], make_float2(t.y, u.y));
        }
    }
    const T *x = static_cast<const T*>(p.X) + a.from, *y = BACK ? static_cast<const T*>(p.dY) + a.from : nullptr;
    T* out = static_cast<T*>(p.out) + a.from;
    const size_t step = static_cast<size_t>(p.rows) * p.C;
    with_act(p.act, [&](auto act) {
        constexpr int ACT = decltype(act)::value;
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
                float2 f[P], fy[P];
                W::load(rx[i], f);
                if (BACK) W::load(ry[i], fy);
#pragma unroll
                for (int j = 0; j < P; ++j) {
                    f[j] = add2(f[j], neg2(mean[j]));
                    const float2 z = fma2(f[j], gamma[j], beta[j]);
                    if constexpr (BACK) {
                        fy[j] = mul2(fy[j], make_float2(norm_slope<ACT, kNormFast<T>>(z.x, p.k), V > 1 ? norm_slope<ACT, kNormFast<T>>(z.y, p.k) : 0.f));
                        f[j] = fma2(fy[j], gamma[j], fma2(f[j], more[j], base[j]));
                    } else {
                        f[j] = make_float2(norm_value<ACT, kNormFast<T>>(z.x, p.k), V > 1 ? norm_value<ACT, kNormFast<T>>(z.y, p.k) : 0.f);
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
