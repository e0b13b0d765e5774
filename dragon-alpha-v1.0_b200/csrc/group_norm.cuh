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
// its channels fits 64 registers, for 32 warps on an SM.  Arithmetic is the second bound.
// 512 x 32 x 32 x 64 fp32: 47 us in a graph, 5.7 TB/s; gradients of 128 x 56 x 56 x 64 fp32: 81 us, 3.8 TB/s.
//
// Streamed: what does not fit (and widths that are no multiple of four, a thread to an element): partial sums of runs of positions, their sum, and a second pass over
// the tensors, from their end, so that it begins with what the first left in L2.
// 512 x 512 x 256 bf16: 78 us; gradients of 8 x 64 x 64 x 640 bf16: 52 us; instruction issue bounds either pass as much as HBM.
//
// Variances come from differences to a mean: within a CTA's part (or eight positions of a thread), and parts are joined by their means; nothing is a
// difference of large sums.  Sums are fp32, joined in a fixed order.
#pragma once
#include "dependent_launch.cuh"
#include "fast_div.cuh"
#include "fc_act.cuh"
#include "pairs.cuh"
#include "sm100_ptx.cuh"

#include <type_traits>

namespace alpha {

constexpr int kNormThreads = 256;

struct Norm {
    const void *X, *dY;
    void* out;                      // Y, or deltaX
    const void *gamma, *beta;       // (or NULL: 1 and 0)
    int affine_f32;                 // gamma and beta are floats
    float *mean, *rstd;             // [N][G]: written by a forward call (may be NULL), read by a backward one
    float2* sums;                   // [N][cluster][C] sums of dz and dz xh
    int N, R, C, G, D;
    float eps, k;
    int act;
    // resident: words of a slab, slabs of a row, CTAs that share a slab, positions of each, rows of threads
    int words, slabs, cluster, part, rows;
    int groups;                     // of a slab
    int slots, span;                // sums of a word that belong to different groups (1, 2 or 4), and how many of a row a group has
    FastDiv by_words, by_slabs, by_cluster, by_D, by_span;
    // streamed: column blocks of `words` words, runs of `part` positions
    int blocks, runs;
    int whole;                      // forward: a column block holds whole groups, whose partial sums are kept and not those of channels
    float2* partial;                // [N][runs][C, or G] mean and sum of squared differences, or sums of dz and dz xh
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
// Backward: dz takes the place of deltaY in shared memory, so that a slope is formed once - in fp32; of 16-bit tensors it would take twice deltaY's room, and slopes are cheaper.
template <class T> constexpr bool kKeepDz = sizeof(T) == 4;

// Activations of 16-bit tensors by s = 1 / (1 + exp(-u)), good to 2^-21 of its value down to u = -87 and 0 below that (1e-38); two values at a time.
__device__ __forceinline__ float2 exp_of(float2 u)                // exp(-u)
{
    u = mul2(u, twice(-1.44269504f));
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(u.x));
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(u.y));
    return u;
}
__device__ __forceinline__ float2 inverse_of(float2 x)
{
    asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(x.x));
    asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(x.y));
    return x;
}
template <int ACT, bool FAST> __device__ __forceinline__ float2 norm_value(float2 z, float k)
{
    if constexpr (ACT == ALPHA_ACT_NONE) return z;
    else if constexpr (FAST && (ACT == ALPHA_ACT_SILU || ACT == ALPHA_ACT_SIGMOID || ACT == ALPHA_ACT_GELU_TANH)) {
        // (gelu_tanh: z sigmoid(2 sqrt(2 / pi) (z + 0.044715 z^3)))
        const float2 u = ACT == ALPHA_ACT_GELU_TANH ? mul2(z, fma2(mul2(z, z), twice(1.59576912f * 0.044715f), twice(1.59576912f))) : z, s = inverse_of(add2(twice(1.f), exp_of(u)));
        return ACT == ALPHA_ACT_SIGMOID ? s : mul2(z, s);
    } else return make_float2(act_value<ACT, FAST>(z.x, k), act_value<ACT, FAST>(z.y, k));
}
template <int ACT, bool FAST> __device__ __forceinline__ float2 norm_slope(float2 z, float k)
{
    if constexpr (ACT == ALPHA_ACT_NONE) return twice(1.f);
    else if constexpr (ACT == ALPHA_ACT_LEAKY_RELU) return make_float2(z.x > 0.f ? 1.f : k, z.y > 0.f ? 1.f : k);
    else if constexpr (FAST && (ACT == ALPHA_ACT_SILU || ACT == ALPHA_ACT_SIGMOID)) {
        z = make_float2(fmaxf(z.x, -87.f), fmaxf(z.y, -87.f));      // (no exponential of Inf; a NaN's gradient is that of deltaY)
        const float2 e = exp_of(z), s = inverse_of(add2(twice(1.f), e)), rest = mul2(e, s);
        return mul2(s, ACT == ALPHA_ACT_SILU ? fma2(z, rest, twice(1.f)) : rest);
    } else {
        float value;
        float2 slope;
        act_both<ACT, FAST>(z.x, k, value, slope.x);
        act_both<ACT, FAST>(z.y, k, value, slope.y);
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
        gamma[j] = twice(1.f);
        beta[j] = twice(0.f);
    }
    if (!p.gamma) return;
    auto load = [&](auto type) {
        using A = decltype(type);
        const A *g = static_cast<const A*>(p.gamma) + c, *b = static_cast<const A*>(p.beta) + c;
#pragma unroll
        for (int j = 0; j < (V + 1) / 2; ++j) {
            gamma[j] = make_float2(static_cast<float>(g[2 * j]), V > 1 ? static_cast<float>(g[2 * j + (V > 1)]) : 0.f);
            beta[j] = make_float2(static_cast<float>(b[2 * j]), V > 1 ? static_cast<float>(b[2 * j + (V > 1)]) : 0.f);
        }
    };
    if (sizeof(T) == 4 || p.affine_f32) load(float{});
    else load(T{});
}

template <int BYTES> __device__ __forceinline__ void copy_async(uint32_t to, const void* from)
{
    if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// (all groups but the last N)
template <int N> __device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void copies_done() { asm volatile("cp.async.wait_all;" ::: "memory"); }
// (after a __syncwarp: the aligned forms take a whole warp)
__device__ __forceinline__ void cluster_arrive() { __syncwarp(); asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { __syncwarp(); asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
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
// The same for sums of groups only: those of a group are added first, where a word lies in one or in two.
__device__ __forceinline__ void put_group_sums(float* red, const Norm& p, const float2 (&s)[2])
{
    if (p.slots == 4) return put_sums(red, s);
    const float a = s[0].x + s[0].y, b = s[1].x + s[1].y;
    red[threadIdx.x] = p.slots == 1 ? a + b : a;
    if (p.slots == 2) red[kNormThreads + threadIdx.x] = b;
}
// Groups' sums over `rows` rows of `span` slots, a warp to a group: f(group, sum) in its first lane.
template <class F> __device__ __forceinline__ void group_sums(const float* red, const Norm& p, int slots, int span, const FastDiv& by_span, int rows, int groups, F&& f)
{
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, shift = slots == 4 ? 2 : slots - 1, count = rows * span;
    for (int g = warp; g < groups; g += kNormThreads / 32) {
        float s = 0.f;
        for (int i = lane; i < count; i += 32) {
            unsigned row, k;
            by_span.divmod(static_cast<unsigned>(i), row, k);
            k += g * span;
            s += red[(k & (slots - 1)) * kNormThreads + row * p.words + (k >> shift)];
        }
        s = warp_sum(s);
        if (lane == 0) f(g, s);
    }
}
// Channels' sums: over the rows of threads, into the first: red[c % 4][c / 4].  `share` threads, neighbouring lanes, add a channel's (a power of two that divides 32).
__device__ __forceinline__ void channel_sums(float* red, const Norm& p, int arrays)
{
    const int total = arrays * 4 * p.words;
    int shift = 0;
    while (shift < 5 && total << (shift + 1) <= kNormThreads) ++shift;
    const int share = 1 << shift, lane = threadIdx.x & (share - 1);
    for (int c0 = 0; c0 < total; c0 += kNormThreads >> shift) {
        const int c = c0 + static_cast<int>(threadIdx.x >> shift);
        unsigned array = 0, word = 0;                             // arrays of a word's channels
        p.by_words.divmod(static_cast<unsigned>(c), array, word);
        float s = 0.f;
        float* at = red + array * kNormThreads + word;
        if (c < total)
            for (int r = lane; r < p.rows; r += share) s += at[r * p.words];
        for (int d = share / 2; d; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
        __syncwarp();
        if (c < total && lane == 0) at[0] = s;
    }
}

__device__ __forceinline__ void st_cluster_f2(uint32_t at, float x, float y) { asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(at), "f"(x), "f"(y) : "memory"); }

// Shared memory of a resident CTA: its words of X, backward of deltaY; four (eight) sums of each thread, the groups' sums of every CTA of the cluster, their total.
__host__ __device__ inline size_t norm_smem(bool back, int size, int part, int words, int groups, int cluster)
{
    const size_t tensors = (static_cast<size_t>(part) * words * 4 * size * (back ? 2 : 1) + 15) & ~static_cast<size_t>(15);
    return tensors + kNormThreads * 16 * (back ? 2 : 1) + static_cast<size_t>(groups) * 8 * (cluster + 1);
}

template <class T, bool BACK>
__global__ void __launch_bounds__(kNormThreads, 4) norm_resident_kernel(const __grid_constant__ Norm p)
{
    using W = NormWord<T, 4>;
    using Raw = typename W::Raw;
    extern __shared__ __align__(128) uint8_t smem[];
    const int cl = p.cluster, rank = cl > 1 ? static_cast<int>(cluster_ctarank()) : 0, groups = p.groups;
    unsigned item, n, slab, ty_, tx_, unused;
    p.by_cluster.divmod(blockIdx.x, item, unused);
    p.by_slabs.divmod(item, n, slab);
    p.by_words.divmod(threadIdx.x, ty_, tx_);
    const int r0 = rank * p.part, mine = min(p.part, p.R - r0);             // (positive: no part is empty)
    const int ty = ty_, tx = tx_, c = slab * p.words * 4 + tx * 4;
    const bool busy = ty < p.rows;
    const int first = busy ? ty * p.words + tx : 0, step = p.rows * p.words, last = busy ? mine * p.words : 0;      // its words: first, first + step, ... < last
    Raw* xs = reinterpret_cast<Raw*>(smem);
    Raw* ys = xs + static_cast<size_t>(p.part) * p.words;                                                            // deltaY; of fp32 tensors dz later
    float* red = reinterpret_cast<float*>(smem + ((static_cast<size_t>(p.part) * p.words * sizeof(Raw) * (BACK ? 2 : 1) + 15) & ~static_cast<size_t>(15)));
    float2* parts = reinterpret_cast<float2*>(red + 4 * kNormThreads * (BACK ? 2 : 1));    // [rank][group], written by every CTA of the cluster
    float2* all = parts + cl * groups;
    const size_t from = (static_cast<size_t>(n) * p.R + r0 + ty) * p.C + c, jump = static_cast<size_t>(p.rows) * p.C, at_group = static_cast<size_t>(n) * p.G + slab * groups;
    grid_dependency_wait();
    grid_dependency_trigger();
    {
        const T *x = static_cast<const T*>(p.X) + from, *y = BACK ? static_cast<const T*>(p.dY) + from : nullptr;
        const uint32_t to = smem_u32(xs), to_y = smem_u32(ys);
#pragma unroll 4
        for (int i = first; i < last; i += step) {
            copy_async<sizeof(Raw)>(to + i * sizeof(Raw), x);
            x += jump;
            if (BACK) { copy_async<sizeof(Raw)>(to_y + i * sizeof(Raw), y); y += jump; }
        }
    }
    int gi[4];                                                                             // groups of its channels, within the slab
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        unsigned g;
        p.by_D.divmod(static_cast<unsigned>(tx * 4 + j), g, unused);
        gi[j] = static_cast<int>(g);
    }
    const float count = static_cast<float>(p.R) * static_cast<float>(p.D);
    float2 gamma[2], beta[2], mean[2], s[2], q[2];            // (means negated)
    load_affine<T, 4>(p, c, gamma, beta);
    T* out = static_cast<T*>(p.out) + from;
#pragma unroll
    for (int j = 0; j < 2; ++j) s[j] = q[j] = make_float2(0.f, 0.f);
    // a group's two sums to every CTA of the cluster; then all have them
    auto share = [&](int g, float x, float y) {
        if (cl == 1) { parts[g] = make_float2(x, y); return; }
        const uint32_t at = smem_u32(parts + rank * groups + g);
        for (int r = 0; r < cl; ++r) st_cluster_f2(mapa_u32(at, r), x, y);
    };
    auto shared_by_all = [&] {
        if (cl > 1) { cluster_arrive(); cluster_wait(); }
        else __syncthreads();
    };
    // (a cluster's CTAs have all begun before one writes to another)
    if (cl > 1) cluster_arrive();
    copies_done();
    if constexpr (!BACK) {
        const float own_count = static_cast<float>(mine) * static_cast<float>(p.D);
#pragma unroll 4
        for (int i = first; i < last; i += step) {
            float2 f[2];
            W::load(xs[i], f);
            s[0] = add2(s[0], f[0]);
            s[1] = add2(s[1], f[1]);
        }
        put_group_sums(red, p, s);
        __syncthreads();
        group_sums(red, p, p.slots, p.span, p.by_span, p.rows, groups, [&](int g, float sum) { all[g].x = sum / own_count; });
        __syncthreads();
        mean[0] = neg2(make_float2(all[gi[0]].x, all[gi[1]].x));
        mean[1] = neg2(make_float2(all[gi[2]].x, all[gi[3]].x));
#pragma unroll 4
        for (int i = first; i < last; i += step) {
            float2 f[2];
            W::load(xs[i], f);
#pragma unroll
            for (int j = 0; j < 2; ++j) { f[j] = add2(f[j], mean[j]); q[j] = fma2(f[j], f[j], q[j]); }
        }
        put_group_sums(red, p, q);
        if (cl > 1) cluster_wait();
        __syncthreads();
        group_sums(red, p, p.slots, p.span, p.by_span, p.rows, groups, [&](int g, float sum) { share(g, all[g].x, sum); });
        shared_by_all();
        // mean and rstd of a group from its parts
        for (int g = threadIdx.x; g < groups; g += kNormThreads) {
            float m = parts[g].x, squares = parts[g].y;
            if (cl > 1) {
                float sum = 0.f;
                for (int r = 0; r < cl; ++r) sum = fmaf(parts[r * groups + g].x, static_cast<float>(min(p.part, p.R - r * p.part)), sum);
                m = sum / static_cast<float>(p.R);
                squares = 0.f;
                for (int r = 0; r < cl; ++r) {
                    const float2 e = parts[r * groups + g];
                    const float d = e.x - m;
                    squares += e.y + d * d * (static_cast<float>(min(p.part, p.R - r * p.part)) * static_cast<float>(p.D));
                }
            }
            const float r = 1.f / sqrtf(squares / count + p.eps);
            all[g] = make_float2(m, r);
            if (rank == 0 && p.mean) {
                p.mean[at_group + g] = m;
                p.rstd[at_group + g] = r;
            }
        }
        __syncthreads();
        mean[0] = neg2(make_float2(all[gi[0]].x, all[gi[1]].x));
        mean[1] = neg2(make_float2(all[gi[2]].x, all[gi[3]].x));
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
                    f[j] = fma2(add2(f[j], mean[j]), gamma[j], beta[j]);
                    f[j] = norm_value<ACT, kNormFast<T>>(f[j], p.k);
                }
                *reinterpret_cast<Raw*>(out) = W::store(f);
                out += jump;
            }
        });
    } else {
        // s: sums of dz, q: of dz (x - mean)
        float2 rstd[2], scale[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            mean[j] = neg2(make_float2(p.mean[at_group + gi[2 * j]], p.mean[at_group + gi[2 * j + 1]]));
            rstd[j] = make_float2(p.rstd[at_group + gi[2 * j]], p.rstd[at_group + gi[2 * j + 1]]);
            scale[j] = mul2(rstd[j], gamma[j]);
        }
        with_act(p.act, [&](auto a) {
            constexpr int ACT = decltype(a)::value;
#pragma unroll 2
            for (int i = first; i < last; i += step) {
                float2 x[2], y[2];
                W::load(xs[i], x);
                W::load(ys[i], y);
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    x[j] = add2(x[j], mean[j]);
                    const float2 z = fma2(x[j], scale[j], beta[j]);
                    if (ACT != ALPHA_ACT_NONE) y[j] = mul2(y[j], norm_slope<ACT, kNormFast<T>>(z, p.k));
                    s[j] = add2(s[j], y[j]);
                    q[j] = fma2(y[j], x[j], q[j]);
                }
                if constexpr (kKeepDz<T>) ys[i] = W::store(y);
            }
        });
#pragma unroll
        for (int j = 0; j < 2; ++j) q[j] = mul2(q[j], rstd[j]);
        put_sums(red, s);
        put_sums(red + 4 * kNormThreads, q);
        __syncthreads();
        channel_sums(red, p, 2);
        __syncthreads();
        if (threadIdx.x < p.words) {
            // the CTA's sums of its channels, for deltaGamma and deltaBeta; weighted by gamma for those of the groups
            const float by[4] = {gamma[0].x, gamma[0].y, gamma[1].x, gamma[1].y};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float *x = red + j * kNormThreads + threadIdx.x, *y = x + 4 * kNormThreads;
                p.sums[(static_cast<size_t>(n) * cl + rank) * p.C + c + j] = make_float2(*x, *y);
                *x *= by[j];
                *y *= by[j];
            }
        }
        if (cl > 1) cluster_wait();
        __syncthreads();
        group_sums(red, p, 4, p.D, p.by_D, 1, groups, [&](int g, float sum) { all[g].x = sum; });
        group_sums(red + 4 * kNormThreads, p, 4, p.D, p.by_D, 1, groups, [&](int g, float sum) { share(g, all[g].x, sum); });
        shared_by_all();
        for (int g = threadIdx.x; g < groups; g += kNormThreads) {
            float2 sum = parts[g];
            for (int r = 1; r < cl; ++r) { sum.x += parts[r * groups + g].x; sum.y += parts[r * groups + g].y; }
            all[g] = make_float2(sum.x / count, sum.y / count);
        }
        __syncthreads();
        // deltaX = scale dz + more (x - mean) + base
        float2 more[2], base[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const float2 d = all[gi[2 * j]], e = all[gi[2 * j + 1]];
            base[j] = neg2(mul2(rstd[j], make_float2(d.x, e.x)));
            more[j] = neg2(mul2(mul2(rstd[j], rstd[j]), make_float2(d.y, e.y)));
        }
        with_act(kKeepDz<T> ? ALPHA_ACT_NONE : p.act, [&](auto a) {
            constexpr int ACT = decltype(a)::value;
#pragma unroll 2
            for (int i = first; i < last; i += step) {
                float2 x[2], d[2];
                W::load(xs[i], x);
                W::load(ys[i], d);
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    x[j] = add2(x[j], mean[j]);
                    if (ACT != ALPHA_ACT_NONE) d[j] = mul2(d[j], norm_slope<ACT, kNormFast<T>>(fma2(x[j], scale[j], beta[j]), p.k));
                    x[j] = fma2(d[j], scale[j], fma2(x[j], more[j], base[j]));
                }
                *reinterpret_cast<Raw*>(out) = W::store(x);
                out += jump;
            }
        });
    }
}

// ---- streamed ---------------------------------------------------------------------------------------------------

// A thread's words of one or two tensors, row after row, U of them at a time.  Words of four elements come by asynchronous copies two batches ahead, through shared
// memory where each thread has places of its own (48 KB a CTA, four of them on an SM: a load into registers for each batch left HBM idle in between, 512 x 512 x 256 bf16
// 89 us instead of 84); single elements are loaded as they are used.
template <class T, int V, bool TWO> struct NormRows {
    using Raw = typename NormWord<T, V>::Raw;
    static constexpr int S = 3, U = (sizeof(T) == 2 ? 8 : 4) / (TWO ? 2 : 1);
    static constexpr size_t kBytes = V == 1 ? 0 : static_cast<size_t>(kNormThreads) * sizeof(Raw) * U * S * (TWO ? 2 : 1);
    const T *x, *y;
    long long step;                  // elements from a row to the thread's next
    int total;                       // its rows
    Raw* ring;
    __device__ Raw* at(int batch, int i, int second) const { return ring + ((batch % S * U + i) * (TWO ? 2 : 1) + second) * kNormThreads + threadIdx.x; }
    __device__ void issue(int batch) const
    {
        if constexpr (V != 1) {
            const int have = min(U, total - batch * U);
            const uint32_t to = smem_u32(at(batch, 0, 0));
            const T *fx = x + batch * U * step, *fy = y + batch * U * step;
            auto copy = [&](int i) {
                copy_async<sizeof(Raw)>(to + i * (TWO ? 2 : 1) * kNormThreads * sizeof(Raw), fx);
                fx += step;
                if (TWO) { copy_async<sizeof(Raw)>(to + (2 * i + 1) * kNormThreads * sizeof(Raw), fy); fy += step; }
            };
            if (have == U) {
#pragma unroll
                for (int i = 0; i < U; ++i) copy(i);
            } else {
                for (int i = 0; i < have; ++i) copy(i);
            }
            copies_commit();
        }
    }
    // f(word of x, word of y) for each row, a few at a time in the instruction stream (batches unrolled as a whole miss the instruction cache)
    template <class F> __device__ void rows(F&& f) const
    {
        if constexpr (V == 1) {
            each([&](int, int have, const Raw (&rx)[U], const Raw (&ry)[U]) {
#pragma unroll
                for (int i = 0; i < U; ++i)
                    if (i < have) f(rx[i], ry[i]);
            });
        } else {
            for (int b = 0; b < S - 1; ++b) issue(b);
            const int batches = (total + U - 1) / U;
            for (int b = 0; b < batches; ++b) {
                const int have = min(U, total - b * U);
                issue(b + S - 1);
                copies_wait<S - 1>();
                const Raw* from = at(b, 0, 0);
#pragma unroll 2
                for (int i = 0; i < have; ++i, from += (TWO ? 2 : 1) * kNormThreads) f(from[0], from[TWO ? kNormThreads : 0]);
            }
        }
    }
    // f(first row, rows, words of x, words of y) for each batch; rows < U: the last
    template <class F> __device__ void each(F&& f) const
    {
        if constexpr (V != 1)
            for (int b = 0; b < S - 1; ++b) issue(b);
        const int batches = (total + U - 1) / U;
        for (int b = 0; b < batches; ++b) {
            Raw rx[U], ry[U];
            const int have = min(U, total - b * U);
            if constexpr (V != 1) {
                issue(b + S - 1);
                copies_wait<S - 1>();
#pragma unroll
                for (int i = 0; i < U; ++i) { rx[i] = *at(b, i, 0); if (TWO) ry[i] = *at(b, i, 1); }
            } else {
#pragma unroll
                for (int i = 0; i < U; ++i) {
                    const long long o = (static_cast<long long>(b) * U + (i < have ? i : 0)) * step;
                    rx[i] = x[o];
                    if (TWO) ry[i] = y[o];
                }
            }
            f(b * U, have, rx, ry);
        }
    }
};

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
    using Rows = NormRows<T, V, BACK>;
    using Raw = typename Rows::Raw;
    constexpr int U = Rows::U, P = (V + 1) / 2;
    extern __shared__ __align__(128) uint8_t smem[];
    float* red = reinterpret_cast<float*>(smem);              // 2 V sums of each thread, over the ring when that has been read
    grid_dependency_wait();
    grid_dependency_trigger();
    const NormAt a = norm_at<V>(p, blockIdx.x);
    float2 s[P], q[P];
#pragma unroll
    for (int j = 0; j < P; ++j) s[j] = q[j] = make_float2(0.f, 0.f);
    if (a.busy && a.ty < a.count) {
        const size_t begin = a.from + static_cast<size_t>(a.ty) * p.C;
        const Rows rows{static_cast<const T*>(p.X) + begin, BACK ? static_cast<const T*>(p.dY) + begin : nullptr, static_cast<long long>(p.rows) * p.C, (a.count - a.ty + p.rows - 1) / p.rows,
                        reinterpret_cast<Raw*>(smem)};
        if constexpr (!BACK) {
            float seen = 0.f;                     // s: mean of what has been seen, q: its squared differences
            rows.each([&](int, int have, const Raw (&raw)[U], const Raw (&)[U]) {
                const float each = static_cast<float>(have), total = seen + each, weight = __fdividef(each, total), inverse = have == U ? 1.f / U : __fdividef(1.f, each);
                float2 m[P], d2[P];
#pragma unroll
                for (int j = 0; j < P; ++j) m[j] = d2[j] = make_float2(0.f, 0.f);
                auto pass = [&](auto whole) {
#pragma unroll
                    for (int i = 0; i < U; ++i) {
                        if (!decltype(whole)::value && i >= have) break;
                        float2 f[P];
                        W::load(raw[i], f);
#pragma unroll
                        for (int j = 0; j < P; ++j) m[j] = add2(m[j], f[j]);
                    }
#pragma unroll
                    for (int j = 0; j < P; ++j) m[j] = mul2(m[j], twice(-inverse));      // (the negated mean)
#pragma unroll
                    for (int i = 0; i < U; ++i) {
                        if (!decltype(whole)::value && i >= have) break;
                        float2 f[P];
                        W::load(raw[i], f);
#pragma unroll
                        for (int j = 0; j < P; ++j) {
                            const float2 d = add2(f[j], m[j]);
                            d2[j] = fma2(d, d, d2[j]);
                        }
                    }
                };
                if (have == U) pass(std::true_type{});
                else pass(std::false_type{});
                const float cross = seen * weight;
#pragma unroll
                for (int j = 0; j < P; ++j) {
                    const float2 d = neg2(add2(m[j], s[j]));
                    s[j] = fma2(d, twice(weight), s[j]);
                    q[j] = add2(q[j], fma2(mul2(d, d), twice(cross), d2[j]));
                }
                seen = total;
            });
        } else {
            float2 mean[P], rstd[P], gamma[P], beta[P];
            load_affine<T, V>(p, a.word * V, gamma, beta);
#pragma unroll
            for (int j = 0; j < P; ++j) {
                const size_t g = static_cast<size_t>(a.n) * p.G + (a.word * V + 2 * j) / p.D, h = static_cast<size_t>(a.n) * p.G + (a.word * V + 2 * j + (V > 1)) / p.D;
                mean[j] = neg2(make_float2(p.mean[g], p.mean[h]));
                rstd[j] = make_float2(p.rstd[g], p.rstd[h]);
                gamma[j] = mul2(gamma[j], rstd[j]);
            }
            with_act(p.act, [&](auto act) {
                constexpr int ACT = decltype(act)::value;
                rows.rows([&](const Raw& rx, const Raw& ry) {
                    float2 fx[P], fy[P];
                    W::load(rx, fx);
                    W::load(ry, fy);
#pragma unroll
                    for (int j = 0; j < P; ++j) {
                        fx[j] = add2(fx[j], mean[j]);
                        if (ACT != ALPHA_ACT_NONE) fy[j] = mul2(fy[j], norm_slope<ACT, kNormFast<T>>(fma2(fx[j], gamma[j], beta[j]), p.k));
                        s[j] = add2(s[j], fy[j]);
                        q[j] = fma2(fy[j], fx[j], q[j]);
                    }
                });
            });
#pragma unroll
            for (int j = 0; j < P; ++j) q[j] = mul2(q[j], rstd[j]);
        }
    }
    copies_done();
    __syncthreads();
#pragma unroll
    for (int j = 0; j < V; ++j) {
        red[j * kNormThreads + threadIdx.x] = j % 2 ? s[j / 2].y : s[j / 2].x;
        red[(V + j) * kNormThreads + threadIdx.x] = j % 2 ? q[j / 2].y : q[j / 2].x;
    }
    __syncthreads();
    const int per = !BACK && p.whole ? p.G : p.C;
    float2* to = p.partial + (static_cast<size_t>(a.n) * p.runs + a.run) * per;
    const int first = (a.word - (static_cast<int>(threadIdx.x) - a.ty * p.words)) * V, wide = min(p.words * V, p.C - first);
    const int rows = min(p.rows, a.count);
    // `share` threads, neighbouring lanes, add a channel's
    int shift = 0;
    while (shift < 5 && wide << (shift + 1) <= kNormThreads) ++shift;
    const int share = 1 << shift, lane = threadIdx.x & (share - 1);
    auto shared_sum = [&](float x) {
        for (int d = share / 2; d; d >>= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
        return x;
    };
    for (int c0 = 0; c0 < wide; c0 += kNormThreads >> shift) {
        const int c = c0 + static_cast<int>(threadIdx.x >> shift);
        float *ms = red + (c % V) * kNormThreads + c / V, *qs = ms + V * kNormThreads;
        const int mine = c < wide ? rows : 0;
        float sum = 0.f, squares = 0.f;
        if constexpr (BACK) {
            for (int r = lane; r < mine; r += share) { sum += ms[r * p.words]; squares += qs[r * p.words]; }
            sum = shared_sum(sum);
            squares = shared_sum(squares);
        } else {
            const int each = a.count / p.rows, left = a.count - each * p.rows;
            auto had = [&](int r) { return static_cast<float>(each + (r < left ? 1 : 0)); };
            for (int r = lane; r < mine; r += share) sum = fmaf(ms[r * p.words], had(r), sum);
            sum = shared_sum(sum) / static_cast<float>(a.count);
            for (int r = lane; r < mine; r += share) { const float d = ms[r * p.words] - sum; squares += fmaf(d * d, had(r), qs[r * p.words]); }
            squares = shared_sum(squares);
        }
        __syncwarp();
        if (c < wide && lane == 0) {
            if (!BACK && p.whole) { ms[0] = sum; qs[0] = squares; }
            else to[first + c] = make_float2(sum, squares);
        }
    }
    if (BACK || !p.whole) return;
    __syncthreads();
    // groups from their channels, a thread to a group (D is 64 * V at most)
    const float count = static_cast<float>(a.count);
    for (int g = threadIdx.x; g < wide / p.D; g += kNormThreads) {
        float sum = 0.f, squares = 0.f;
        for (int d = 0; d < p.D; ++d) { const int c = g * p.D + d; sum += red[(c % V) * kNormThreads + c / V]; }
        sum /= static_cast<float>(p.D);
        for (int d = 0; d < p.D; ++d) {
            const int c = g * p.D + d;
            const float e = red[(c % V) * kNormThreads + c / V] - sum;
            squares += fmaf(e * e, count, red[(V + c % V) * kNormThreads + c / V]);
        }
        to[first / p.D + g] = make_float2(sum, squares);
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
    const float count = static_cast<float>(p.R) * static_cast<float>(p.D);
    if constexpr (!BACK) {
        const int D = p.whole ? 1 : p.D, per = p.whole ? p.G : p.C, entries = p.runs * D;
        const float channels = static_cast<float>(p.whole ? p.D : 1);
        const float2* from = p.partial + static_cast<size_t>(n) * p.runs * per + g * D;
        float sum = 0.f, squares = 0.f;
#pragma unroll 4
        for (int i = threadIdx.x; i < entries; i += kJoinNormThreads) {
            const int run = i / D;
            sum = fmaf(from[static_cast<size_t>(run) * per + i - run * D].x, static_cast<float>(min(p.part, p.R - run * p.part)), sum);
        }
        const float mean = block_sum(sum, shared) * channels / count;
#pragma unroll 4
        for (int i = threadIdx.x; i < entries; i += kJoinNormThreads) {
            const int run = i / D;
            const float2 e = from[static_cast<size_t>(run) * per + i - run * D];
            const float d = e.x - mean;
            squares += fmaf(d * d, static_cast<float>(min(p.part, p.R - run * p.part)) * channels, e.y);
        }
        const float rstd = 1.f / sqrtf(block_sum(squares, shared) / count + p.eps);
        if (threadIdx.x == 0) {
            p.group[blockIdx.x] = make_float2(mean, rstd);
            if (p.mean) { p.mean[blockIdx.x] = mean; p.rstd[blockIdx.x] = rstd; }
        }
    } else {
        const float2* from = p.partial + static_cast<size_t>(n) * p.runs * p.C + g * p.D;
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
                p.sums[static_cast<size_t>(n) * p.C + c] = make_float2(a, b);     // (streamed: a row for each sample)
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
    using Rows = NormRows<T, V, BACK>;
    using Raw = typename Rows::Raw;
    constexpr int P = (V + 1) / 2;
    extern __shared__ __align__(128) uint8_t smem[];
    grid_dependency_wait();
    grid_dependency_trigger();
    const NormAt a = norm_at<V>(p, gridDim.x - 1 - blockIdx.x);
    if (!a.busy || a.ty >= a.count) return;
    float2 mean[P], gamma[P], beta[P], more[P], base[P];
    load_affine<T, V>(p, a.word * V, gamma, beta);
#pragma unroll
    for (int j = 0; j < P; ++j) {
        const size_t g = static_cast<size_t>(a.n) * p.G + (a.word * V + 2 * j) / p.D, h = static_cast<size_t>(a.n) * p.G + (a.word * V + 2 * j + (V > 1)) / p.D;
        const float2 t = p.group[g], u = p.group[h];
        if constexpr (BACK) {
            const float2 rstd = make_float2(p.rstd[g], p.rstd[h]);
            mean[j] = neg2(make_float2(p.mean[g], p.mean[h]));
            gamma[j] = mul2(gamma[j], rstd);
            base[j] = neg2(mul2(rstd, make_float2(t.x, u.x)));
            more[j] = neg2(mul2(mul2(rstd, rstd), make_float2(t.y, u.y)));
        } else {
            mean[j] = neg2(make_float2(t.x, u.x));
            gamma[j] = mul2(gamma[j], make_float2(t.y, u.y));
        }
    }
    // from the last row to the first
    const int total = (a.count - a.ty + p.rows - 1) / p.rows;
    const long long step = -static_cast<long long>(p.rows) * p.C;
    const size_t begin = a.from + (a.ty + static_cast<size_t>(total - 1) * p.rows) * p.C;
    const Rows rows{static_cast<const T*>(p.X) + begin, BACK ? static_cast<const T*>(p.dY) + begin : nullptr, step, total, reinterpret_cast<Raw*>(smem)};
    T* out = static_cast<T*>(p.out) + begin;
    with_act(p.act, [&](auto act) {
        constexpr int ACT = decltype(act)::value;
        rows.rows([&](const Raw& rx, const Raw& ry) {
            float2 f[P], fy[P];
            W::load(rx, f);
            if (BACK) W::load(ry, fy);
#pragma unroll
            for (int j = 0; j < P; ++j) {
                f[j] = add2(f[j], mean[j]);
                const float2 z = fma2(f[j], gamma[j], beta[j]);
                if constexpr (BACK) {
                    if (ACT != ALPHA_ACT_NONE) fy[j] = mul2(fy[j], norm_slope<ACT, kNormFast<T>>(z, p.k));
                    f[j] = fma2(fy[j], gamma[j], fma2(f[j], more[j], base[j]));
                } else {
                    f[j] = norm_value<ACT, kNormFast<T>>(z, p.k);
                }
            }
            *reinterpret_cast<Raw*>(out) = W::store(f);
            out += step;
        });
    });
}

// deltaGamma and deltaBeta: the sums of a channel over the samples (and the CTAs of their clusters), 32 rows of 32 threads.
constexpr int kAffineThreads = 1024;
template <class T>
__global__ void __launch_bounds__(kAffineThreads) norm_affine_kernel(const float2* __restrict__ sums, int rows, int C, void* dgamma, void* dbeta, int f32)
{
    __shared__ float2 red[32][33];
    grid_dependency_wait();
    grid_dependency_trigger();
    const int x = threadIdx.x & 31, y = threadIdx.x >> 5, c = blockIdx.x * 32 + x;
    float a = 0.f, b = 0.f;
    if (c < C)
#pragma unroll 4
        for (int n = y; n < rows; n += 32) { const float2 s = sums[static_cast<size_t>(n) * C + c]; a += s.x; b += s.y; }
    red[y][x] = make_float2(a, b);
    __syncthreads();
    // a warp to a channel
    const float2 s = red[x][y];
    a = warp_sum(s.x);
    b = warp_sum(s.y);
    const int mine = blockIdx.x * 32 + y;
    if (x || mine >= C) return;
    if (f32) { static_cast<float*>(dgamma)[mine] = b; static_cast<float*>(dbeta)[mine] = a; }
    else { static_cast<T*>(dgamma)[mine] = static_cast<T>(b); static_cast<T*>(dbeta)[mine] = static_cast<T>(a); }
}

}  // namespace alpha
