// A FullConnect layer over few rows (tokens of a serving program): Y = act(X W^T + b) + R, or the gated block.
//
// Bound: one read of W.  A warp owns two rows of W (glu: the gate and the up row of a unit), or a KS-th of their words, and
// streams them past L1 in 16-byte words, UNROLL of each row in flight per lane; X (R rows) is read again by every warp and stays in L1.
// Sums are fp32, two terms to an instruction (fma.rn.f32x2); lanes, and then the KS warps of a row, are added in a fixed order.
#pragma once
#include "fc_act.cuh"
#include "gemm_f32.cuh"

namespace alpha {

struct FcSmall {
    int rows, IC, OC, ks;          // ks: warps that share two rows of W (1, 2, 4, 8)
    int act; float k;
    const void *X, *W, *bias, *residual;
    void *Z, *Y;
};

// Two floats of a word of 16 (or 32) bits elements, as an f32x2 operand.
template <class T> __device__ __forceinline__ void word_pairs(const uint4& w, unsigned long long (&v)[Word16<T>::N / 2])
{
    float f[Word16<T>::N];
    Word16<T>::load(w, f);
#pragma unroll
    for (int i = 0; i < Word16<T>::N / 2; ++i) v[i] = pack2(f[2 * i], f[2 * i + 1]);
}
__device__ __forceinline__ uint4 load_streamed(const uint4* p)
{
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
template <class T> __device__ __forceinline__ float to_float(T x);
template <> __device__ __forceinline__ float to_float<float>(float x) { return x; }
template <> __device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
template <> __device__ __forceinline__ float to_float<__half>(__half x) { return __half2float(x); }
template <class T> __device__ __forceinline__ T from_float(float x);
template <> __device__ __forceinline__ float from_float<float>(float x) { return x; }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <> __device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }

template <class T, int R, bool GLU>
__global__ void __launch_bounds__(256) fc_small_kernel(const __grid_constant__ FcSmall p)
{
    constexpr int N = Word16<T>::N, UNROLL = R == 1 ? 4 : 2;
    __shared__ float part[8][2 * R];
    grid_dependency_wait();
    grid_dependency_trigger();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, teams = 8 / p.ks;
    const int words = p.IC / N, units = GLU ? p.OC : (p.OC + 1) / 2;
    const int unit = blockIdx.x * teams + warp / p.ks, slice = warp % p.ks;
    float sums[2][R];
#pragma unroll
    for (int r = 0; r < R; ++r) sums[0][r] = sums[1][r] = 0.f;
    if (unit < units) {
        // (an odd last row of W is read twice)
        const int row0 = GLU ? unit : 2 * unit, row1 = GLU ? unit + p.OC : (2 * unit + 1 < p.OC ? 2 * unit + 1 : 2 * unit);
        const uint4* w0 = reinterpret_cast<const uint4*>(p.W) + static_cast<size_t>(row0) * words;
        const uint4* w1 = reinterpret_cast<const uint4*>(p.W) + static_cast<size_t>(row1) * words;
        const uint4* x = reinterpret_cast<const uint4*>(p.X);
        const int each = (words + p.ks - 1) / p.ks, begin = slice * each, end = begin + each < words ? begin + each : words;
        unsigned long long acc[2][R];
#pragma unroll
        for (int r = 0; r < R; ++r) acc[0][r] = acc[1][r] = 0ull;
        auto madd = [&](const uint4& a, const uint4& b, int at) {
            unsigned long long v0[N / 2], v1[N / 2];
            word_pairs<T>(a, v0);
            word_pairs<T>(b, v1);
#pragma unroll
            for (int r = 0; r < R; ++r) {
                if (R > 1 && r >= p.rows) break;
                unsigned long long xv[N / 2];
                word_pairs<T>(__ldg(x + static_cast<size_t>(r) * words + at), xv);
#pragma unroll
                for (int i = 0; i < N / 2; ++i) { ffma2(acc[0][r], v0[i], xv[i]); ffma2(acc[1][r], v1[i], xv[i]); }
            }
        };
        int at = begin + lane;
        for (; at + 32 * (UNROLL - 1) < end; at += 32 * UNROLL) {
            uint4 a[UNROLL], b[UNROLL];
#pragma unroll
            for (int u = 0; u < UNROLL; ++u) { a[u] = load_streamed(w0 + at + 32 * u); b[u] = load_streamed(w1 + at + 32 * u); }
#pragma unroll
            for (int u = 0; u < UNROLL; ++u) madd(a[u], b[u], at + 32 * u);
        }
        for (; at < end; at += 32) madd(load_streamed(w0 + at), load_streamed(w1 + at), at);
#pragma unroll
        for (int o = 0; o < 2; ++o)
#pragma unroll
            for (int r = 0; r < R; ++r) {
                float a, b;
                unpack2(acc[o][r], a, b);
                float s = a + b;
#pragma unroll
                for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
                sums[o][r] = s;
            }
    }
    if (lane == 0) {
#pragma unroll
        for (int r = 0; r < R; ++r) { part[warp][r] = sums[0][r]; part[warp][R + r] = sums[1][r]; }
    }
    __syncthreads();
    // a thread per output: (team, row of X) and, without gates, which of the two
    constexpr int PER = GLU ? R : 2 * R;
    if (threadIdx.x >= teams * PER) return;
    const int team = threadIdx.x / PER, q = threadIdx.x % PER, r = q % R, u = blockIdx.x * teams + team;
    const int col = GLU ? u : 2 * u + q / R;
    if (u >= units || r >= p.rows || col >= p.OC) return;
    float z = 0.f, up = 0.f;
    for (int s = 0; s < p.ks; ++s) {
        z += part[team * p.ks + s][q];
        if (GLU) up += part[team * p.ks + s][R + r];
    }
    const T* bias = static_cast<const T*>(p.bias);
    T *Z = static_cast<T*>(p.Z), *Y = static_cast<T*>(p.Y);
    const size_t at = static_cast<size_t>(r) * p.OC + col;
    if (bias) z += to_float(bias[col]);
    if (GLU && bias) up += to_float(bias[p.OC + col]);
    if (Z) {
        Z[GLU ? at + static_cast<size_t>(r) * p.OC : at] = from_float<T>(z);
        if (GLU) Z[at + static_cast<size_t>(r + 1) * p.OC] = from_float<T>(up);
    }
    with_act(p.act, [&](auto a) { z = act_value<decltype(a)::value, Word16<T>::kFast>(z, p.k); });
    if (GLU) z *= up;
    else if (p.residual) z += to_float(static_cast<const T*>(p.residual)[at]);
    Y[at] = from_float<T>(z);
}

}  // namespace alpha
