// From deltaY to the gradient of a layer's sums, and the gradient of its bias.
//
//   fc    dZ = deltaY act'(Z)                                   deltaB = column sums of dZ
//   glu   dG = deltaY U act'(G),  dU = deltaY act(G)            Z = [G | U], dZ = [dG | dU]
// One pass at HBM speed: a lane holds 16 bytes of columns, a warp 512 consecutive bytes of a row, the eight warps of a CTA every eighth of its
// rows.  deltaZ is rounded to the tensors' type, because the tensor cores read it as an operand; the column sums are fp32 sums of what it was before, first
// down a warp's rows, then over the warps, and the partial rows of the CTAs are added by a second launch, all in a fixed order.
// deltaZ may be Z itself: an element is read before it is written, by the same thread.
#pragma once
#include "fc_act.cuh"
#include "dependent_launch.cuh"

namespace alpha {

struct FcDelta {
    long long rows;
    int cols, OC;                   // columns of a half with their padding, and without: deltaZ's padding is zeros
    int act; float k;
    const void *dY, *Z;
    void* dZ;                       // nullptr: column sums only (no activation)
    float* part;                    // [gridDim.y][cols, glu: 2 cols] or nullptr
};

// CTAs of an SM, each warp with one row in flight: rows ahead in registers, or the loop unrolled, cost more than they hid, as the grid then no longer
// sweeps one band of rows.  us with deltaB, before with two or four rows ahead on three CTAs / now: 8192 x 11008 glu silu 182 / 151, 4096 x 16384 silu 109 / 84
// and leakyRelu 87 / 66 (5.1 and 6.1 TB/s: an exponential and a quotient an element), fp32 4096 x 16384 165 / 125.
// Layers of few columns leave lanes idle, and take what 128 columns take: 65536 rows fp32 silu with deltaB, 10 columns 17, 128 20 (101 MB), 512 66.
template <bool GLU> __host__ __device__ constexpr int delta_ctas() { return GLU ? 3 : 6; }
template <class T, bool GLU>
__global__ void __launch_bounds__(256, delta_ctas<GLU>()) fc_delta_kernel(const __grid_constant__ FcDelta p)
{
    using V = Word16<T>;
    constexpr int N = V::N, HALVES = GLU ? 2 : 1;
    __shared__ float sums[8][HALVES][32 * N];
    grid_dependency_wait();
    grid_dependency_trigger();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, words = p.cols / N, word = blockIdx.x * 32 + lane;
    const uint4 *dY = static_cast<const uint4*>(p.dY), *Z = static_cast<const uint4*>(p.Z);
    uint4* dZ = static_cast<uint4*>(p.dZ);
    const int whole = p.OC - word * N;                                   // columns of the lane's word that are not padding
    float acc[HALVES][N];
#pragma unroll
    for (int i = 0; i < N; ++i)
        for (int h = 0; h < HALVES; ++h) acc[h][i] = 0.f;
    if (word < words) {
        with_act(p.act, [&](auto a) {
            constexpr int ACT = decltype(a)::value;
#pragma unroll 1
            for (long long r = blockIdx.y * 8 + warp; r < p.rows; r += gridDim.y * 8) {
                const size_t at = static_cast<size_t>(r) * words + word, zt = GLU ? at + static_cast<size_t>(r) * words : at;
                const uint4 wd = __ldg(dY + at);
                uint4 wz[HALVES];
                if constexpr (GLU || ACT != ALPHA_ACT_NONE) wz[0] = Z[zt];
                if constexpr (GLU) wz[HALVES - 1] = Z[zt + words];
                float d[N];
                V::load(wd, d);
                if constexpr (GLU) {
                    float g[N], u[N];
                    V::load(wz[0], g);
                    V::load(wz[HALVES - 1], u);
#pragma unroll
                    for (int i = 0; i < N; ++i) {
                        float value, slope;
                        act_both<ACT, V::kFast>(g[i], p.k, value, slope);
                        g[i] = d[i] * u[i] * slope;
                        u[i] = d[i] * value;
                        if (i >= whole) g[i] = u[i] = 0.f;
                        acc[0][i] += g[i];
                        acc[1][i] += u[i];
                    }
                    dZ[zt] = V::store(g);
                    dZ[zt + words] = V::store(u);
                } else {
                    if constexpr (ACT != ALPHA_ACT_NONE) {
                        float z[N];
                        V::load(wz[0], z);
#pragma unroll
                        for (int i = 0; i < N; ++i) {
                            float value, slope;
                            act_both<ACT, V::kFast>(z[i], p.k, value, slope);
                            d[i] = i >= whole ? 0.f : d[i] * slope;
                        }
                        dZ[zt] = V::store(d);
                    }
#pragma unroll
                    for (int i = 0; i < N; ++i) acc[0][i] += d[i];
                }
            }
        });
    }
    if (!p.part) return;
#pragma unroll
    for (int h = 0; h < HALVES; ++h)
#pragma unroll
        for (int i = 0; i < N; ++i) sums[warp][h][lane * N + i] = acc[h][i];
    __syncthreads();
    for (int e = threadIdx.x; e < HALVES * 32 * N; e += 256) {
        const int h = e / (32 * N), c = e % (32 * N), col = blockIdx.x * 32 * N + c;
        if (col >= p.cols) continue;
        float s = 0.f;
#pragma unroll
        for (int w = 0; w < 8; ++w) s += sums[w][h][c];
        p.part[static_cast<size_t>(blockIdx.y) * (HALVES * p.cols) + h * p.cols + col] = s;
    }
}

// deltaB[c] = sum of the partial rows: 32 columns a CTA, a warp every eighth row.
template <class T>
__global__ void __launch_bounds__(256) fc_bias_kernel(const float* __restrict__ part, int rows, int cols, T* __restrict__ deltaB)
{
    __shared__ float sums[8][32];
    grid_dependency_wait();
    grid_dependency_trigger();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, col = blockIdx.x * 32 + lane;
    float s = 0.f;
    if (col < cols)
#pragma unroll 8
        for (int r = warp; r < rows; r += 8) s += part[static_cast<size_t>(r) * cols + col];
    sums[warp][lane] = s;
    __syncthreads();
    if (warp || col >= cols) return;
    s = 0.f;
#pragma unroll
    for (int w = 0; w < 8; ++w) s += sums[w][lane];
    if constexpr (sizeof(T) == 4) deltaB[col] = s;
    else if constexpr (std::is_same<T, __half>::value) deltaB[col] = __float2half_rn(s);
    else deltaB[col] = __float2bfloat16_rn(s);
}

}  // namespace alpha
