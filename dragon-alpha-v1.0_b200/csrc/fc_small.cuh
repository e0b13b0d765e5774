// A FullConnect layer over few rows (tokens of a serving program): Y = act(X W^T + b) + R, or the gated block; first fp32, 16-bit tensors below.
//
// Bound: one read of W.  A warp owns two rows of W (glu: the gate and the up row of a unit), or a KS-th of their words, and
// streams them past L1 in 16-byte words, UNROLL of each row in flight per lane; X (R rows) is read again by every warp and stays in L1.
// Sums are fp32, two terms to an instruction (fma.rn.f32x2); lanes, and then the KS warps of a row, are added in a fixed order.
#pragma once
#include "fc_act.cuh"
#include "gemm_f32.cuh"
#include "sm100_ptx.cuh"

namespace alpha {

struct FcSmall {
    int rows, IC, OC, pitch, ks;   // pitch: of Y and R, and of either half of Z and the bias; ks: warps of a CTA that share two rows of W, or a row group (1, 2, 4, 8)
    int split;                     // CTAs of a cluster that share a row group (16-bit)
    int act; float k;
    const void *X, *W, *bias, *residual;
    void *Z, *Y;
};

__device__ __forceinline__ uint4 load_streamed(const uint4* p)
{
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.L2::256B.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
// 32 bytes: with four lanes to a row of an operand a whole 128-byte line.
__device__ __forceinline__ void load_streamed_32(const uint4* p, uint4 (&v)[2])
{
    asm volatile("ld.global.nc.L1::no_allocate.L2::256B.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(v[0].x), "=r"(v[0].y), "=r"(v[0].z), "=r"(v[0].w), "=r"(v[1].x), "=r"(v[1].y), "=r"(v[1].z), "=r"(v[1].w) : "l"(p));
}
template <class T> __device__ __forceinline__ float to_float(T x);
template <> __device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
template <> __device__ __forceinline__ float to_float<__half>(__half x) { return __half2float(x); }
template <class T> __device__ __forceinline__ T from_float(float x);
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <> __device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }

template <int R, bool GLU>
__global__ void __launch_bounds__(256) fc_small_kernel(const __grid_constant__ FcSmall p)
{
    constexpr int N = 4, UNROLL = R == 1 ? 4 : 2;
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
            auto two = [](uint32_t lo, uint32_t hi) { return pack2(__uint_as_float(lo), __uint_as_float(hi)); };
            const unsigned long long a0 = two(a.x, a.y), a1 = two(a.z, a.w), b0 = two(b.x, b.y), b1 = two(b.z, b.w);
#pragma unroll
            for (int r = 0; r < R; ++r) {
                if (R > 1 && r >= p.rows) break;
                const uint4 v = __ldg(x + static_cast<size_t>(r) * words + at);
                const unsigned long long x0 = two(v.x, v.y), x1 = two(v.z, v.w);
                ffma2(acc[0][r], a0, x0); ffma2(acc[1][r], b0, x0);
                ffma2(acc[0][r], a1, x1); ffma2(acc[1][r], b1, x1);
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
    const float* bias = static_cast<const float*>(p.bias);
    float *Z = static_cast<float*>(p.Z), *Y = static_cast<float*>(p.Y);
    const size_t at = static_cast<size_t>(r) * p.pitch + col;
    if (bias) z += bias[col];
    if (GLU && bias) up += bias[p.pitch + col];
    if (Z) {
        Z[GLU ? at + static_cast<size_t>(r) * p.pitch : at] = z;
        if (GLU) Z[at + static_cast<size_t>(r + 1) * p.pitch] = up;
    }
    with_act(p.act, [&](auto a) { z = act_value<decltype(a)::value, false>(z, p.k); });
    if (GLU) z *= up;
    else if (p.residual) z += static_cast<const float*>(p.residual)[at];
    Y[at] = z;
}

// ---- 16-bit tensors ----------------------------------------------------------------------------------------------
//
// The same over up to 8 NT rows, with the multiplications of a warp's 16 rows of W by 8 rows of X and 16 steps one mma.sync: no FMA, conversion or
// reduction over lanes is left, so that the kernel is bound by the stream of W for every row count (by FMAs four rows of X took 52 us for 180 MB of W).
// tcgen05 would want W staged in shared memory for 128 x 8 outputs a CTA; here a warp's operand goes from memory to its registers.
// The order of the reduction is free as long as both operands follow it: of 32 steps lane (g, t) holds eight consecutive ones of rows g and
// g + 8 of W and of row g of X, 32 bytes of W a load, and the first four of them are steps 2 t, 2 t + 1, 2 t + 8, 2 t + 9 of one
// instruction, the others of a second.  glu: the rows of W are 16 gate rows and 16 up rows.
// us for W from DRAM, 1 / 8 / 16 rows (5.6 TB/s besides 2.5 us of a launch): 4096 x 11008 19 / 20 / 22, glu 2 x 11008 x 4096 35 / 36 / 39, 4096 x 4096 9.4 / 9.7 / 11; with 16-byte
// loads, half a line to a row, 23.5 for the first.  Where row groups leave SMs to fill (256 groups, 148 SMs) clusters of
// CTAs share them and add up through distributed shared memory: 21 -> 19.  Sums are added in a fixed order, warps and then CTAs.
template <class T> __device__ __forceinline__ void mma_16x8x16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1);
template <> __device__ __forceinline__ void mma_16x8x16<__nv_bfloat16>(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1)
{
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <> __device__ __forceinline__ void mma_16x8x16<__half>(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1)
{
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

template <class T, int NT, bool GLU>
__global__ void __launch_bounds__(256) fc_token_kernel(const __grid_constant__ FcSmall p)
{
    constexpr int MT = GLU ? 2 : 1, UNROLL = (GLU ? 2 : 4) / NT, COLS = 8 * NT;
    __shared__ float part[8][MT][16][COLS + 1];
    const int rank = p.split > 1 ? static_cast<int>(cluster_ctarank()) : 0, block = blockIdx.x / p.split;
    grid_dependency_wait();
    grid_dependency_trigger();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, teams = 8 / p.ks;
    const int words = p.IC / 8, groups = (p.OC + 15) / 16;
    const int group = block * teams + warp / p.ks, slices = p.split * p.ks, slice = rank * p.ks + warp % p.ks;
    if (group < groups) {
        // (rows past the last are read as the last, and not stored)
        const uint4 *w[MT][2], *x[NT];
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int row = group * 16 + g + 8 * h;
                w[m][h] = static_cast<const uint4*>(p.W) + (static_cast<size_t>(m) * p.OC + (row < p.OC ? row : p.OC - 1)) * words;
            }
#pragma unroll
        for (int n = 0; n < NT; ++n) x[n] = static_cast<const uint4*>(p.X) + static_cast<size_t>(8 * n + g < p.rows ? 8 * n + g : p.rows - 1) * words;
        float acc[MT][NT][4] = {};
        // the warps of a group take UNROLL blocks of 64 steps in turn: together they walk along whole DRAM pages of their rows
        const int blocks = (words + 7) / 8;
        auto multiply = [&](const uint4 (&a)[MT][2][2], const uint4 (&b)[NT][2]) {
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int m = 0; m < MT; ++m)
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        mma_16x8x16<T>(acc[m][n], a[m][0][j].x, a[m][1][j].x, a[m][0][j].y, a[m][1][j].y, b[n][j].x, b[n][j].y);
                        mma_16x8x16<T>(acc[m][n], a[m][0][j].z, a[m][1][j].z, a[m][0][j].w, a[m][1][j].w, b[n][j].z, b[n][j].w);
                    }
        };
        int k = slice * UNROLL;
        if (words % 2 == 0 && (reinterpret_cast<uintptr_t>(p.W) & 31) == 0) {           // (rows of whole, aligned 32-byte words)
            for (; 8 * (k + UNROLL) <= words; k += UNROLL * slices) {
                uint4 a[UNROLL][MT][2][2], b[UNROLL][NT][2];
#pragma unroll
                for (int u = 0; u < UNROLL; ++u) {
                    const int at = 8 * (k + u) + 2 * t;
#pragma unroll
                    for (int m = 0; m < MT; ++m) { load_streamed_32(w[m][0] + at, a[u][m][0]); load_streamed_32(w[m][1] + at, a[u][m][1]); }
#pragma unroll
                    for (int n = 0; n < NT; ++n) { b[u][n][0] = __ldg(x[n] + at); b[u][n][1] = __ldg(x[n] + at + 1); }
                }
#pragma unroll
                for (int u = 0; u < UNROLL; ++u) multiply(a[u], b[u]);
            }
        }
        for (; k < blocks; k += UNROLL * slices) {
            for (int q = k; q < k + UNROLL && q < blocks; ++q) {
                uint4 a[MT][2][2], b[NT][2];
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const int at = 8 * q + 2 * t + j;
                    const bool in = at < words;
#pragma unroll
                    for (int m = 0; m < MT; ++m)
#pragma unroll
                        for (int h = 0; h < 2; ++h) a[m][h][j] = in ? load_streamed(w[m][h] + at) : make_uint4(0, 0, 0, 0);
#pragma unroll
                    for (int n = 0; n < NT; ++n) b[n][j] = in ? __ldg(x[n] + at) : make_uint4(0, 0, 0, 0);
                }
                multiply(a, b);
            }
        }
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) part[warp][m][g + 8 * (i >> 1)][8 * n + 2 * t + (i & 1)] = acc[m][n][i];
    }
    __syncthreads();
    if (p.split > 1) {
        // the sums of this CTA into its first rows, then those of the cluster's CTAs, a share of the outputs each
        constexpr int SUMS = MT * 16 * COLS;
        float mine[SUMS / 256 + 1];
        for (int team = 0; team < teams; ++team) {
            int i = 0;
            for (int e = threadIdx.x; e < SUMS; e += 256, ++i) {
                const int m = e / (16 * COLS), o = e / COLS % 16, r = e % COLS;
                float v = 0.f;
                for (int q = 0; q < p.ks; ++q) v += part[team * p.ks + q][m][o][r];
                mine[i] = v;
            }
            __syncthreads();
            i = 0;
            for (int e = threadIdx.x; e < SUMS; e += 256, ++i) part[team * p.ks][e / (16 * COLS)][e / COLS % 16][e % COLS] = mine[i];
        }
        cluster_sync_all();
    }
    const int per = p.split > 1 ? 1 : p.ks;
    auto sum = [&](int team, int m, int o, int r) {
        float v = 0.f;
        if (p.split > 1) {
            const uint32_t at = smem_u32(&part[team * p.ks][m][o][r]);
            for (int q = 0; q < p.split; ++q) v += ld_shared_cluster(mapa_u32(at, q));
        } else {
            for (int q = 0; q < per; ++q) v += part[team * per + q][m][o][r];
        }
        return v;
    };
    const T *bias = static_cast<const T*>(p.bias), *residual = static_cast<const T*>(p.residual);
    T *Z = static_cast<T*>(p.Z), *Y = static_cast<T*>(p.Y);
    for (int e = rank * 256 + threadIdx.x; e < teams * 16 * COLS; e += 256 * p.split) {
        const int o = e & 15, r = (e >> 4) % COLS, team = e / (16 * COLS), col = (block * teams + team) * 16 + o;
        if (r >= p.rows || col >= p.OC) continue;
        float z = sum(team, 0, o, r), up = GLU ? sum(team, MT - 1, o, r) : 0.f;
        const size_t at = static_cast<size_t>(r) * p.pitch + col;
        if (bias) z += to_float(bias[col]);
        if (GLU && bias) up += to_float(bias[p.pitch + col]);
        if (Z) {
            Z[GLU ? at + static_cast<size_t>(r) * p.pitch : at] = from_float<T>(z);
            if (GLU) Z[at + static_cast<size_t>(r + 1) * p.pitch] = from_float<T>(up);
        }
        with_act(p.act, [&](auto a) { z = act_value<decltype(a)::value, true>(z, p.k); });
        if (GLU) z *= up;
        else if (residual) z += to_float(residual[at]);
        Y[at] = from_float<T>(z);
    }
    if (p.split > 1) cluster_sync_all();   // no CTA leaves while another may still read its shared memory
}

}  // namespace alpha
