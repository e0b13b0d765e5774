// Products of 16-bit matrices on the tensor cores with the epilogue of a FullConnect layer.
//
//   D[m][n] = sum_k A[m][k] B[n][k]        fp32 sums in tensor memory
//   plain / fc:   z = D + bias[n],  Y = act(z) + R,  Z = z where it is kept for the backward pass
//   glu:          B holds gate rows and up rows; g and u the two sums of a unit, Y = act(g) u, Z = [g | u]
// Forward A = X, B = W; deltaX A = dZ, B = W read along its rows (MN-major); deltaW A = dZ, B = X, both MN-major.  Either operand's memory
// may run along k (a box of 64 steps x rows, 128-byte rows) or along its rows (boxes of 64 rows x 64 steps): the MMA's descriptors take both,
// so nothing is transposed.  What a box reads past a matrix is zeros and past a half of W belongs to columns that are not stored.
//
// PAIR: two CTAs of a cluster form 256 x BN outputs (tcgen05 cta_group::2): each holds its 128 rows of A and half of the rows of B, so that
// shared memory is read and filled with half of B.  Otherwise a CTA forms 128 x BN.  Persistent: a CTA (pair) walks over tiles, in groups of
// kGroupM row tiles so that the tiles in flight share rows of A and B in L2; accumulators alternate between two halves of tensor memory, so that
// the epilogue of a tile runs beside the MMAs of the next.
// Warps: 0 TMA producer, 1 MMA issuer, 2-9 epilogue (two per quarter of the lanes, chunks of 32 columns in turn).
#pragma once
#include "fc_act.cuh"
#include "sm100_ptx.cuh"

namespace alpha {

constexpr int kFcThreads = 320, kFcBK = 64, kFcGroupM = 8;
template <bool PAIR, int BN> struct FcTile {
    static constexpr int BR = PAIR ? BN / 2 : BN;                       // rows of B in a CTA
    static constexpr uint32_t kA = 128 * 128, kB = BR * 128, kStage = kA + kB;
    static constexpr int kStages = 196608 / kStage > 8 ? 8 : 196608 / kStage;
    static constexpr uint32_t kStaging = 8 * 4096;                      // two boxes of 32 x 32 elements for each epilogue warp
    static constexpr uint32_t kSmem = kStages * kStage + kStaging + 1024 + 256;
    static constexpr uint32_t kTmem = 2 * BN;
};

struct FcMma {
    int rows, cols, K;            // outputs (glu: columns of a half), reduction
    int m_tiles, n_tiles, kb;     // tiles, blocks of 64 steps
    int a_mn, b_mn, a_rows;       // operands that run along their rows; rows of a box of A that runs along k
    int b_up;                     // glu: first row of the up half of B
    uint32_t idesc;
    int act, keep_z; float k;
    const void *bias, *residual;
    int* status;
};

template <class T, bool PAIR, int BN, bool GLU>
__global__ void __launch_bounds__(kFcThreads, 1)
    fc_mma_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const __grid_constant__ CUtensorMap tmY,
                  const __grid_constant__ CUtensorMap tmZ, const __grid_constant__ FcMma p)
{
    using G = FcTile<PAIR, BN>;
    constexpr int CTAS = PAIR ? 2 : 1, OUT = GLU ? BN / 2 : BN, S = G::kStages;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S * G::kStage + G::kStaging);
    uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(bars + 2 * S + 4);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = PAIR ? cluster_ctarank() : 0u;
    const uint32_t full_a = smem_u32(bars), empty_a = full_a + 8 * S, afull_a = empty_a + 8 * S, aempty_a = afull_a + 16;

    if (threadIdx.x == 0) {
        for (int i = 0; i < S; ++i) { mbar_init(&bars[i], 1); mbar_init(&bars[S + i], 1); }
        for (int i = 0; i < 2; ++i) { mbar_init(&bars[2 * S + i], 1); mbar_init(&bars[2 * S + 2 + i], 8 * CTAS); }
        fence_barrier_init();
        prefetch_tmap(&tmA); prefetch_tmap(&tmB); prefetch_tmap(&tmY);
        if (p.keep_z) prefetch_tmap(&tmZ);
    }
    if (warp == 1) {
        if constexpr (PAIR) { tmem_alloc_pair(tmem_holder, G::kTmem); tmem_relinquish_pair(); }
        else { tmem_alloc(tmem_holder, G::kTmem); tmem_relinquish(); }
    }
    tc_fence_before_sync();
    grid_dependency_wait();
    __syncthreads();
    if constexpr (PAIR) cluster_sync_all();   // the peer's barriers are initialised before anything reaches them
    grid_dependency_trigger();
    tc_fence_after_sync();
    const uint32_t tmem_base = *tmem_holder;

    const int total = p.m_tiles * p.n_tiles, step = gridDim.x / CTAS, first = blockIdx.x / CTAS;
    auto tile_at = [&](int t, int& m0, int& n0) {
        const int per = kFcGroupM * p.n_tiles, g = t / per, r = t - g * per, left = p.m_tiles - g * kFcGroupM, rows = left < kFcGroupM ? left : kFcGroupM;
        const int n = r / rows;
        m0 = (g * kFcGroupM + r - n * rows) * (128 * CTAS) + static_cast<int>(rank) * 128;
        n0 = n * OUT;
    };
    const uint32_t smem_a = smem_u32(smem);

    if (warp == 0) {
        if (lane == 0) {
            const uint32_t full_L = PAIR ? mapa_u32(full_a, 0) : full_a;
            const uint32_t tx = CTAS * ((p.a_mn ? G::kA : static_cast<uint32_t>(p.a_rows) * 128) + G::kB);
            auto load = [&](uint32_t dst, const CUtensorMap* m, uint32_t bar, int c0, int c1) {
                if constexpr (PAIR) tma_load_2d_pair(dst, m, bar, c0, c1);
                else tma_load_2d_a(dst, m, bar, c0, c1);
            };
            RingPos rp;
            bool ok = true;
            for (int t = first; t < total && ok; t += step) {
                int m0, n0;
                tile_at(t, m0, n0);
                for (int kb = 0; kb < p.kb; ++kb) {
                    if (!mbar_wait_a(empty_a + 8 * rp.idx, rp.phase ^ 1)) { report(p.status, kStatusProducerTimeout); settle(); ok = false; break; }
                    if (rank == 0) mbar_arrive_expect_tx_a(full_a + 8 * rp.idx, tx);
                    const uint32_t bar = full_L + 8 * rp.idx, a = smem_a + rp.idx * G::kStage, b = a + G::kA;
                    const int k0 = kb * kFcBK;
                    if (p.a_mn) {
#pragma unroll
                        for (int j = 0; j < 2; ++j) load(a + j * 8192, &tmA, bar, m0 + 64 * j, k0);
                    } else {
                        load(a, &tmA, bar, k0, m0);
                    }
                    if constexpr (GLU) {
                        // columns [gate | up] of the accumulator
                        if constexpr (PAIR) load(b, &tmB, bar, k0, n0 + (rank ? p.b_up : 0));
                        else { load(b, &tmB, bar, k0, n0); load(b + G::kB / 2, &tmB, bar, k0, n0 + p.b_up); }
                    } else {
                        const int b0 = n0 + static_cast<int>(rank) * G::BR;
                        if (p.b_mn) {
#pragma unroll
                            for (int j = 0; j < G::BR / 64; ++j) load(b + j * 8192, &tmB, bar, b0 + 64 * j, k0);
                        } else {
                            load(b, &tmB, bar, k0, b0);
                        }
                    }
                    rp.advance(S);
                }
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        if (lane == 0 && rank == 0) {
            constexpr uint32_t dhi = (1024u >> 4) | (1u << 14) | (static_cast<uint32_t>(kSwizzle128B) << 29);
            const uint32_t a_k = p.a_mn ? 128u : 2u, b_k = p.b_mn ? 128u : 2u;               // 16 steps further, in 16-byte units
            const uint32_t a_lo0 = smem_desc_lo(smem_a, p.a_mn ? 8192u : 16u), b_lo0 = smem_desc_lo(smem_a + G::kA, p.b_mn ? 8192u : 16u);
            const uint32_t empty_1 = PAIR ? mapa_u32(empty_a, 1) : 0u, afull_1 = PAIR ? mapa_u32(afull_a, 1) : 0u;
            const uint32_t empty_0 = PAIR ? mapa_u32(empty_a, 0) : empty_a, afull_0 = PAIR ? mapa_u32(afull_a, 0) : afull_a;
            auto commit = [&](uint32_t mine, uint32_t peer) {
                if constexpr (PAIR) { mma_commit_pair(mine); mma_commit_pair(peer); }
                else mma_commit_a(mine);
            };
            auto wait = [&](uint32_t bar, uint32_t parity) {
                if (PAIR ? mbar_wait_cluster_a(bar, parity) : mbar_wait_a(bar, parity)) return true;
                report(p.status, kStatusMmaTimeout);
                settle();
                return false;
            };
            RingPos rp, ap;
            bool ok = true;
            for (int t = first; t < total && ok; t += step) {
                if (!wait(aempty_a + 8 * ap.idx, ap.phase ^ 1)) break;
                tc_fence_after_sync();
                const uint32_t d = tmem_base + ap.idx * BN;
                for (int kb = 0; kb < p.kb; ++kb) {
                    if (!wait(full_a + 8 * rp.idx, rp.phase)) { ok = false; break; }
                    tc_fence_after_sync();
                    const uint32_t a = a_lo0 + rp.idx * (G::kStage >> 4), b = b_lo0 + rp.idx * (G::kStage >> 4);
#pragma unroll
                    for (uint32_t kk = 0; kk < 4; ++kk) mma_16bit<PAIR>(d, a + kk * a_k, dhi, b + kk * b_k, dhi, p.idesc, (kb | kk) ? 1u : 0u);
                    commit(empty_0 + 8 * rp.idx, empty_1 + 8 * rp.idx);
                    rp.advance(S);
                }
                commit(afull_0 + 8 * ap.idx, afull_1 + 8 * ap.idx);
                ap.advance(2);
            }
        }
        __syncwarp();
    } else {
        const int quad = warp & 3, half = (warp - 2) >> 2;
        const uint32_t lanes = tmem_base + (static_cast<uint32_t>(quad * 32) << 16);
        const uint32_t stage_a = smem_a + S * G::kStage + (warp - 2) * 4096, aempty_L = PAIR ? mapa_u32(aempty_a, 0) : aempty_a;
        const T* bias = static_cast<const T*>(p.bias);
        const T* residual = static_cast<const T*>(p.residual);
        uint32_t sbuf = 0;
        // A lane's 32 columns leave through shared memory as a box of 32 rows x 64 bytes.
        auto put = [&](const float (&f)[32], auto&& store) {
            if (lane == 0) tma_store_wait_read<1>();
            __syncwarp();
            const uint32_t buf = stage_a + sbuf * 2048;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const uint4 w = Word16<T>::store(f + 8 * q);
                st_shared_v4(buf + lane * 64 + ((q ^ ((lane >> 1) & 3)) << 4), make_float4(__uint_as_float(w.x), __uint_as_float(w.y), __uint_as_float(w.z), __uint_as_float(w.w)));
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) { store(buf); tma_store_commit(); }
            sbuf ^= 1u;
        };
        // f += 32 columns of a vector or a row (its width a multiple of 8; R may be Y itself, so not by the read-only path)
        auto add = [&](float (&f)[32], const T* from, int col0) {
#pragma unroll
            for (int q = 0; q < 4; ++q)
                if (col0 + 8 * q < p.cols) {
                    float b[8];
                    Word16<T>::load(*reinterpret_cast<const uint4*>(from + col0 + 8 * q), b);
#pragma unroll
                    for (int i = 0; i < 8; ++i) f[8 * q + i] += b[i];
                }
        };
        auto load32 = [&](uint32_t at, float (&f)[32]) {
            uint32_t v[32];
            tmem_ld_32x32(at, v);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 32; ++i) f[i] = __uint_as_float(v[i]);
        };
        RingPos ap;
        for (int t = first; t < total; t += step) {
            int m0, n0;
            tile_at(t, m0, n0);
            if (!mbar_wait_a(afull_a + 8 * ap.idx, ap.phase)) { report(p.status, kStatusEpilogueTimeout); settle(); break; }
            tc_fence_after_sync();
            const uint32_t d = lanes + ap.idx * BN;
            const int row0 = m0 + quad * 32, row = row0 + lane;
            if (row0 < p.rows) {
#pragma unroll 1
                for (int c = half * 32; c < OUT; c += 64) {
                    const int col0 = n0 + c;
                    if (col0 >= p.cols) break;
                    float z[32];
                    load32(d + c, z);
                    if constexpr (GLU) {
                        float u[32];
                        load32(d + OUT + c, u);
                        if (bias) { add(z, bias, col0); add(u, bias + p.cols, col0); }
                        if (p.keep_z) {
                            put(z, [&](uint32_t buf) { tma_store_3d_a(&tmZ, buf, col0, 0, row0); });
                            put(u, [&](uint32_t buf) { tma_store_3d_a(&tmZ, buf, col0, 1, row0); });
                        }
                        with_act(p.act, [&](auto a) {
#pragma unroll
                            for (int i = 0; i < 32; ++i) z[i] = act_value<decltype(a)::value, true>(z[i], p.k) * u[i];
                        });
                    } else {
                        if (bias) add(z, bias, col0);
                        if (p.keep_z) put(z, [&](uint32_t buf) { tma_store_3d_a(&tmZ, buf, col0, 0, row0); });
                        with_act(p.act, [&](auto a) {
#pragma unroll
                            for (int i = 0; i < 32; ++i) z[i] = act_value<decltype(a)::value, true>(z[i], p.k);
                        });
                        if (residual && row < p.rows) add(z, residual + static_cast<size_t>(row) * p.cols, col0);
                    }
                    put(z, [&](uint32_t buf) { tma_store_3d_a(&tmY, buf, col0, 0, row0); });
                }
            }
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) {
                if constexpr (PAIR) mbar_arrive_cluster(aempty_L + 8 * ap.idx);
                else mbar_arrive_a(aempty_L + 8 * ap.idx);
            }
            ap.advance(2);
        }
        if (lane == 0) tma_store_wait_all();
    }
    tc_fence_before_sync();
    __syncthreads();
    if constexpr (PAIR) cluster_sync_all();   // neither CTA leaves while the other may still reach its shared memory
    if (warp == 1) {
        if constexpr (PAIR) tmem_dealloc_pair(tmem_base, G::kTmem);
        else tmem_dealloc(tmem_base, G::kTmem);
    }
}

}  // namespace alpha
