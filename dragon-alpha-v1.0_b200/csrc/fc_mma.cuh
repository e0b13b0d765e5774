// Products of 16-bit matrices on the tensor cores with the epilogue of a FullConnect layer.
//
//   D[m][n] = sum_k A[m][k] B[n][k]        fp32 sums in tensor memory
//   plain / fc:   z = D + bias[n],  Y = act(z) + R,  Z = z where it is kept for the backward pass
//   glu:          B holds gate rows and up rows; g and u the two sums of a unit, Y = act(g) u, Z = [g | u]
// Forward A = X, B = W; deltaX A = dZ, B = W read along its rows (MN-major); deltaW A = dZ, B = X, both MN-major.  Either operand's memory
// may run along k (a box of 64 steps x rows, 128-byte rows) or along its rows (boxes of 64 rows x 64 steps): the MMA's descriptors take both,
// so nothing is transposed.  Gate and up rows of W, and the halves of Z, are one more dimension of the maps, (step, half, row) or (step, row, half), so
// that what a box reads past a matrix or past a half of it is zeros: no size but IC has to be a multiple of anything.
//
// PAIR: two CTAs of a cluster form 256 x 256 outputs (tcgen05 cta_group::2): each holds its 128 rows of A and half of the rows of B, so that
// shared memory is read and filled with half of B.  Persistent: a pair walks over tiles, in groups of kFcGroupM row tiles so that the tiles in
// flight share rows of A and B in L2; accumulators alternate between two halves of tensor memory, so that the epilogue of a tile runs
// beside the MMAs of the next.  8192 x 22016 x 4096, Z kept: 935 us in short runs, 1090 in long ones, 1.58 and 1.36 PFLOP/s (the power limit: cuBLAS falls from 1.68 to 1.39).
//
// With 256 x 128 outputs, in stages of two blocks of 64 steps, tiles that would fill no wave of the wide ones: an SM takes in 112 KB a us, of which a pair of
// 128 columns needs three quarters of what two CTAs of 128 x 128 do (512 x 4096 x 4096 us: 19.7, CTAs 22, pairs of 256 columns 27).
//
// Otherwise a CTA forms 128 x bn outputs, bn a multiple of 16 that the host picks so that the tiles fill the SMs evenly, in stages of two
// blocks of 64 steps (a stage costs its issuing warp some 400 clocks whatever it holds: 64 columns, 16384 steps 55 -> 35 us).  Of few rows only
// those are staged, which leaves the ring to B: it streams 160 KB of W ahead.  Where tiles are fewer than SMs a cluster of `split` CTAs
// shares a tile's reduction; each leaves its sums in its shared memory, and the cluster's CTAs finish a share of the columns each, adding
// the parts through distributed shared memory in order.
// Warps: 0 TMA producer, 1 MMA issuer, 2-9 epilogue (two per quarter of the lanes, chunks of 32 columns in turn).
#pragma once
#include "fc_act.cuh"
#include "sm100_ptx.cuh"

namespace alpha {

constexpr int kFcThreads = 320, kFcBK = 64, kFcGroupM = 8, kFcMaxStages = 16;
constexpr uint32_t kFcRing = 196608, kFcStaging = 8 * 4096;              // staging: two buffers of 32 x 32 elements for each epilogue warp

struct FcMma {
    int rows, cols;               // outputs: rows of a half, pitch (glu: of a half of Z too)
    int m_tiles, n_tiles, kb;     // tiles, stages of the reduction
    int m_half, k_half;           // tiles of rows, blocks of 64 steps of the first half (deltaW, deltaX with gates)
    int bn, stages, split;        // columns of a CTA's accumulator (glu: of both halves), stages of its ring, CTAs that share a tile
    int a_mn, b_mn, a_rows;       // operands that run along their rows; rows of a box of A that runs along k
    uint32_t idesc, tmem;         // tmem: columns of tensor memory
    int act, keep_z; float k;
    const void *bias, *residual;
    void *Y, *Z;
    int* status;
};
// Blocks of 64 steps of a stage, and its bytes.
__host__ __device__ constexpr int fc_blocks(bool pair, int bn) { return pair && bn == 256 ? 1 : 2; }
__host__ __device__ constexpr uint32_t fc_block_bytes(bool pair, int a_rows, int bn) { return static_cast<uint32_t>(a_rows + (pair ? bn / 2 : bn)) * 128; }

// Elements from a row of a tensor to the one `rows` further (a pitch alone may be 2^31 - 1024).
__host__ __device__ constexpr size_t fc_rows_on(int rows, size_t pitch) { return rows * pitch; }

// PAIR: columns of a pair's tiles, 256 or 128, or 0.  TWO: the tiles of a second product of the same geometry follow those of the first (deltaX and deltaW, neither of which may fill the SMs).
template <class T, int PAIR, bool GLU, bool TWO>
__global__ void __launch_bounds__(kFcThreads, 1)
    fc_mma_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const __grid_constant__ FcMma p, const __grid_constant__ CUtensorMap tmA2,
                  const __grid_constant__ CUtensorMap tmB2, const __grid_constant__ FcMma p2)
{
    constexpr int CTAS = PAIR ? 2 : 1, KB = fc_blocks(PAIR != 0, PAIR);
    const int BN = PAIR ? PAIR : p.bn, OUT = GLU ? BN / 2 : BN, S = PAIR ? static_cast<int>(kFcRing / (KB * fc_block_bytes(true, 128, PAIR))) : p.stages, split = PAIR ? 1 : p.split;
    const uint32_t kA = PAIR ? 16384u : static_cast<uint32_t>(p.a_rows) * 128, kB = PAIR ? PAIR * 64u : static_cast<uint32_t>(BN) * 128, kBlock = kA + kB, kStage = KB * kBlock;
    const int acc_pitch = (BN + 31) & ~31;        // columns from one accumulator to the other
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S * kStage + kFcStaging);
    uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(bars + 2 * kFcMaxStages + 4);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = PAIR || split > 1 ? cluster_ctarank() : 0u;       // of the pair, or of those that share a tile
    const uint32_t full_a = smem_u32(bars), empty_a = full_a + 8 * kFcMaxStages, afull_a = empty_a + 8 * kFcMaxStages, aempty_a = afull_a + 16;

    if (threadIdx.x == 0) {
        for (int i = 0; i < S; ++i) { mbar_init(&bars[i], 1); mbar_init(&bars[kFcMaxStages + i], 1); }
        for (int i = 0; i < 2; ++i) { mbar_init(&bars[2 * kFcMaxStages + i], 1); mbar_init(&bars[2 * kFcMaxStages + 2 + i], 8 * CTAS); }
        fence_barrier_init();
        prefetch_tmap(&tmA); prefetch_tmap(&tmB);
        if (TWO) { prefetch_tmap(&tmA2); prefetch_tmap(&tmB2); }
    }
    if (warp == 1) {
        if constexpr (PAIR) { tmem_alloc_pair(tmem_holder, 512); tmem_relinquish_pair(); }
        else { tmem_alloc(tmem_holder, p.tmem); tmem_relinquish(); }
    }
    tc_fence_before_sync();
    grid_dependency_wait();
    __syncthreads();
    if constexpr (PAIR) cluster_sync_all();   // the peer's barriers are initialised before anything reaches them
    grid_dependency_trigger();
    tc_fence_after_sync();
    const uint32_t tmem_base = *tmem_holder;

    // (shared tiles: the launch has a cluster for each)
    const int tiles = p.m_tiles * p.n_tiles, total = tiles + (TWO ? p2.m_tiles * p2.n_tiles : 0), step = gridDim.x / (CTAS * split), first = blockIdx.x / (CTAS * split);
    const FcMma* cur = &p;                        // the product of the tile at hand
    int hm = 0;                                   // the half of its rows
    auto tile_at = [&](int t, int& m0, int& n0) {
        if (TWO) cur = t < tiles ? &p : &p2;
        if (TWO && t >= tiles) t -= tiles;
        const int per = kFcGroupM * cur->n_tiles, g = t / per, r = t - g * per, left = cur->m_tiles - g * kFcGroupM, rows = left < kFcGroupM ? left : kFcGroupM;
        const int n = r / rows, m = g * kFcGroupM + r - n * rows;
        hm = m >= cur->m_half ? 1 : 0;
        m0 = (m - hm * cur->m_half) * (128 * CTAS) + (PAIR ? static_cast<int>(rank) * 128 : 0);
        n0 = n * OUT;
    };
    auto steps_of = [&](int& begin, int& end) {
        const int each = (cur->kb + split - 1) / split;
        begin = PAIR ? 0 : static_cast<int>(rank) * each;
        end = begin + each < cur->kb ? begin + each : cur->kb;
    };
    const uint32_t smem_a = smem_u32(smem);
    const int quad = warp & 3, half = (warp - 2) >> 2;
    const uint32_t stage_a = smem_a + S * kStage + (warp - 2) * 4096;
    uint32_t sbuf = 0;
    bool ok = true;
    // A warp's 32 rows x 32 columns change hands in shared memory between lanes that hold a row (the accumulator's layout) and lanes that hold 16 bytes of
    // row 8 j + lane / 4, eight rows of 64 bytes to an instruction, as global memory is read and written.  Two buffers in turn, so that one barrier of the
    // warp serves each.  (By TMA stores, with their fence and the wait for the buffer, 7966 x 64 x 8136 with silu
    // and R took 182 us, with what follows 87.)
    const uint32_t row_at = stage_a + lane * 64, word_at = stage_a + (lane >> 2) * 64 + (((lane & 3) ^ ((lane >> 3) & 3)) << 4);
    auto row_word = [&](int q) { return row_at + sbuf * 2048 + ((q ^ ((lane >> 1) & 3)) << 4); };
    // word j of a lane lies 8 rows further: the swizzle is that of its row
    auto lane_word = [&](int j) { return word_at + sbuf * 2048 + j * 512; };
    auto inside = [&](int row0, int col0, int width, int j) {
        const int c = 8 * (lane & 3);
        return row0 + 8 * j + (lane >> 2) < cur->rows && c < width && col0 + c < cur->cols;
    };
    auto put = [&](const float (&f)[32], T* tensor, size_t pitch, int row0, int col0, int width) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const uint4 w = Word16<T>::store(f + 8 * q);
            st_shared_v4(row_word(q), make_float4(__uint_as_float(w.x), __uint_as_float(w.y), __uint_as_float(w.z), __uint_as_float(w.w)));
        }
        __syncwarp();
        T* to = tensor + static_cast<size_t>(row0 + (lane >> 2)) * pitch + col0 + 8 * (lane & 3);
#pragma unroll
        for (int j = 0; j < 4; ++j, to += fc_rows_on(8, pitch)) {
            const float4 w = ld_shared_v4(lane_word(j));
            if (inside(row0, col0, width, j)) *reinterpret_cast<float4*>(to) = w;
        }
        sbuf ^= 1u;
    };
    // The words of R that put() will write over, or zeros (R may be Y itself: not by the read-only path).
    auto fetch = [&](uint4 (&r)[4], int row0, int col0, int width) {
        const T* from = static_cast<const T*>(cur->residual) + static_cast<size_t>(row0 + (lane >> 2)) * cur->cols + col0 + 8 * (lane & 3);
#pragma unroll
        for (int j = 0; j < 4; ++j, from += fc_rows_on(8, cur->cols)) r[j] = inside(row0, col0, width, j) ? *reinterpret_cast<const uint4*>(from) : make_uint4(0, 0, 0, 0);
    };
    auto add_fetched = [&](float (&f)[32], const uint4 (&r)[4]) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            st_shared_v4(lane_word(j), make_float4(__uint_as_float(r[j].x), __uint_as_float(r[j].y), __uint_as_float(r[j].z), __uint_as_float(r[j].w)));
        __syncwarp();
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const float4 w = ld_shared_v4(row_word(q));
            float b[8];
            Word16<T>::load(make_uint4(__float_as_uint(w.x), __float_as_uint(w.y), __float_as_uint(w.z), __float_as_uint(w.w)), b);
#pragma unroll
            for (int i = 0; i < 8; ++i) f[8 * q + i] += b[i];
        }
        sbuf ^= 1u;
    };
    // f += 32 columns of the bias (its length a multiple of 8)
    auto add_bias = [&](float (&f)[32], const T* from, int col0) {
#pragma unroll
        for (int q = 0; q < 4; ++q)
            if (col0 + 8 * q < cur->cols) {
                float b[8];
                Word16<T>::load(__ldg(reinterpret_cast<const uint4*>(from + col0 + 8 * q)), b);
#pragma unroll
                for (int i = 0; i < 8; ++i) f[8 * q + i] += b[i];
            }
    };
    // The epilogue of 32 rows x (up to) 32 columns: the sums of a lane's row in z (glu: and u), the words of R in r.
    auto finish = [&](float (&z)[32], float (&u)[32], const uint4 (&r)[4], int row0, int col0, int width) {
        const T* bias = static_cast<const T*>(cur->bias);
        T *Y = static_cast<T*>(cur->Y) + (hm ? static_cast<size_t>(cur->rows) * cur->cols : 0), *Z = static_cast<T*>(cur->Z);
        if constexpr (GLU) {
            if (bias) { add_bias(z, bias, col0); add_bias(u, bias + cur->cols, col0); }
            if (cur->keep_z) {
                const size_t pitch = 2 * static_cast<size_t>(cur->cols);
                put(z, Z, pitch, row0, col0, width);
                put(u, Z + cur->cols, pitch, row0, col0, width);
            }
            with_act(cur->act, [&](auto a) {
#pragma unroll
                for (int i = 0; i < 32; ++i) z[i] = act_value<decltype(a)::value, true>(z[i], cur->k) * u[i];
            });
        } else {
            if (bias) add_bias(z, bias, col0);
            if (cur->keep_z) put(z, Z, cur->cols, row0, col0, width);
            with_act(cur->act, [&](auto a) {
#pragma unroll
                for (int i = 0; i < 32; ++i) z[i] = act_value<decltype(a)::value, true>(z[i], cur->k);
            });
            if (cur->residual) add_fetched(z, r);
        }
        put(z, Y, cur->cols, row0, col0, width);
    };

    // Both issuing warps walk their loops as a whole, so that counters, coordinates and descriptors are uniform values; one lane issues.
    if (warp == 0) {
        const uint32_t base = __shfl_sync(0xffffffffu, smem_a, 0), full_0 = __shfl_sync(0xffffffffu, full_a, 0), empty_0 = full_0 + 8 * kFcMaxStages;
        const uint32_t full_L = PAIR ? __shfl_sync(0xffffffffu, mapa_u32(full_a, 0), 0) : full_0, elected = elect_one();
        const uint32_t tx = CTAS * kStage;
        const int my = PAIR ? __shfl_sync(0xffffffffu, static_cast<int>(rank), 0) : 0;
        auto load = [&](uint32_t dst, const CUtensorMap* m, uint32_t bar, int c0, int c1, int c2) {
            if constexpr (PAIR) tma_load_3d_pair(dst, m, bar, c0, c1, c2);
            else tma_load_3d_a(dst, m, bar, c0, c1, c2);
        };
        RingPos rp;
        for (int t = first; t < total && ok; t += step) {
            int m0, n0;
            tile_at(t, m0, n0);
            int k_begin, k_end;
            steps_of(k_begin, k_end);
            const CUtensorMap *mA = TWO && t >= tiles ? &tmA2 : &tmA, *mB = TWO && t >= tiles ? &tmB2 : &tmB;
            const int a_mn = cur->a_mn, b_mn = cur->b_mn, k_half = cur->k_half;
            for (int kb = k_begin; kb < k_end; ++kb) {
                ok = __all_sync(0xffffffffu, mbar_wait_a(empty_0 + 8 * rp.idx, rp.phase ^ 1));
                if (!ok) { report(p.status, kStatusProducerTimeout); settle(); break; }
                if (elected) {
                    if (my == 0) mbar_arrive_expect_tx_a(full_0 + 8 * rp.idx, tx);
                    const uint32_t bar = full_L + 8 * rp.idx;
#pragma unroll
                    for (int q = 0; q < KB; ++q) {
                        const uint32_t a = base + rp.idx * kStage + q * kBlock, b = a + kA;
                        // (the block after the last of an odd number lies past both halves)
                        const int block = kb * KB + q, hk = block >= k_half ? (block - k_half >= k_half ? 2 : 1) : 0, k0 = (block - hk * k_half) * kFcBK;
                        if (a_mn) {
#pragma unroll
                            for (int j = 0; j < 2; ++j) load(a + j * 8192, mA, bar, m0 + 64 * j, hm, k0);
                        } else {
                            load(a, mA, bar, k0, hk, m0);
                        }
                        if constexpr (GLU) {
                            // columns [gate | up] of the accumulator
                            if constexpr (PAIR) load(b, mB, bar, k0, n0, my);
                            else { load(b, mB, bar, k0, n0, 0); load(b + kB / 2, mB, bar, k0, n0, 1); }
                        } else {
                            const int b0 = n0 + my * (BN / 2);
                            if (b_mn) {
                                for (int j = 0; j < static_cast<int>(kB >> 13); ++j) load(b + j * 8192, mB, bar, b0 + 64 * j, k0, hk);
                            } else {
                                load(b, mB, bar, k0, b0, 0);
                            }
                        }
                    }
                }
                __syncwarp();
                if (++rp.idx == S) { rp.idx = 0; rp.phase ^= 1u; }
            }
        }
    } else if (warp == 1) {
        if (!PAIR || rank == 0) {
            constexpr uint32_t dhi = (1024u >> 4) | (1u << 14) | (static_cast<uint32_t>(kSwizzle128B) << 29);
            const uint32_t base = __shfl_sync(0xffffffffu, smem_a, 0), tmem = __shfl_sync(0xffffffffu, tmem_base, 0), elected = elect_one();
            const uint32_t full_0 = __shfl_sync(0xffffffffu, full_a, 0), empty_0 = full_0 + 8 * kFcMaxStages, afull_0 = empty_0 + 8 * kFcMaxStages, aempty_0 = afull_0 + 16;
            auto commit = [&](uint32_t bar) {
                if constexpr (PAIR) mma_commit_both(bar);
                else mma_commit_a(bar);
            };
            auto wait = [&](uint32_t bar, uint32_t parity) {
                if (__all_sync(0xffffffffu, PAIR ? mbar_wait_cluster_a(bar, parity) : mbar_wait_a(bar, parity))) return true;
                report(p.status, kStatusMmaTimeout);
                settle();
                return false;
            };
            RingPos rp, ap;
            bool next = false;                            // the stage at rp is known to be full
            for (int t = first; t < total && ok; t += step) {
                if (TWO) cur = t < tiles ? &p : &p2;
                int k_begin, k_end;
                steps_of(k_begin, k_end);
                const uint32_t a_k = cur->a_mn ? 128u : 2u, b_k = cur->b_mn ? 128u : 2u, idesc = cur->idesc;      // 16 steps further, in 16-byte units
                const uint32_t a_lo0 = smem_desc_lo(base, cur->a_mn ? 8192u : 16u), b_lo0 = smem_desc_lo(base + kA, cur->b_mn ? 8192u : 16u);
                if (!wait(aempty_0 + 8 * ap.idx, ap.phase ^ 1)) break;
                tc_fence_after_sync();
                const uint32_t d = tmem + ap.idx * acc_pitch;
                for (int kb = k_begin; kb < k_end; ++kb) {
                    if (!__all_sync(0xffffffffu, next) && !wait(full_0 + 8 * rp.idx, rp.phase)) { ok = false; break; }
                    tc_fence_after_sync();
                    const uint32_t a = a_lo0 + rp.idx * (kStage >> 4), b = b_lo0 + rp.idx * (kStage >> 4), done = empty_0 + 8 * rp.idx;
#pragma unroll
                    for (uint32_t q = 0; q < KB; ++q)
#pragma unroll
                        for (uint32_t kk = 0; kk < 4; ++kk)
                            mma_16bit<PAIR != 0>(d, a + q * (kBlock >> 4) + kk * a_k, dhi, b + q * (kBlock >> 4) + kk * b_k, dhi, idesc, kb > k_begin || q || kk ? 1u : 0u, elected);
                    if (elected) commit(done);
                    if (++rp.idx == S) { rp.idx = 0; rp.phase ^= 1u; }
                    next = mbar_test_a<PAIR != 0>(full_0 + 8 * rp.idx, rp.phase);     // (beside the MMAs just issued)
                }
                if (ok && elected) commit(afull_0 + 8 * ap.idx);
                ap.advance(2);
            }
        }
        __syncwarp();
    } else {
        const uint32_t lanes = tmem_base + (static_cast<uint32_t>(quad * 32) << 16), aempty_L = PAIR ? mapa_u32(aempty_a, 0) : aempty_a;
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
            const int row0 = m0 + quad * 32;
            // R: the next tile's to L2, and the first chunk of this one before the sums are there (8192 x 64 x 8192 with R 90 us without the former)
            uint4 r[4] = {};
            const bool fetching = !GLU && cur->residual && row0 < cur->rows && (PAIR || split == 1);
            if (!GLU && cur->residual && (PAIR || split == 1)) {
                int m1, n1;
                tile_at(t + step < total ? t + step : t, m1, n1);       // (one half: R goes with a forward product)
                const int row = m1 + quad * 32 + lane;
                for (int c = half * 32; c < OUT; c += 64)
                    if (row < cur->rows && n1 + c < cur->cols) prefetch_l2(static_cast<const T*>(cur->residual) + static_cast<size_t>(row) * cur->cols + n1 + c);
            }
            if (fetching) fetch(r, row0, n0 + half * 32, OUT - half * 32);
            ok = mbar_wait_a(afull_a + 8 * ap.idx, ap.phase);
            if (!ok) { report(p.status, kStatusEpilogueTimeout); settle(); break; }
            tc_fence_after_sync();
            const uint32_t d = lanes + ap.idx * acc_pitch;
            // The accumulator is given back when its last columns are in registers, before they are stored; the arrival orders no memory (a release
            // across the pair waited for the tile's stores: 7592 x 24 x 2 x 3968 45 us instead of 35).
            auto give_back = [&] {
                tc_fence_before_sync();
                __syncwarp();
                if (lane == 0) {
                    if constexpr (PAIR) mbar_arrive_cluster_relaxed(aempty_L + 8 * ap.idx);
                    else mbar_arrive_relaxed_a(aempty_L + 8 * ap.idx);
                }
            };
            bool held = true;
            if (row0 < cur->rows) {
                if (!PAIR && split > 1) {
                    // the ring is idle: [row][column] with four floats more, so that the words of eight rows lie in different banks
                    const uint32_t to = smem_a + static_cast<uint32_t>(quad * 32 + lane) * (BN + 4) * 4;
#pragma unroll 1
                    for (int c = half * 32; c < BN; c += 64) {
                        float z[32];
                        load32(d + c, z);
                        if (row0 + lane < cur->rows)
#pragma unroll
                            for (int q = 0; q < 8; ++q)
                                if (c + 4 * q < BN) st_shared_v4(to + (c + 4 * q) * 4, make_float4(z[4 * q], z[4 * q + 1], z[4 * q + 2], z[4 * q + 3]));
                    }
                } else {
#pragma unroll 1
                    for (int c = half * 32; c < OUT; c += 64) {
                        if (n0 + c >= cur->cols) break;
                        float z[32], u[32];
                        load32(d + c, z);
                        if constexpr (GLU) load32(d + OUT + c, u);
                        if (c + 64 >= OUT || n0 + c + 64 >= cur->cols) { give_back(); held = false; }
                        finish(z, u, r, row0, n0 + c, OUT - c);
                        if (fetching && c + 64 < OUT) fetch(r, row0, n0 + c + 64, OUT - c - 64);
                    }
                }
            }
            if (held) give_back();
            ap.advance(2);
        }
    }
    if (!PAIR && split > 1) {
        ok = __syncthreads_and(ok) != 0;
        cluster_sync_all();
        if (warp >= 2 && ok) {
            int m0, n0;
            tile_at(first, m0, n0);
            // shares of 32 rows x 32 columns, CTAs and warps in turn
            const int quads = (cur->rows - m0 + 31) / 32 < 4 ? (cur->rows - m0 + 31) / 32 : 4, chunks = (OUT + 31) / 32;
            for (int i = static_cast<int>(rank) * 8 + warp - 2; i < quads * chunks; i += split * 8) {
                const int q4 = i / chunks, c = (i - q4 * chunks) * 32, row0 = m0 + q4 * 32;
                if (n0 + c >= cur->cols) continue;
                const uint32_t from = smem_a + static_cast<uint32_t>(q4 * 32 + lane) * (BN + 4) * 4;
                float z[32], u[32];
#pragma unroll
                for (int j = 0; j < 32; ++j) z[j] = u[j] = 0.f;
                if (row0 + lane < cur->rows)
                    for (int r = 0; r < split; ++r) {
                        const uint32_t peer = mapa_u32(from, r);
#pragma unroll
                        for (int q = 0; q < 8; ++q) {
                            if (c + 4 * q >= OUT) continue;
                            const float4 v = ld_shared_cluster_v4(peer + (c + 4 * q) * 4);
                            z[4 * q] += v.x; z[4 * q + 1] += v.y; z[4 * q + 2] += v.z; z[4 * q + 3] += v.w;
                            if constexpr (GLU) {
                                const float4 w = ld_shared_cluster_v4(peer + (OUT + c + 4 * q) * 4);
                                u[4 * q] += w.x; u[4 * q + 1] += w.y; u[4 * q + 2] += w.z; u[4 * q + 3] += w.w;
                            }
                        }
                    }
                uint4 r[4] = {};
                if (!GLU && cur->residual) fetch(r, row0, n0 + c, OUT - c);
                finish(z, u, r, row0, n0 + c, OUT - c);
            }
        }
    }
    tc_fence_before_sync();
    __syncthreads();
    if (PAIR || split > 1) cluster_sync_all();   // no CTA leaves while another may still reach its shared memory
    if (warp == 1) {
        if constexpr (PAIR) tmem_dealloc_pair(tmem_base, 512);
        else tmem_dealloc(tmem_base, p.tmem);
    }
}

}  // namespace alpha
