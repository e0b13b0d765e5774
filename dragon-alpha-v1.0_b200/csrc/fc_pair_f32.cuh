// Large fp32 products of a FullConnect layer as three bf16 planes on CTA pairs.
//
// The arithmetic is that of the gathering kernel (x = h + m + l; hh in one accumulator, hm, mh, mm, hl, lh in another; after every 64 steps the
// hh sum, which the tensor core truncates as it adds, goes to running sums in registers, rounded to nearest).  That kernel splits its operands as it
// stages them, once for each tile that reads them, and its 128 x 128 tiles read 8 KB of shared memory for 64 clocks of MMAs.  Here both operands are split
// once, into planes in scratch (10 bytes of traffic an element), copied by TMA, and multiplied by pairs of CTAs: 256 x 256 outputs,
// six cta_group::2 MMAs of 128 clocks for 16 steps, each CTA's tensor memory holding hh in 256 columns and the rest in the other 256.
// hh needs no second buffer: its four MMAs of a window of 64 steps come first, and while the twenty others run (2560 clocks) the epilogue
// warps fetch it.  Bound: the MMAs, a sixth of the bf16 rate (280 TFLOP/s of fp32 products at the measured 1.68 PFLOP/s, 232 under the
// power limit).  us here / gathering: 8192 x 4096 x 4096 1110 / 2020 (247 TFLOP/s), 2048 x 2048 x 2048 85 / 135; of few tiles the other is faster.
// Operands: [plane][row][pitch]; a slot of the ring holds one plane of both for 64 steps, boxes of 64 steps x 128 rows, or of 64 rows x 64
// steps where memory runs along the rows (128-byte rows either way: the copies take two clocks a row, and with boxes of 32 steps bound the kernel).
// BN: 256 columns, or 128, whose tiles cost 0.6 of one and fill the waves of a launch more evenly (us, 256 / 128: gated 1000 x 1024 x 2 x 2752, 88 or 172 tiles
// on 74 pairs, 82 / 76; 4381 x 1004 x 2 x 182 37.5 / 34; 2048 x 2048 x 2048 85 / 97).
// The MMAs of a window go with the slots: hh; hm, mh, mm; hl, lh.  A work item is a tile and a part of the reduction; parts are added by another launch.
// Words that are not the sum of their planes arrive as NaN.  A warp that finds a sum that is not finite, or below 2^-110 and not zero, forms its
// 32 rows x 128 columns once more by FMAs from the fp32 tensors, in ascending k.
// Warps: 0 TMA producer, 1 MMA issuer (of the leader), 2-9 epilogue: 128 running sums a thread.
#pragma once
#include "fc_f32.cuh"

namespace alpha {

constexpr int kPairF32Threads = 320, kPairF32Slots = 6;
constexpr uint32_t kPairF32Operand = 128 * 128;                                    // 128 rows of A of a CTA, 64 steps of a plane
__host__ __device__ constexpr uint32_t pair_f32_slot(int bn) { return kPairF32Operand + bn / 2 * 128; }
__host__ __device__ constexpr uint32_t pair_f32_smem(int bn) { return kPairF32Slots * pair_f32_slot(bn) + 8 * 4096 + 1024 + 256; }

// Up to three fp32 matrices as planes, dst[plane][row][pitch]; columns past cols are zeros.
struct SplitJob { const float* src; uint2* dst; unsigned rows, cols4, first; FastDiv by_pitch4; };
struct SplitJobs { SplitJob job[3]; int n; unsigned total; };
__global__ void __launch_bounds__(256) fc_split_kernel(const __grid_constant__ SplitJobs p)
{
    grid_dependency_wait();
    grid_dependency_trigger();
    for (unsigned w = blockIdx.x * 256 + threadIdx.x; w < p.total; w += gridDim.x * 256) {
        int q = 0;
        while (q + 1 < p.n && w >= p.job[q + 1].first) ++q;
        const SplitJob& j = p.job[q];
        const unsigned i = w - j.first;
        unsigned r, c;
        j.by_pitch4.divmod(i, r, c);
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        if (c < j.cols4) v = __ldg(reinterpret_cast<const float4*>(j.src) + static_cast<size_t>(r) * j.cols4 + c);
        uint2 h, m, l;
        uint32_t lost = 0;
        split_planes(v, h, m, l, lost);
        if (lost & 0xffffu) h = make_uint2(0x7fff7fffu, 0x7fff7fffu);
        const size_t plane = static_cast<size_t>(j.rows) * j.by_pitch4.d;
        j.dst[i] = h; j.dst[plane + i] = m; j.dst[2 * plane + i] = l;
    }
}

struct PairF32 {
    int rows, cols, pitch, K;      // outputs (glu: columns of a half; rows of a half), pitch of Y, R and halves of Z and the bias; steps (of a half)
    int m_tiles, n_tiles, windows, parts;   // windows: of 64 steps
    int m_half, w_half;            // tiles of rows, windows of the first half (deltaW, deltaX with gates)
    int a_mn, b_mn;
    uint32_t idesc;
    // the fp32 operands: element (row, k) of half h at A[h * a_half + row * a_row + k * a_k], (column, k) at B[h * b_half + column * b_col + k * b_k]
    const float *A, *B;
    long long a_row, a_k, a_half, b_col, b_k, b_half;
    const float *bias, *residual;
    int act, keep_z; float k;
    int* status;
};

// 32 columns of a row from col0 on, of halves ha and hb of the operands' rows, over windows [w0, w1), as sums of FMAs in ascending k.  Columns past
// the last are formed as the last.
static __device__ __noinline__ void form_row_f32(const PairF32& p, int row, int col0, int ha, int hb, int w0, int w1, float* z)
{
    float acc[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) acc[i] = 0.f;
    for (int w = w0; w < w1; ++w) {
        const int hk = w >= p.w_half ? 1 : 0, k0 = (w - hk * p.w_half) * 64, k1 = k0 + 64 < p.K ? k0 + 64 : p.K;
        const float *a = p.A + (ha + hk) * p.a_half + row * p.a_row, *b = p.B + (hb + hk) * p.b_half;
        for (int k = k0; k < k1; ++k) {
            const float av = __ldg(a + k * p.a_k);
#pragma unroll
            for (int i = 0; i < 32; ++i) acc[i] = fmaf(av, __ldg(b + (col0 + i < p.cols ? col0 + i : p.cols - 1) * p.b_col + k * p.b_k), acc[i]);
        }
    }
#pragma unroll
    for (int i = 0; i < 32; ++i) z[i] = acc[i];
}

// tmY: the result, or where parts > 1 the sums, as (column, half, row, part)
template <bool GLU, int BN>
__global__ void __launch_bounds__(kPairF32Threads, 1)
    fc_pair_f32_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const __grid_constant__ CUtensorMap tmY,
                       const __grid_constant__ CUtensorMap tmZ, const __grid_constant__ PairF32 p)
{
    constexpr int S = kPairF32Slots, OUT = GLU ? BN / 2 : BN, HALF = BN / 2, QUARTER = BN / 4;
    constexpr uint32_t kPairF32Slot = pair_f32_slot(BN);
    constexpr uint32_t kHh = 0, kSide = 256;          // columns of tensor memory
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S * kPairF32Slot + 8 * 4096);
    uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(bars + 2 * S + 4);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_ctarank();
    const uint32_t full_a = smem_u32(bars), empty_a = full_a + 8 * S, hh_full_a = empty_a + 8 * S, hh_free_a = hh_full_a + 8, side_full_a = hh_free_a + 8, side_free_a = side_full_a + 8;

    if (threadIdx.x == 0) {
        for (int i = 0; i < 2 * S; ++i) mbar_init(&bars[i], 1);
        mbar_init(&bars[2 * S], 1); mbar_init(&bars[2 * S + 1], 16);
        mbar_init(&bars[2 * S + 2], 1); mbar_init(&bars[2 * S + 3], 16);
        fence_barrier_init();
        prefetch_tmap(&tmA); prefetch_tmap(&tmB); prefetch_tmap(&tmY);
        if (p.keep_z) prefetch_tmap(&tmZ);
    }
    if (warp == 1) {
        tmem_alloc_pair(tmem_holder, 512);
        tmem_relinquish_pair();
    }
    tc_fence_before_sync();
    grid_dependency_wait();
    __syncthreads();
    cluster_sync_all();   // the peer's barriers are initialised before anything reaches them
    grid_dependency_trigger();
    tc_fence_after_sync();
    const uint32_t tmem_base = *tmem_holder, smem_a = smem_u32(smem);

    const int tiles = p.m_tiles * p.n_tiles, total = tiles * p.parts, step = gridDim.x / 2, first = blockIdx.x / 2;
    struct Item { int m0, n0, w0, w1, part, hm; };
    auto item_at = [&](int t) {
        Item i;
        i.part = t / tiles;
        t -= i.part * tiles;
        constexpr int GROUP = 4;                      // row tiles that are walked together: what is in flight shares rows in L2
        const int per = GROUP * p.n_tiles, g = t / per, r = t - g * per, left = p.m_tiles - g * GROUP, rows = left < GROUP ? left : GROUP, n = r / rows, m = g * GROUP + r - n * rows;
        i.hm = m >= p.m_half ? 1 : 0;
        i.m0 = (m - i.hm * p.m_half) * 256 + static_cast<int>(rank) * 128;
        i.n0 = n * OUT;
        const int each = (p.windows + p.parts - 1) / p.parts;
        i.w0 = i.part * each < p.windows ? i.part * each : p.windows;
        i.w1 = i.w0 + each < p.windows ? i.w0 + each : p.windows;
        return i;
    };
    bool ok = true;

    if (warp == 0) {
        const uint32_t base = __shfl_sync(0xffffffffu, smem_a, 0), full_0 = __shfl_sync(0xffffffffu, full_a, 0), empty_0 = full_0 + 8 * S;
        const uint32_t full_L = __shfl_sync(0xffffffffu, mapa_u32(full_a, 0), 0), elected = elect_one();
        const int my = __shfl_sync(0xffffffffu, static_cast<int>(rank), 0);
        RingPos rp;
        for (int t = first; t < total && ok; t += step) {
            const Item it = item_at(t);
            const int b0 = GLU ? it.n0 : it.n0 + my * HALF;
            for (int s = 3 * it.w0; s < 3 * it.w1; ++s) {
                ok = __all_sync(0xffffffffu, mbar_wait_a(empty_0 + 8 * rp.idx, rp.phase ^ 1));
                if (!ok) { report(p.status, kStatusProducerTimeout); settle(); break; }
                if (elected) {
                    if (my == 0) mbar_arrive_expect_tx_a(full_0 + 8 * rp.idx, 2 * kPairF32Slot);
                    const uint32_t bar = full_L + 8 * rp.idx, a = base + rp.idx * kPairF32Slot, b = a + kPairF32Operand;
                    const int w = s / 3, plane = s % 3, hk = w >= p.w_half ? 1 : 0, k0 = (w - hk * p.w_half) * 64;
                    if (p.a_mn) {
#pragma unroll
                        for (int j = 0; j < 2; ++j) tma_load_4d_pair(a + j * 8192, &tmA, bar, it.m0 + 64 * j, it.hm, k0, plane);
                    } else {
                        tma_load_4d_pair(a, &tmA, bar, k0, hk, it.m0, plane);
                    }
                    if (p.b_mn) {
#pragma unroll
                        for (int j = 0; j < BN / 128; ++j) tma_load_4d_pair(b + j * 8192, &tmB, bar, b0 + 64 * j, k0, hk, plane);
                    } else {
                        tma_load_4d_pair(b, &tmB, bar, k0, b0, GLU ? my : 0, plane);
                    }
                }
                __syncwarp();
                rp.advance(S);
            }
        }
    } else if (warp == 1) {
        if (rank == 0) {
            const uint32_t base = __shfl_sync(0xffffffffu, smem_a, 0), tmem = __shfl_sync(0xffffffffu, tmem_base, 0), elected = elect_one();
            const uint32_t full_0 = __shfl_sync(0xffffffffu, full_a, 0), empty_0 = full_0 + 8 * S, hh_full = empty_0 + 8 * S, hh_free = hh_full + 8, side_full = hh_free + 8, side_free = side_full + 8;
            constexpr uint32_t dhi = (1024u >> 4) | (1u << 14) | (static_cast<uint32_t>(kSwizzle128B) << 29);
            const uint32_t a_k = p.a_mn ? 128u : 2u, b_k = p.b_mn ? 128u : 2u;               // 16 steps further, in 16-byte units
            const uint32_t a_lo0 = smem_desc_lo(base, p.a_mn ? 8192u : 16u), b_lo0 = smem_desc_lo(base + kPairF32Operand, p.b_mn ? 8192u : 16u);
            auto wait = [&](uint32_t bar, uint32_t parity) {
                if (__all_sync(0xffffffffu, mbar_wait_cluster_a(bar, parity))) return true;
                report(p.status, kStatusMmaTimeout);
                settle();
                return false;
            };
            // four steps of 16 of plane x of A times plane y of B, given by their slots
            auto multiply = [&](uint32_t d, uint32_t x, uint32_t y, bool fresh) {
                const uint32_t a = a_lo0 + x * (kPairF32Slot >> 4), b = b_lo0 + y * (kPairF32Slot >> 4);
#pragma unroll
                for (uint32_t kk = 0; kk < 4; ++kk) mma_16bit<true>(tmem + d, a + kk * a_k, dhi, b + kk * b_k, dhi, p.idesc, fresh && kk == 0 ? 0u : 1u, elected);
            };
            auto commit = [&](uint32_t bar) {
                if (elected) mma_commit_both(bar);
                __syncwarp();
            };
            RingPos rp;
            uint32_t window = 0, item = 0;
            for (int t = first; t < total && ok; t += step, ++item) {
                const Item it = item_at(t);
                for (int w = it.w0; w < it.w1; ++w, ++window) {
                    const uint32_t h = rp.idx, m = h + 1, l = h + 2, phase = rp.phase;       // (slots of a window follow one another: S is a multiple of 3)
                    ok = wait(full_0 + 8 * h, phase) && wait(hh_free, (window & 1) ^ 1);
                    if (!ok) break;
                    tc_fence_after_sync();
                    multiply(kHh, h, h, true);
                    commit(hh_full);
                    ok = (w > it.w0 || wait(side_free, (item & 1) ^ 1)) && wait(full_0 + 8 * m, phase);
                    if (!ok) break;
                    tc_fence_after_sync();
                    multiply(kSide, h, m, w == it.w0);
                    multiply(kSide, m, h, false);
                    multiply(kSide, m, m, false);
                    commit(empty_0 + 8 * m);
                    ok = wait(full_0 + 8 * l, phase);
                    if (!ok) break;
                    tc_fence_after_sync();
                    multiply(kSide, h, l, false);
                    multiply(kSide, l, h, false);
                    commit(empty_0 + 8 * h);
                    commit(empty_0 + 8 * l);
                    rp.advance(S); rp.advance(S); rp.advance(S);
                }
                if (ok) commit(side_full);
            }
        }
        __syncwarp();
    } else {
        const int quad = warp & 3, half = (warp - 2) >> 2;
        // QUARTER sums from either column on (glu: gates, and the units' other halves)
        const int col_a = (GLU ? QUARTER : HALF) * half, col_b = GLU ? HALF + col_a : col_a + QUARTER;
        const uint32_t lanes = tmem_base + (static_cast<uint32_t>(quad * 32) << 16), hh_free_L = mapa_u32(hh_free_a, 0), side_free_L = mapa_u32(side_free_a, 0);
        const uint32_t buf = smem_a + S * kPairF32Slot + (warp - 2) * 4096;
        unsigned long long acc[QUARTER];
        auto add_columns = [&](uint32_t from) {
#pragma unroll
            for (int x = 0; x < HALF; x += 16) {
                uint32_t v[16];
                tmem_ld_32x16(lanes + from + (x < QUARTER ? col_a + x : col_b + x - QUARTER), v);
                tmem_ld_wait();
#pragma unroll
                for (int q = 0; q < 16; q += 2) acc[(x + q) / 2] = add2(acc[(x + q) / 2], pack2(__uint_as_float(v[q]), __uint_as_float(v[q + 1])));
            }
        };
        auto wait = [&](uint32_t bar, uint32_t parity) {
            ok = __all_sync(0xffffffffu, mbar_wait_a(bar, parity));
            if (!ok) { report(p.status, kStatusEpilogueTimeout); settle(); }
            return ok;
        };
        auto release = [&](uint32_t bar) {
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster_relaxed(bar);
        };
        // 32 columns of a lane's row leave as a box of 32 rows x 128 bytes
        auto put = [&](const float (&f)[32], auto&& store) {
            if (lane == 0) tma_store_wait_read<0>();
            __syncwarp();
#pragma unroll
            for (int q = 0; q < 8; ++q) st_shared_v4(buf + lane * 128 + ((q ^ (lane & 7)) << 4), make_float4(f[4 * q], f[4 * q + 1], f[4 * q + 2], f[4 * q + 3]));
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) { store(); tma_store_commit(); }
        };
        uint32_t window = 0, item = 0;
        for (int t = first; t < total && ok; t += step, ++item) {
            const Item it = item_at(t);
#pragma unroll
            for (int x = 0; x < QUARTER; ++x) acc[x] = 0ull;
            // R to L2, while the windows run
            if (!GLU && p.residual && p.parts == 1 && it.m0 + quad * 32 + lane < p.rows)
                for (int c = it.n0 + col_a; c < it.n0 + col_a + HALF && c < p.cols; c += 32) prefetch_l2(p.residual + static_cast<size_t>(it.m0 + quad * 32 + lane) * p.pitch + c);
            for (int w = it.w0; w < it.w1; ++w, ++window) {
                if (!wait(hh_full_a, window & 1)) break;
                tc_fence_after_sync();
                add_columns(kHh);
                release(hh_free_L);
            }
            if (!ok || !wait(side_full_a, item & 1)) break;
            tc_fence_after_sync();
            if (it.w1 > it.w0) add_columns(kSide);
            const int row0 = it.m0 + quad * 32;
            if (row0 >= p.rows) { release(side_free_L); continue; }
            uint32_t most = 0, least = 0xffffffffu;
#pragma unroll
            for (int x = 0; x < QUARTER; ++x) {
                float a, b;
                unpack2(acc[x], a, b);
                const uint32_t u = __float_as_uint(a) << 1, v = __float_as_uint(b) << 1;
                most = max(most, max(u, v));
                least = min(least, min(u - 1, v - 1));          // (zero as the largest)
            }
            const bool again = __any_sync(0xffffffffu, most >= 0xff000000u || least < 2u * 0x08800000u);
            const int row = row0 + lane;
            // The sums go back to the side columns, which are free now, and come chunk by chunk through one copy of the code below: unrolled over the
            // registers that hold them it took 25 us to fetch (of 111, 2048 x 2048 x 2048), and indexed they would live in local memory.
#pragma unroll
            for (int x = 0; x < HALF; x += 16) {
                uint32_t v[16];
#pragma unroll
                for (int q = 0; q < 16; q += 2) {
                    float a, b;
                    unpack2(acc[(x + q) / 2], a, b);
                    v[q] = __float_as_uint(a); v[q + 1] = __float_as_uint(b);
                }
                tmem_st_32x16(lanes + kSide + (x < QUARTER ? col_a + x : col_b + x - QUARTER), v);
            }
            tmem_st_wait();
            // 32 sums from column c on, or, where some of the warp's do not stand, formed once more (rows past the last as the last)
            auto take = [&](int c, int col0, int hb, float (&f)[32]) {
                if (again) {
                    float formed[32];
                    form_row_f32(p, row < p.rows ? row : p.rows - 1, col0, it.hm, hb, it.w0, it.w1, formed);
#pragma unroll
                    for (int i = 0; i < 32; ++i) f[i] = formed[i];
                    return;
                }
                uint32_t v[32];
                tmem_ld_32x32(lanes + kSide + c, v);
                tmem_ld_wait();
#pragma unroll
                for (int i = 0; i < 32; ++i) f[i] = __uint_as_float(v[i]);
            };
            // (all loads before the first addition; with R in L2 by then 7664 x 420 x 7248 with R and Z took 512 us, now 477)
            auto add = [&](float (&f)[32], const float* from, int col0) {
                float4 v[8];
#pragma unroll
                for (int q = 0; q < 8; ++q) {
                    const float4* at = reinterpret_cast<const float4*>(from + (col0 + 4 * q < p.pitch ? col0 + 4 * q : 0));
                    asm volatile("ld.global.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v[q].x), "=f"(v[q].y), "=f"(v[q].z), "=f"(v[q].w) : "l"(at) : "memory");
                }
#pragma unroll
                for (int q = 0; q < 8; ++q)
                    if (col0 + 4 * q < p.pitch) { f[4 * q] += v[q].x; f[4 * q + 1] += v[q].y; f[4 * q + 2] += v[q].z; f[4 * q + 3] += v[q].w; }
            };
            if constexpr (GLU) {
#pragma unroll 1
                for (int c = 0; c < QUARTER; c += 32) {
                    const int col0 = it.n0 + col_a + c;
                    if (col0 >= p.cols) break;
                    float z[32], u[32];
                    take(col_a + c, col0, 0, z);
                    take(col_b + c, col0, 1, u);
                    if (p.parts > 1) {
                        put(z, [&] { tma_store_4d_a(&tmY, buf, col0, 0, row0, it.part); });
                        put(u, [&] { tma_store_4d_a(&tmY, buf, col0, 1, row0, it.part); });
                        continue;
                    }
                    if (p.bias) { add(z, p.bias, col0); add(u, p.bias + p.pitch, col0); }
                    if (p.keep_z) {
                        put(z, [&] { tma_store_4d_a(&tmZ, buf, col0, 0, row0, 0); });
                        put(u, [&] { tma_store_4d_a(&tmZ, buf, col0, 1, row0, 0); });
                    }
                    with_act(p.act, [&](auto a) {
#pragma unroll
                        for (int i = 0; i < 32; ++i) z[i] = act_value<decltype(a)::value, false>(z[i], p.k) * u[i];
                    });
                    put(z, [&] { tma_store_4d_a(&tmY, buf, col0, 0, row0, 0); });
                }
            } else {
#pragma unroll 1
                for (int c = 0; c < HALF; c += 32) {
                    const int col0 = it.n0 + col_a + c;
                    if (col0 >= p.cols) break;
                    float z[32];
                    take(col_a + c, col0, 0, z);
                    if (p.parts == 1) {
                        if (p.bias) add(z, p.bias, col0);
                        if (p.keep_z) put(z, [&] { tma_store_4d_a(&tmZ, buf, col0, 0, row0, 0); });
                        with_act(p.act, [&](auto a) {
#pragma unroll
                            for (int i = 0; i < 32; ++i) z[i] = act_value<decltype(a)::value, false>(z[i], p.k);
                        });
                        if (p.residual && row < p.rows) add(z, p.residual + static_cast<size_t>(row) * p.pitch, col0);
                    }
                    put(z, [&] { tma_store_4d_a(&tmY, buf, col0, it.hm, row0, it.part); });
                }
            }
            release(side_free_L);
        }
        if (lane == 0) tma_store_wait_all();
    }
    tc_fence_before_sync();
    __syncthreads();
    cluster_sync_all();   // neither CTA leaves while the other may still reach its shared memory
    if (warp == 1) tmem_dealloc_pair(tmem_base, 512);
}

}  // namespace alpha
