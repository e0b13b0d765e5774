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
// Elements that planes cannot hold (Inf, NaN, what rounds to Inf in h) arrive as NaN; of elements below 2^-110 the planes drop bits below 2^-133, and
// the launch that splits says so, with the largest magnitude it saw.  A warp that finds a sum that is not finite, or below 2^-110 and not zero, or so small that
// what its operands lost may matter to it, forms those 32 rows x 32 columns once more by FMAs from the fp32 tensors, in ascending k, staged through its own
// shared memory.  us of the gradients of 512 x 4096 -> 1000 / 4096 x 1024 -> 2048: ordinary data 73 / 180, a softmax with tails to 1e-45 in deltaY 88 / 195 (where
// every word with a tiny element became NaN, and a lane read its operands from global memory step by step, 3930 / 16200), dead units beside one tiny
// element 135 / 400, an Inf 500 / 1860 (4060 / 17640), all elements times 1e-36 515 / 1895.
// Warps: 0 TMA producer, 1 MMA issuer (of the leader), 2-9 epilogue: 128 running sums a thread.
#pragma once
#include "fc_f32.cuh"

namespace alpha {

constexpr int kPairF32Threads = 320, kPairF32Slots = 6;
constexpr uint32_t kPairF32Operand = 128 * 128;                                    // 128 rows of A of a CTA, 64 steps of a plane
__host__ __device__ constexpr uint32_t pair_f32_slot(int bn) { return kPairF32Operand + bn / 2 * 128; }
__host__ __device__ constexpr uint32_t pair_f32_smem(int bn) { return kPairF32Slots * pair_f32_slot(bn) + 8 * 4096 + 1024 + 256; }

// Magnitudes are compared as bits shifted left by one, without their sign: these are Inf and 2^-110.
constexpr uint32_t kInfBits = 0xff000000u, kTinyBits = 2u * 0x08800000u;

// Up to three fp32 matrices as planes, dst[plane][row][pitch]; columns past cols are zeros.  seen[CTA]: the largest magnitude that it split, and in the lowest
// bit whether planes lost bits of an element.
struct SplitJob { const float* src; uint2* dst; unsigned rows, cols4, first; FastDiv by_pitch4; };
struct SplitJobs { SplitJob job[3]; int n; unsigned total; uint32_t* seen; };
__global__ void __launch_bounds__(256) fc_split_kernel(const __grid_constant__ SplitJobs p)
{
    __shared__ uint32_t of_warp[8];
    grid_dependency_wait();
    grid_dependency_trigger();
    uint32_t top = 0, dropped = 0;
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
        uint32_t x0 = __float_as_uint(v.x) << 1, x1 = __float_as_uint(v.y) << 1, x2 = __float_as_uint(v.z) << 1, x3 = __float_as_uint(v.w) << 1;
        if (lost & 0xffffu) {
            auto look = [&](uint32_t& x, uint32_t& word, int shift) {
                if ((word >> shift & 0x7f80u) == 0x7f80u) { word |= 0x7fffu << shift; x = 0; }
                else if (x && x < kTinyBits) dropped = 1;
            };
            look(x0, h.x, 0); look(x1, h.x, 16); look(x2, h.y, 0); look(x3, h.y, 16);
        }
        top = max(max(top, max(x0, x1)), max(x2, x3));
        const size_t plane = static_cast<size_t>(j.rows) * j.by_pitch4.d;
        j.dst[i] = h; j.dst[plane + i] = m; j.dst[2 * plane + i] = l;
    }
    top = __reduce_max_sync(0xffffffffu, top);
    dropped = __reduce_or_sync(0xffffffffu, dropped);
    if ((threadIdx.x & 31) == 0) of_warp[threadIdx.x >> 5] = top | dropped;
    __syncthreads();
    if (threadIdx.x) return;
    top = dropped = 0;
    for (uint32_t w : of_warp) { top = max(top, w & ~1u); dropped |= w & 1u; }
    p.seen[blockIdx.x] = top | dropped;
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
    const uint32_t* seen; int seen_n;   // of the launch that split the operands
};

// 32 rows of an operand x 16 steps, as a warp loads them: four words of four a lane, zeros past the last row or step.
struct OperandRows {
    const float* at; long long row, k; int rows;     // element (r, k) at at[r * row + k * k]; one of the two strides is 1
    int lane;
    __device__ bool along_k() const { return k == 1; }
    __device__ int r_of(int j) const { return along_k() ? (lane >> 2) + 8 * j : 4 * (lane & 7); }
    __device__ int k_of(int j) const { return along_k() ? 4 * (lane & 3) : (lane >> 3) + 4 * j; }
    // rows r0 ... r0 + 31, steps k0 ... k0 + 15 of K
    __device__ void load(float4 (&v)[4], int r0, int k0, int K) const
    {
        const float* first = at + (r0 + r_of(0)) * row + (k0 + k_of(0)) * k;
        const long long next = along_k() ? 8 * row : 4 * k;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            v[j] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (r0 + r_of(j) < rows && k0 + k_of(j) < K) v[j] = __ldg(reinterpret_cast<const float4*>(first + j * next));
        }
        if (along_k() && k0 + 16 > K)
#pragma unroll
            for (int j = 0; j < 4; ++j) keep_first(v[j], K - k0 - k_of(j));
    }
    // As [step][row] of 16 x 32 floats, rows rotated by 8 for every four steps so that neither form of store meets a bank twice.
    __device__ void stage(uint32_t to, const float4 (&v)[4]) const
    {
        if (along_k()) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t a = to + (k_of(j) * 32 + ((r_of(j) + 2 * k_of(j)) & 31)) * 4;
                const float f[4] = {v[j].x, v[j].y, v[j].z, v[j].w};
#pragma unroll
                for (int e = 0; e < 4; ++e) asm volatile("st.shared.f32 [%0], %1;" ::"r"(a + e * 128), "f"(f[e]) : "memory");
            }
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) st_shared_v4(to + (k_of(j) * 32 + ((r_of(j) + 8 * j) & 31)) * 4, v[j]);
        }
    }
};
__device__ __forceinline__ OperandRows rows_of_a(const PairF32& p, int h, int lane) { return OperandRows{p.A + h * p.a_half, p.a_row, p.a_k, p.rows, lane}; }
__device__ __forceinline__ OperandRows rows_of_b(const PairF32& p, int h, int lane) { return OperandRows{p.B + h * p.b_half, p.b_col, p.b_k, p.cols, lane}; }

// 32 rows x 32 columns of a product, of halves ha and hb of the operands' rows, over windows [w0, w1).
struct SumsAt { int row0, col0, ha, hb, w0, w1; };

// Those sums as FMAs in ascending k, by a whole warp over its own 4 KB of shared memory: four rows x eight columns a lane, then the lane's row to z.
__device__ __forceinline__ void form_sums_f32(const PairF32& p, const SumsAt& s, uint32_t buf, float* z)
{
    const int lane = threadIdx.x & 31, rows4 = 4 * (lane >> 2), cols8 = 8 * (lane & 3), blocks = (s.w1 - s.w0) * 4;
    unsigned long long acc[4][4];
#pragma unroll
    for (int y = 0; y < 4; ++y)
#pragma unroll
        for (int x = 0; x < 4; ++x) acc[y][x] = 0ull;
    float4 a[4], b[4];
    auto load = [&](int i) {
        const int w = s.w0 + (i >> 2), hk = w >= p.w_half ? 1 : 0, k0 = (w - hk * p.w_half) * 64 + (i & 3) * 16;
        rows_of_a(p, s.ha + hk, lane).load(a, s.row0, k0, p.K);
        rows_of_b(p, s.hb + hk, lane).load(b, s.col0, k0, p.K);
    };
    const OperandRows ra = rows_of_a(p, 0, lane), rb = rows_of_b(p, 0, lane);
    load(0);
    for (int i = 0; i < blocks; ++i) {
        __syncwarp();
        ra.stage(buf, a);
        rb.stage(buf + 2048, b);
        __syncwarp();
        if (i + 1 < blocks) load(i + 1);
#pragma unroll
        for (int k = 0; k < 16; ++k) {
            const float4 x = ld_shared_v4(buf + (k * 32 + ((rows4 + 8 * (k >> 2)) & 31)) * 4);
            const float4 y = ld_shared_v4(buf + 2048 + (k * 32 + ((cols8 + 8 * (k >> 2)) & 31)) * 4);
            const float4 u = ld_shared_v4(buf + 2048 + (k * 32 + ((cols8 + 4 + 8 * (k >> 2)) & 31)) * 4);
            const unsigned long long b0 = pack2(y.x, y.y), b1 = pack2(y.z, y.w), b2 = pack2(u.x, u.y), b3 = pack2(u.z, u.w);
            const float f[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const unsigned long long v = pack2(f[r], f[r]);
                ffma2(acc[r][0], v, b0); ffma2(acc[r][1], v, b1); ffma2(acc[r][2], v, b2); ffma2(acc[r][3], v, b3);
            }
        }
    }
    __syncwarp();
    // to the lanes of the rows: 16-byte word q of row r at place q ^ (r & 7)
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float4 o;
            unpack2(acc[r][2 * h], o.x, o.y);
            unpack2(acc[r][2 * h + 1], o.z, o.w);
            st_shared_v4(buf + (rows4 + r) * 128 + (((cols8 >> 2) + h) ^ ((rows4 + r) & 7)) * 16, o);
        }
    __syncwarp();
#pragma unroll
    for (int q = 0; q < 8; ++q) {
        const float4 o = ld_shared_v4(buf + lane * 128 + (q ^ (lane & 7)) * 16);
        z[4 * q] = o.x; z[4 * q + 1] = o.y; z[4 * q + 2] = o.z; z[4 * q + 3] = o.w;
    }
}

// Which of 32 rows of an operand hold anything, and anything below 2^-110 (bit r, in all lanes).
struct RowsHold { uint32_t any, tiny; };
template <bool ALONG_K>
__device__ __forceinline__ RowsHold look_at(const PairF32& p, bool b, int r0, int h, int w0, int w1)
{
    const int lane = threadIdx.x & 31;
    uint32_t bits[4] = {}, least[4] = {0xffffffffu, 0xffffffffu, 0xffffffffu, 0xffffffffu};     // of a word's row, or of its four
    const int blocks = (w1 - w0) * 4;
    for (int i = 0; i < blocks; i += 4) {
        float4 v[4][4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int w = w0 + (i >> 2), hk = w >= p.w_half ? 1 : 0, k0 = (w - hk * p.w_half) * 64 + u * 16;
            const OperandRows o = b ? rows_of_b(p, h + hk, lane) : rows_of_a(p, h + hk, lane);
            o.load(v[u], r0, k0, p.K);
        }
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t x[4] = {__float_as_uint(v[u][j].x) << 1, __float_as_uint(v[u][j].y) << 1, __float_as_uint(v[u][j].z) << 1, __float_as_uint(v[u][j].w) << 1};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    bits[ALONG_K ? j : e] |= x[e];
                    least[ALONG_K ? j : e] = min(least[ALONG_K ? j : e], x[e] - 1);               // (zero as the largest)
                }
            }
    }
    RowsHold o{0, 0};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int r = ALONG_K ? (lane >> 2) + 8 * j : 4 * (lane & 7) + j;
        if (bits[j]) o.any |= 1u << r;
        if (least[j] < kTinyBits) o.tiny |= 1u << r;
    }
    o.any = __reduce_or_sync(0xffffffffu, o.any);
    o.tiny = __reduce_or_sync(0xffffffffu, o.tiny);
    return o;
}
static __device__ __noinline__ RowsHold rows_hold(const PairF32& p, bool b, int r0, int h, int w0, int w1)
{
    return (b ? p.b_mn : p.a_mn) ? look_at<false>(p, b, r0, h, w0, w1) : look_at<true>(p, b, r0, h, w0, w1);
}

// A lane's row z of sums, some of which may not stand: those that are not finite, or below 2^-110 and not zero; or below `least` (as bits) where what the planes
// dropped may matter, that is where row and column both hold something and either of them something tiny.  (A row or column of zeros gives zeros: dead
// units, padded batches.)  Where any of the warp's does not, all are formed once more.
static __device__ __noinline__ void stand_or_form(const PairF32& p, const SumsAt& s, uint32_t least, uint32_t buf, RowsHold& rows, bool& known, float* z)
{
    const int lane = threadIdx.x & 31;
    bool again = false;
    uint32_t small = 0;
#pragma unroll
    for (int i = 0; i < 32; ++i) {
        const uint32_t x = __float_as_uint(z[i]) << 1;
        if (x >= kInfBits || x - 1 < kTinyBits) again = true;
        if (x < least && s.col0 + i < p.cols) small |= 1u << i;
    }
    if (s.row0 + lane >= p.rows) small = 0;
    again = __any_sync(0xffffffffu, again);
    if (!again && __any_sync(0xffffffffu, small)) {
        if (!known) { rows = rows_hold(p, false, s.row0, s.ha, s.w0, s.w1); known = true; }
        if (!(rows.any >> lane & 1)) small = 0;
        if (__any_sync(0xffffffffu, small)) {
            const RowsHold cols = rows_hold(p, true, s.col0, s.hb, s.w0, s.w1);
            small &= cols.any & (rows.tiny >> lane & 1 ? 0xffffffffu : cols.tiny);
            again = __any_sync(0xffffffffu, small);
        }
    }
    if (!again) return;
    if (lane == 0) tma_store_wait_read<0>();
    form_sums_f32(p, s, buf, z);
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
    uint32_t *tmem_holder = reinterpret_cast<uint32_t*>(bars + 2 * S + 4), *of_warp = tmem_holder + 1;
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
        // what the launch that split has seen, while the first copies are under way: an eighth of it a warp
        uint32_t top = 0, dropped = 0;
        for (int i = threadIdx.x - 64; i < p.seen_n; i += 256) {
            const uint32_t w = p.seen[i];
            top = max(top, w & ~1u);
            dropped |= w & 1u;
        }
        top = __reduce_max_sync(0xffffffffu, top);
        dropped = __reduce_or_sync(0xffffffffu, dropped);
        if (lane == 0) of_warp[warp - 2] = top | dropped;
        asm volatile("bar.sync 1, 256;" ::: "memory");
#pragma unroll
        for (int i = 0; i < 8; ++i) { top = max(top, of_warp[i] & ~1u); dropped |= of_warp[i] & 1u; }
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
            // less than 2^-133 of an element, times its partner, for each of two operands and every step, is less than 2^-24 of a sum from here on
            const uint32_t least = dropped ? __float_as_uint(__uint_as_float(top >> 1) * static_cast<float>((it.w1 - it.w0) * 64) * 0x1p-108f) << 1 : 0u;
            RowsHold rows_hold_ = {0, 0};
            bool rows_known = false;
            // 32 sums from column c on, formed once more where some of the warp's do not stand.  (What few tiles need is kept out of line: the code is fetched once a tile.)
            auto take = [&](int c, int col0, int hb, float (&f)[32]) {
                uint32_t v[32], most = 0, none = 0xffffffffu;
                tmem_ld_32x32(lanes + kSide + c, v);
                tmem_ld_wait();
#pragma unroll
                for (int i = 0; i < 32; ++i) {
                    f[i] = __uint_as_float(v[i]);
                    most = max(most, v[i] << 1);
                    none = min(none, (v[i] << 1) - 1);               // (zero as the largest)
                }
                if (!__any_sync(0xffffffffu, most >= kInfBits || none < kTinyBits || least)) return;
                float formed[32];
#pragma unroll
                for (int i = 0; i < 32; ++i) formed[i] = f[i];
                stand_or_form(p, SumsAt{row0, col0, it.hm, hb, it.w0, it.w1}, least, buf, rows_hold_, rows_known, formed);
#pragma unroll
                for (int i = 0; i < 32; ++i) f[i] = formed[i];
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
