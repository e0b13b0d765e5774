// Which kernel a product of 16-bit matrices runs on, and its launch.
#pragma once
#include "fc_mma.cuh"
#include "host_checks.h"

#include <algorithm>

namespace alpha {
namespace {

// Columns from one row (half) to the next of tensors that are OC wide.
int fc_pitch(int OC) { return (OC + 7) / 8 * 8; }

constexpr int kMostDim = 2147483647 - 1023;
int check_fc(const char* what, const AlphaFcShape* s, bool glu)
{
    if (!s) return fail(ALPHA_E_ARG, "%s: null shape", what);
    if (s->rows <= 0 || s->IC <= 0 || s->OC <= 0) return fail(ALPHA_E_ARG, "%s: non-positive dimension (rows=%d IC=%d OC=%d)", what, s->rows, s->IC, s->OC);
    // (a tile's last row or column, past the tensor's, is an int too)
    if (s->rows > kMostDim || s->IC > kMostDim || s->OC > kMostDim) return fail(ALPHA_E_ARG, "%s: dimension of more than %d (rows=%d IC=%d OC=%d)", what, kMostDim, s->rows, s->IC, s->OC);
    if (s->dtype != ALPHA_F32 && s->dtype != ALPHA_BF16 && s->dtype != ALPHA_F16) return fail(ALPHA_E_ARG, "%s: unknown element type %d", what, s->dtype);
    if (s->act < ALPHA_ACT_NONE || s->act > ALPHA_ACT_GELU_TANH) return fail(ALPHA_E_ARG, "%s: unknown activation %d", what, s->act);
    if (s->act == ALPHA_ACT_LEAKY_RELU && !(s->k == s->k)) return fail(ALPHA_E_ARG, "%s: slope is NaN", what);
    const int unit = s->dtype == ALPHA_F32 ? 4 : 8;
    if (s->IC % unit) return fail(ALPHA_E_ARG, "%s: IC=%d must be a multiple of %d (rows of 16-byte words)", what, s->IC, unit);
    const long long wide = (glu ? 2LL : 1LL) * (((long long)s->OC + 7) / 8 * 8), most = 2147483647LL;
    if (wide > most) return fail(ALPHA_E_ARG, "%s: more than 2^31-1 rows of W", what);
    // the fp32 kernels address a tensor's elements with 32 bits
    if (s->dtype == ALPHA_F32 && ((long long)s->rows * s->IC > most || wide * s->IC > most || s->rows * wide > most))
        return fail(ALPHA_E_ARG, "%s: tensor has more than 2^31-1 elements", what);
    return ALPHA_OK;
}

// An operand as three dimensions, innermost first, with the strides of the outer two (elements).
struct Operand { const void* ptr; bool mn; long long d0, d1, d2, s1, s2; };

int make_map(CUtensorMap* m, int dtype, const Operand& o, int b0, int b1, int b2)
{
    const cuuint64_t dims[3] = {(cuuint64_t)o.d0, (cuuint64_t)o.d1, (cuuint64_t)o.d2}, st[2] = {(cuuint64_t)o.s1 * 2, (cuuint64_t)o.s2 * 2};
    const cuuint32_t box[3] = {(cuuint32_t)b0, (cuuint32_t)b1, (cuuint32_t)b2};
    return encode_tiled(m, dtype == ALPHA_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, o.ptr, dims, st, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

// rows x cols outputs (glu: cols of a half; rows of each of m_halves halves) over k_halves halves of K steps.
// A: (step, half, row), or (row, half, step) where it runs along its rows (mn); B: (step, column, half) or (column, step, half).
struct Product {
    int dtype, rows, cols, pitch, K, m_halves, k_halves;
    bool glu;
    Operand A, B;
    const void *bias, *residual;
    void *Z, *Y;
    int act; float k;
    FcLoss loss;                 // epilogues of a loss only
};

// What a product of 16-bit operands runs on: CTA pairs of 256 x 256 outputs, or CTAs of 128 x bn, `split` of which share a tile.
struct FcPlan { bool pair; int bn, split; };

uint32_t tmem_columns(int bn, bool glu)
{
    // two accumulators from multiples of 32 columns on, read by chunks of 32 (glu: from their half on too)
    auto up = [](int n) { return (n + 31) & ~31; };
    const int last = glu && bn / 2 + up(bn / 2) > up(bn) ? bn / 2 + up(bn / 2) : up(bn);
    uint32_t c = 32;
    while (c < static_cast<uint32_t>(up(bn) + last)) c <<= 1;
    return c;
}

// The plan of least estimated time (512 x 4096 x 4096 in us: 64 columns 27.6, 128 22, pairs of 256 columns 27, of 128 19.7; 64 x 4096 x 1024: 64
// columns 13, shared by two 11.6, 32 shared by four 9.7; 2048 x 2048 x 2048: pairs of 256 columns 17.8, of 128 18.7, 128 20).  64 steps of a tile
// take 0.139 us (four MMAs of up to 128 columns, 64 clocks each whatever they hold, as A is read from shared memory), or what the ring's stages leave of a
// copy's latency, or their bytes at the 112 KB/us that one SM takes in: 128 x 128 is bound by these, a pair of 256 x 128 brings three quarters of
// them, one of 256 x 256 (0.32 us) half of them an output.  All tiles' operands come through L2 at 15 TB/s, tensors from and to DRAM at 5.9; a launch 4.4 us
// until its first tile and after its last (pairs 5.8), and a shared tile its exchange, eight CTAs also the wait for a place for them.  Fitted to 1750 measured
// plans of 220 products: 13 % about the measured time, and what is chosen takes 1.009 of the best.
double plan_time(const Product& q, bool pair, int bn, int split, int sms, double* fixed, bool* fits)
{
    const long long cols = q.glu ? 2LL * q.cols : q.cols, blocks = (long long)q.k_halves * ((q.K + kFcBK - 1) / kFcBK);
    const int out = q.glu ? bn / 2 : bn, bm = pair ? 256 : 128, ctas = pair ? 2 : 1;
    const long long tiles = (long long)q.m_halves * ((q.rows + bm - 1) / bm) * ((q.cols + out - 1) / out), most = sms / (ctas * split);
    // (clusters of four or more do not fill every group of SMs: 32 of 37, and a second wave costs as much as the first)
    *fits = most >= 1 && (split == 1 || tiles <= (split < 4 ? most : most * 87 / 100));
    if (!*fits) return 0.0;
    const long long waves = (tiles + most - 1) / most, each = (blocks + split - 1) / split;
    const int a_rows = pair || q.A.mn || q.rows >= 128 ? 128 : (q.rows + 7) / 8 * 8;
    const uint32_t block = fc_block_bytes(pair, a_rows, bn);
    const int ring = static_cast<int>(kFcRing / (fc_blocks(pair, bn) * block));
    const double in = block / 112e3, step = pair ? (bn == 256 ? 0.32 : in) : std::max(std::max(0.139, in), 0.49 / (std::min(ring, (int)kFcMaxStages) - 1));
    const double tile = std::max(each * step, (pair ? 0.28 : 0.68) + 0.0053 * bn);
    const double l2 = (double)tiles * blocks * block * ctas / 15e6;
    const double mma = waves * tile, n = (double)q.rows * q.m_halves;
    const double outputs = q.loss.part ? 0.0 : q.cols + (q.Z ? cols : 0) + (q.residual ? q.cols : 0) + (q.loss.sums ? 4.0 * q.cols : 0.0);
    const double dram = 2e-6 * ((n + cols) * q.K * q.k_halves + n * outputs) / 5.9;
    const double most_of = std::max(mma, std::max(l2, dram));
    *fixed = (pair ? 5.8 : 4.4 + 0.0078 * bn) + (split == 1 ? 0.0 : split == 2 ? 3.0 : split == 4 ? 5.3 : 12.0);
    return 0.86 * most_of + 0.14 * (mma + l2 + dram);                // (the others are not quite hidden)
}
// Two products by one launch: their tiles fill the same waves.
double two_time(const Product& x, const Product& w, const FcPlan& plan, int sms)
{
    double time = 0.0, fixed = 0.0;
    const int most = sms / (plan.pair ? 2 : 1), bm = plan.pair ? 256 : 128;
    double busy = 0.0;
    for (const Product* q : {&x, &w}) {
        bool fits;
        const double t = plan_time(*q, plan.pair, plan.bn, 1, sms, &fixed, &fits);
        const long long tiles = (long long)q->m_halves * ((q->rows + bm - 1) / bm) * ((q->cols + plan.bn - 1) / plan.bn), whole = (tiles + most - 1) / most;
        time += t * tiles / (whole * most);                                      // (what it would be without idle places)
        busy = std::max(busy, t / whole);
    }
    return fixed + std::max(busy, time + 0.5 * busy);
}

// (most_split: a tile's CTAs at most; the epilogues of a loss take whole rows of a tile, which shared tiles do not have)
FcPlan pick_plan(const Product& q, int sms, double* time_of = nullptr, int most_split = 8)
{
    const int forced = option_fc_tile() == 2 || option_fc_tile() == 3 ? 0 : option_fc_tile();
    const long long stages = ((long long)q.k_halves * ((q.K + kFcBK - 1) / kFcBK) + 1) / 2;
    FcPlan best{false, 64, 1};
    double least = 1e300;
    auto look = [&](bool pair, int bn, int split) {
        bool fits;
        double fixed = 0.0, time = plan_time(q, pair, bn, split, sms, &fixed, &fits);
        if (!fits) return;
        time += fixed;
        if (time < least) { least = time; best = FcPlan{pair, bn, split}; }
    };
    // (an operand that runs along its rows comes in boxes of 64 of them; no part of a shared tile is empty)
    const int unit = q.B.mn ? 64 : 16;
    auto parts = [&](int split) { return split == 1 || (split - 1) * ((stages + split - 1) / split) < stages; };
    if ((forced == 1 || forced == 11) && sms >= 2) { look(true, forced == 1 ? 256 : 128, 1); best = FcPlan{true, forced == 1 ? 256 : 128, 1}; }
    else if (forced >= 1000) {
        const int bn = forced % 1000 / unit * unit;
        // (half as many CTAs, and so on, where a part would be empty or the clusters do not run at once)
        for (int split = std::min(forced / 1000, most_split); split > 1 && bn >= unit && bn <= 256 && least == 1e300; split /= 2)
            if (split <= 8 && parts(split)) look(false, bn, split);
        if (least == 1e300 && bn >= unit && bn <= 256) look(false, bn, 1);
    } else {
        look(true, 256, 1);
        look(true, 128, 1);
        for (int bn = unit; bn <= 128; bn += unit)
            for (int split = 1; split <= most_split; split *= 2)
                if (parts(split)) look(false, bn, split);
    }
    if (time_of) *time_of = least;
    return best;
}

// A product as the kernel takes it.
struct Prepared { FcMma p; CUtensorMap a, b; };

int prepare(const Product& q, const FcPlan& plan, int a_rows, int* status, Prepared* out)
{
    const int bm = plan.pair ? 256 : 128, bn = plan.bn, cols_of = q.glu ? bn / 2 : bn, steps = kFcBK * fc_blocks(plan.pair, bn);
    FcMma& p = out->p;
    p = FcMma{};
    p.rows = q.rows; p.cols = q.pitch;
    const int k_blocks = (q.K + kFcBK - 1) / kFcBK;
    p.m_half = (q.rows + bm - 1) / bm; p.n_tiles = (q.cols + cols_of - 1) / cols_of;
    p.k_half = q.k_halves > 1 ? k_blocks : 1 << 29;
    p.kb = static_cast<int>(((long long)k_blocks * q.k_halves * kFcBK + steps - 1) / steps);
    if ((long long)p.m_half * q.m_halves * p.n_tiles > 2147483647LL / (2 * kFcGroupM)) return fail(ALPHA_E_ARG, "fullConnect: more tiles than a launch takes");
    p.m_tiles = p.m_half * q.m_halves;
    p.bn = bn; p.split = plan.split;
    p.a_mn = q.A.mn; p.b_mn = q.B.mn; p.a_rows = a_rows;
    const uint32_t stage = fc_blocks(plan.pair, bn) * fc_block_bytes(plan.pair, a_rows, bn);
    p.stages = kFcRing / stage < kFcMaxStages ? kFcRing / stage : kFcMaxStages;
    // shared tiles: the ring holds a part's sums afterwards
    const uint32_t sums = (q.rows < 128 ? q.rows : 128) * (bn + 4) * 4;
    while (p.split > 1 && p.stages * stage < sums && (p.stages + 1) * stage <= kFcRing) ++p.stages;
    if (p.split > 1 && p.stages * stage < sums) return fail(ALPHA_E_ARG, "fullConnect: no plan");
    p.idesc = q.dtype == ALPHA_BF16 ? make_idesc_bf16(bm, bn, q.A.mn, q.B.mn) : make_idesc_f16(bm, bn, q.A.mn, q.B.mn);
    p.tmem = tmem_columns(bn, q.glu);
    p.act = q.act; p.k = q.k; p.keep_z = q.Z != nullptr;
    p.bias = q.bias; p.residual = q.residual; p.Y = q.Y; p.Z = q.Z; p.status = status;
    p.loss = q.loss;
    if (p.loss.parts < 1) p.loss.parts = 1;
    const int rc = q.A.mn ? make_map(&out->a, q.dtype, q.A, 64, 1, 64) : make_map(&out->a, q.dtype, q.A, 64, 1, a_rows);
    if (rc) return rc;
    return q.B.mn ? make_map(&out->b, q.dtype, q.B, 64, 64, 1) : make_map(&out->b, q.dtype, q.B, 64, plan.pair ? bn / 2 : cols_of, 1);
}

template <class T, int PAIR, bool GLU, bool TWO, int EPI>
void launch_mma(const Prepared& x, const Prepared& y, int sms, cudaStream_t stream)
{
    const FcMma& p = x.p;
    const int group = PAIR ? 2 : p.split, total = p.m_tiles * p.n_tiles * p.loss.parts + (TWO ? y.p.m_tiles * y.p.n_tiles : 0), most = sms / group;
    const unsigned grid = static_cast<unsigned>(p.split > 1 || total < most ? total : most) * group;
    const uint32_t smem = p.stages * fc_blocks(PAIR != 0, p.bn) * fc_block_bytes(PAIR != 0, p.a_rows, p.bn) + kFcStaging + 1024 + 512;
    allow_smem<fc_mma_kernel<T, PAIR, GLU, TWO, EPI>>();
    launch_after_clusters(fc_mma_kernel<T, PAIR, GLU, TWO, EPI>, dim3(grid), kFcThreads, group > 1 ? group : 0, smem, stream, x.a, x.b, x.p, y.a, y.b, y.p);
}

// One product, or (other != nullptr) two of one type without gates by one launch.
template <int EPI = kFcLayer>
int launch_planned(const Product& q, const Product* other, const FcPlan& plan, int sms, int* status, cudaStream_t stream)
{
    Prepared x, y;
    const int a_rows = plan.pair || q.A.mn || other || q.rows >= 128 ? 128 : (q.rows + 7) / 8 * 8;
    int rc = prepare(q, plan, a_rows, status, &x);
    if (!rc && other) rc = prepare(*other, plan, a_rows, status, &y);
    if (rc) return rc;
    const Prepared& z = other ? y : x;
    auto go = [&](auto t) {
        using T = decltype(t);
        auto by = [&](auto pair) {
            constexpr int PAIR = decltype(pair)::value;
            if constexpr (EPI == kFcLayer || EPI == kFcSum)
                if (other) return launch_mma<T, PAIR, false, true, EPI>(x, z, sms, stream);
            if constexpr (EPI == kFcLayer)
                if (q.glu) return launch_mma<T, PAIR, true, false, EPI>(x, z, sms, stream);
            launch_mma<T, PAIR, false, false, EPI>(x, z, sms, stream);
        };
        if (!plan.pair) by(std::integral_constant<int, 0>{});
        else if (plan.bn == 256) by(std::integral_constant<int, 256>{});
        else by(std::integral_constant<int, 128>{});
    };
    if (q.dtype == ALPHA_BF16) go(__nv_bfloat16{});
    else go(__half{});
    note_launch("fc");
    note_plan("fc %s%s%dx%d split=%d", other ? "two " : "", plan.pair ? "pair " : "", plan.pair ? 256 : 128, plan.bn, plan.split);
    return launched("fc_mma_kernel");
}

template <int EPI = kFcLayer>
int launch_product(const Product& q, cudaStream_t stream)
{
    int sms = 0, *status = nullptr;
    int rc = device_sms(&sms);
    if (!rc) rc = device_status_word(&status);
    return rc ? rc : launch_planned<EPI>(q, nullptr, pick_plan(q, sms, nullptr, EPI == kFcStats || EPI == kFcSoftmaxDelta ? 1 : 8), sms, status, stream);
}

// deltaX and deltaW: by a launch each, or together where the waves of both take less than those of either and a second launch's fill and drain.
// (Chosen for 120 drawn bf16 shapes: 1.30 times as fast as apart in the geometric mean, 395 x 344 x 480 6.3 us instead of 11.9; slower for 15 of them, 5330 x 400 x 600 36 instead of 30.
// Estimates within 3 % of one another are no reason for it.)
template <int EPI = kFcLayer>
int launch_products(const Product& x, const Product& w, cudaStream_t stream)
{
    int sms = 0, *status = nullptr;
    int rc = device_sms(&sms);
    if (!rc) rc = device_status_word(&status);
    if (rc) return rc;
    FcPlan plan{false, 0, 1}, best{false, 0, 1};
    double apart = 0.0, least = 1e300;
    const FcPlan px = pick_plan(x, sms, &apart), pw = pick_plan(w, sms, &least);
    apart += least;
    least = 1e300;
    const int forced = option_fc_tile();
    for (int form = 0; form < 4 && x.rows >= 128; ++form) {
        plan = form < 2 ? FcPlan{true, form ? 128 : 256, 1} : FcPlan{false, form == 2 ? 128 : 64, 1};
        if ((plan.pair && sms < 2) || (forced == 1 && form != 0) || (forced == 11 && form != 1) || forced == 3 || forced >= 1000) continue;
        const double time = two_time(x, w, plan, sms);
        if (time < least) { least = time; best = plan; }
    }
    if (best.bn && least < 0.97 * apart) return launch_planned<EPI>(x, &w, best, sms, status, stream);
    rc = launch_planned<EPI>(x, nullptr, px, sms, status, stream);
    return rc ? rc : launch_planned<EPI>(w, nullptr, pw, sms, status, stream);
}
// deltaX of a loss, its reduction over the classes in parts of its own tiles, beside deltaW (or alone) in one launch of CTA pairs.
struct PartsPlan { int bn, parts; double time; };
PartsPlan pick_parts(const Product& x, const Product* w, int sms)
{
    PartsPlan best{0, 1, 1e300};
    const int pairs = sms / 2, forced = option_fc_tile();
    if (pairs < 1 || forced == 3 || forced >= 1000) return best;
    const long long kx = (x.K + 63) / 64, kw = w ? (w->K + 63) / 64 : 0;
    double bytes = 2.0 * ((double)(x.rows + x.cols) * x.K + (double)x.rows * x.cols);
    if (w) bytes += 2.0 * ((double)(w->rows + w->cols) * w->K + (double)w->rows * w->cols);
    for (int bn = 256; bn >= 128; bn /= 2) {
        if (forced == (bn == 256 ? 11 : 1)) continue;
        // (a stage holds two blocks of 64 steps where columns are 128)
        const int unit = fc_blocks(true, bn);
        const double step = bn == 256 ? 0.32 : fc_block_bytes(true, 128, bn) / 112e3, least = 0.28 + 0.0053 * bn;
        const long long tx = (long long)((x.rows + 255) / 256) * ((x.cols + bn - 1) / bn), tw = w ? (long long)((w->rows + 255) / 256) * ((w->cols + bn - 1) / bn) : 0, stages = (kx + unit - 1) / unit;
        // (where the tiles alone fill the pairs parts save nothing)
        for (int parts = 2; parts <= 16 && parts <= stages && tx < pairs; ++parts) {
            const long long each = (stages + parts - 1) / parts, items = tx * parts;
            if ((parts - 1) * each >= stages) continue;
            const double cx = std::max(each * unit * step, least) + 0.3, cw = std::max(kw * step, least) + 0.3;
            double busy = 0.0;
            for (int i = 0; i < pairs; ++i) {
                const long long nx = items > i ? (items - i + pairs - 1) / pairs : 0, all = items + tw > i ? (items + tw - i + pairs - 1) / pairs : 0;
                busy = std::max(busy, nx * cx + (all - nx) * cw);
            }
            const double joined = 3.5 + (double)x.rows * x.cols * 4e-6 * (parts + 1) / 5.0;
            const double time = 5.8 + std::max(busy, bytes * 1e-6 / 5.9) + joined;
            if (time < best.time) best = PartsPlan{bn, parts, time};
        }
    }
    return best;
}

}  // namespace
}  // namespace alpha
