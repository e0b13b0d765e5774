// FullConnect layers of a transformer: products with bias, activation and residual in their epilogue, the gated block, and their gradients.
#include "../../include/alpha_conv_b200.h"
#include "fc_delta.cuh"
#include "fc_f32.cuh"
#include "fc_mma.cuh"
#include "fc_pair_f32.cuh"
#include "fc_small.cuh"
#include "host_common.h"

#include <algorithm>
#include <initializer_list>

using namespace alpha;

namespace {

size_t type_bytes(int dtype) { return dtype == ALPHA_F32 ? 4 : 2; }
// Columns from one row (half) to the next of tensors that are OC wide.
int fc_pitch(int OC) { return (OC + 7) / 8 * 8; }

struct Span { const void* ptr; size_t bytes; };
bool overlap(const Span& a, const Span& b)
{
    const uintptr_t x = reinterpret_cast<uintptr_t>(a.ptr), y = reinterpret_cast<uintptr_t>(b.ptr);
    return a.ptr && b.ptr && x < y + b.bytes && y < x + a.bytes;
}
// What a call writes must overlap neither what it reads nor what else it writes.
int check_spans(const char* what, std::initializer_list<Span> in, std::initializer_list<Span> out)
{
    for (const Span* o = out.begin(); o != out.end(); ++o) {
        for (const Span& i : in)
            if (overlap(*o, i)) return fail(ALPHA_E_ARG, "%s: an output overlaps an input", what);
        for (const Span* q = out.begin(); q != o; ++q)
            if (overlap(*o, *q)) return fail(ALPHA_E_ARG, "%s: two outputs overlap", what);
    }
    for (auto list : {in, out})
        for (const Span& s : list)
            if (reinterpret_cast<uintptr_t>(s.ptr) & 15) return fail(ALPHA_E_ARG, "%s: tensor pointers must be 16-byte aligned", what);
    return ALPHA_OK;
}

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

int launched(const char* what)
{
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? ALPHA_OK : fail(ALPHA_E_CUDA, "%s launch failed: %s", what, cudaGetErrorString(e));
}

// ---- 16-bit products --------------------------------------------------------------------------------------------

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
    const double dram = 2e-6 * ((n + cols) * q.K * q.k_halves + n * (q.cols + (q.Z ? cols : 0) + (q.residual ? q.cols : 0))) / 5.9;
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

FcPlan pick_plan(const Product& q, int sms, double* time_of = nullptr)
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
        for (int split = forced / 1000; split > 1 && bn >= unit && bn <= 256 && least == 1e300; split /= 2)
            if (split <= 8 && parts(split)) look(false, bn, split);
        if (least == 1e300 && bn >= unit && bn <= 256) look(false, bn, 1);
    } else {
        look(true, 256, 1);
        look(true, 128, 1);
        for (int bn = unit; bn <= 128; bn += unit)
            for (int split = 1; split <= 8; split *= 2)
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
    const int rc = q.A.mn ? make_map(&out->a, q.dtype, q.A, 64, 1, 64) : make_map(&out->a, q.dtype, q.A, 64, 1, a_rows);
    if (rc) return rc;
    return q.B.mn ? make_map(&out->b, q.dtype, q.B, 64, 64, 1) : make_map(&out->b, q.dtype, q.B, 64, plan.pair ? bn / 2 : cols_of, 1);
}

template <class T, int PAIR, bool GLU, bool TWO>
void launch_mma(const Prepared& x, const Prepared& y, int sms, cudaStream_t stream)
{
    const FcMma& p = x.p;
    const int group = PAIR ? 2 : p.split, total = p.m_tiles * p.n_tiles + (TWO ? y.p.m_tiles * y.p.n_tiles : 0), most = sms / group;
    const unsigned grid = static_cast<unsigned>(p.split > 1 || total < most ? total : most) * group;
    const uint32_t smem = p.stages * fc_blocks(PAIR != 0, p.bn) * fc_block_bytes(PAIR != 0, p.a_rows, p.bn) + kFcStaging + 1024 + 512;
    allow_smem<fc_mma_kernel<T, PAIR, GLU, TWO>>();
    launch_after_clusters(fc_mma_kernel<T, PAIR, GLU, TWO>, dim3(grid), kFcThreads, group > 1 ? group : 0, smem, stream, x.a, x.b, x.p, y.a, y.b, y.p);
}

// One product, or (other != nullptr) two of one type without gates by one launch.
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
            if (other) launch_mma<T, PAIR, false, true>(x, z, sms, stream);
            else if (q.glu) launch_mma<T, PAIR, true, false>(x, z, sms, stream);
            else launch_mma<T, PAIR, false, false>(x, z, sms, stream);
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

int launch_product(const Product& q, cudaStream_t stream)
{
    int sms = 0, *status = nullptr;
    int rc = device_sms(&sms);
    if (!rc) rc = device_status_word(&status);
    return rc ? rc : launch_planned(q, nullptr, pick_plan(q, sms), sms, status, stream);
}

// deltaX and deltaW: by a launch each, or together where the waves of both take less than those of either and a second launch's fill and drain.
// (Chosen for 120 drawn bf16 shapes: 1.30 times as fast as apart in the geometric mean, 395 x 344 x 480 6.3 us instead of 11.9; slower for 15 of them, 5330 x 400 x 600 36 instead of 30.
// Estimates within 3 % of one another are no reason for it.)
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
    if (best.bn && least < 0.97 * apart) return launch_planned(x, &w, best, sms, status, stream);
    rc = launch_planned(x, nullptr, px, sms, status, stream);
    return rc ? rc : launch_planned(w, nullptr, pw, sms, status, stream);
}

// ---- fp32 products ----------------------------------------------------------------------------------------------

template <bool GLU>
int launch_parts(const float* part, size_t size, int parts, int rows, const FcEpilogue& e, int sms, cudaStream_t stream)
{
    const int per_row = e.cols / (GLU ? 2 : 4);
    const size_t words = static_cast<size_t>(rows) * per_row, blocks = (words + 255) / 256;
    launch_after(fc_parts_kernel<GLU>, static_cast<unsigned>(blocks < sms * 8u ? blocks : sms * 8u), 256, 0, stream, part, size, parts, fast_div(per_row), words, e);
    note_launch("fc");
    return launched("fc_parts_kernel");
}

// A product of fp32 matrices as PlaneFc forms it: rows x cols sums over K steps (padding of both halves of Z among rows, columns or steps).
struct ProductF32 { const float *A, *B; int rows, cols, K, OC, pitch, halves, lda, ldb; FcEpilogue e; };

// Planes of a matrix in scratch: [plane][row][pitch], pitch in bf16 elements.
struct Planes { void* ptr = nullptr; const float* src = nullptr; int rows = 0, cols = 0, pitch = 0; };
Planes planes_of(const float* src, int rows, int cols) { return Planes{nullptr, src, rows, cols, (cols + 7) / 8 * 8}; }
size_t plane_bytes(const Planes& p) { return (6 * static_cast<size_t>(p.rows) * p.pitch + 255) & ~static_cast<size_t>(255); }
unsigned most_split_ctas(int sms) { return static_cast<unsigned>(sms) * 16; }
int launch_split(const Planes* const* list, int n, uint32_t* seen, int* ctas, int sms, cudaStream_t stream)
{
    SplitJobs j{};
    j.seen = seen;
    for (int i = 0; i < n; ++i) {
        const Planes& p = *list[i];
        j.job[j.n++] = SplitJob{p.src, static_cast<uint2*>(p.ptr), static_cast<unsigned>(p.rows), static_cast<unsigned>(p.cols / 4), j.total, fast_div(p.pitch / 4)};
        j.total += static_cast<unsigned>(p.rows) * static_cast<unsigned>(p.pitch / 4);
    }
    const unsigned blocks = (j.total + 255) / 256, most = most_split_ctas(sms);
    *ctas = static_cast<int>(blocks < most ? blocks : most);
    launch_after(fc_split_kernel, *ctas, 256, 0, stream, j);
    note_launch("fc");
    return launched("fc_split_kernel");
}

// Columns of a pair's tile, parts of the reduction, and the time of that product (us): a window of 64 steps of a tile 2.26 (1.34 with 128 columns, whose tiles
// fill the waves more evenly), a tile 2 (1.8), a launch 5; the parts written and read.  Measured / estimated, with the split of the operands, over 150 products
// of 2 to 60 GFLOP: 0.97 with a deviation of 10 % (0.95, 7 %); what is chosen takes 1.003 of the best.
struct PairPlan { int bn, parts; double time; };
PairPlan pick_pair(int rows, int m_halves, int out_cols, bool glu, int K, int k_halves, int sms)
{
    const int pairs = sms / 2, windows = k_halves * ((K + 63) / 64);
    PairPlan best{256, 1, 1e300};
    if (pairs < 1) return best;
    for (int bn = 256; bn >= 128; bn /= 2) {
        if (option_fc_tile() == (bn == 256 ? 11 : 1)) continue;
        const int out = glu ? bn / 2 : bn;
        const double tiles = static_cast<double>(m_halves) * ((rows + 255) / 256) * ((out_cols + out - 1) / out), size = static_cast<double>(rows) * m_halves * out_cols * (glu ? 2 : 1);
        for (int parts = 1; parts <= 32 && parts <= windows; ++parts) {
            const int each = (windows + parts - 1) / parts;
            if ((parts - 1) * each >= windows) continue;                      // (no part is empty)
            // (sums formed once more take 0.1 us a step and 32 columns, 0.8 s of 32768 windows: a pair's next item waits 2 s at most.  All SMs need no such
            // tensor as fits for a second item of that length, a few of them may)
            if (each > 32768 && tiles * parts > pairs) continue;
            const double waves = static_cast<double>(static_cast<long long>((tiles * parts + pairs - 1) / pairs));
            const double time = 5.0 + waves * (bn == 256 ? each * 2.26 + 2.0 : each * 1.34 + 1.8) + (parts > 1 ? 3.0 + size * 4e-6 * (2 * parts + 1) / 6.0 : 0.0);
            if (time < best.time) best = PairPlan{bn, parts, time};
        }
    }
    return best;
}
double split_time(size_t elements) { return 2.0 + elements * 10e-6 / 8.0; }

template <int FORM>
int launch_pair(const ProductF32& q, const Planes& A, const Planes& B, const PairPlan& plan, void* part, const uint32_t* seen, int seen_n, int sms, int* status, cudaStream_t stream)
{
    constexpr bool GLU = FORM == kFcGlu, A_MN = FORM == kFcDeltaW, B_MN = FORM == kFcDeltaX || FORM == kFcDeltaW;
    const bool forward = FORM == kFcForward || FORM == kFcGlu;
    const int bn = plan.bn, parts = plan.parts, out = GLU ? bn / 2 : bn, m_halves = A_MN ? q.halves : 1, k_halves = FORM == kFcDeltaX ? q.halves : 1;
    const int cols = forward ? q.OC : q.cols, steps = FORM == kFcDeltaX ? q.OC : q.K;
    PairF32 p{};
    p.rows = A_MN ? q.OC : q.rows; p.cols = cols; p.pitch = q.e.cols; p.K = steps;
    p.m_half = (p.rows + 255) / 256; p.m_tiles = p.m_half * m_halves; p.n_tiles = (cols + out - 1) / out;
    const int windows = (steps + 63) / 64;
    p.w_half = k_halves > 1 ? windows : 1 << 29; p.windows = windows * k_halves; p.parts = parts;
    p.a_mn = A_MN; p.b_mn = B_MN;
    p.idesc = make_idesc_bf16(256, bn, A_MN, B_MN);
    p.A = q.A; p.B = q.B;
    p.a_row = A_MN ? 1 : q.lda; p.a_k = A_MN ? q.lda : 1; p.a_half = q.pitch;
    p.b_col = B_MN ? 1 : q.ldb; p.b_k = B_MN ? q.ldb : 1; p.b_half = static_cast<long long>(q.OC) * q.ldb;
    p.bias = q.e.bias; p.residual = q.e.residual; p.act = q.e.act; p.k = q.e.k; p.keep_z = parts == 1 && q.e.Z;
    p.status = status; p.seen = seen; p.seen_n = seen_n;
    // sums and results: (column, half of the columns or rows, row, part)
    const int out_pitch = forward ? q.pitch : q.cols;
    const size_t size = static_cast<size_t>(p.rows) * m_halves * out_pitch * (GLU ? 2 : 1);
    void* ws = parts > 1 ? part : q.e.Y;
    // operands: (step, half, row, plane) or (row, half, step, plane) for A; (step, column, half, plane) or (column, step, half, plane) for B
    auto map = [](CUtensorMap* m, const Planes& s, long long d0, long long d1, long long d2, long long s1, long long s2, int b1, int b2) {
        const cuuint64_t dims[4] = {(cuuint64_t)d0, (cuuint64_t)d1, (cuuint64_t)d2, 3}, st[3] = {(cuuint64_t)s1 * 2, (cuuint64_t)s2 * 2, (cuuint64_t)s.pitch * 2 * s.rows};
        const cuuint32_t box[4] = {64, (cuuint32_t)b1, (cuuint32_t)b2, 1};
        return encode_tiled(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, s.ptr, dims, st, box, CU_TENSOR_MAP_SWIZZLE_128B);
    };
    auto out_map = [&](CUtensorMap* m, const void* base, int h, bool by_rows, int copies) {
        const long long row = by_rows ? out_pitch : static_cast<long long>(out_pitch) * h, half = by_rows ? static_cast<long long>(out_pitch) * p.rows : out_pitch;
        const cuuint64_t dims[4] = {(cuuint64_t)cols, (cuuint64_t)h, (cuuint64_t)p.rows, (cuuint64_t)copies}, st[3] = {(cuuint64_t)half * 4, (cuuint64_t)row * 4, (cuuint64_t)out_pitch * 4 * h * p.rows};
        const cuuint32_t box[4] = {32, 1, 32, 1};
        return encode_tiled(m, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 4, base, dims, st, box, CU_TENSOR_MAP_SWIZZLE_128B);
    };
    CUtensorMap a, b, y, z;
    const long long OC = q.OC, pa = A.pitch, pb = B.pitch;
    int rc;
    if constexpr (FORM == kFcDeltaX) {
        rc = map(&a, A, OC, q.halves, q.rows, q.pitch, pa, 1, 128);
        if (!rc) rc = map(&b, B, q.cols, OC, q.halves, pb, OC * pb, 64, 1);
    } else if constexpr (FORM == kFcDeltaW) {
        rc = map(&a, A, OC, q.halves, q.K, q.pitch, pa, 1, 64);
        if (!rc) rc = map(&b, B, q.cols, q.K, 1, pb, q.K * pb, 64, 1);
    } else {
        rc = map(&a, A, q.K, 1, q.rows, pa, pa, 1, 128);
        if (!rc) rc = map(&b, B, q.K, OC, q.halves, pb, OC * pb, bn / 2, 1);
    }
    if (!rc) rc = A_MN ? out_map(&y, ws, q.halves, true, parts) : out_map(&y, ws, GLU && parts > 1 ? 2 : 1, false, parts);
    if (!rc) rc = p.keep_z ? out_map(&z, q.e.Z, GLU ? 2 : 1, false, 1) : (z = y, ALPHA_OK);
    if (rc) return rc;
    const long long items = static_cast<long long>(p.m_tiles) * p.n_tiles * parts;
    const unsigned pairs = static_cast<unsigned>(items < sms / 2 ? items : sms / 2);
    auto go = [&](auto width) {
        constexpr int BN = decltype(width)::value;
        allow_smem<fc_pair_f32_kernel<GLU, BN>>();
        launch_after_clusters(fc_pair_f32_kernel<GLU, BN>, dim3(2 * pairs), kPairF32Threads, 2, pair_f32_smem(BN), stream, a, b, y, z, p);
    };
    if (bn == 256) go(std::integral_constant<int, 256>{});
    else go(std::integral_constant<int, 128>{});
    note_launch("fc");
    note_plan("fc planes pair 256x%d parts=%d", bn, parts);
    rc = launched("fc_pair_f32_kernel");
    return rc || parts == 1 ? rc : launch_parts<GLU>(static_cast<const float*>(ws), size, parts, p.rows * m_halves, q.e, sms, stream);
}

// The same from the fp32 tensors as they lie; without `may_split` in no scratch.
template <int FORM>
int launch_gathered(const ProductF32& q, const PlanePlan& plan, int sms, int* status, cudaStream_t stream)
{
    int slice = 0;
    int rc = planes_launch_slice(&slice);
    if (rc) return rc;
    PlaneFc<FORM> p{};
    p.A = q.A; p.B = q.B; p.rows = q.rows; p.cols = q.cols; p.K = q.K; p.OC = q.OC; p.pitch = q.pitch; p.lda = q.lda; p.ldb = q.ldb; p.e = q.e;
    const int out_rows = FORM == kFcDeltaW ? q.halves * q.OC : q.rows;
    p.size = static_cast<size_t>(out_rows) * q.cols;
    p.ksplit = plan.ksplit;
    if (p.ksplit > 1) {
        void* ws = nullptr;
        rc = call_scratch(stream, p.ksplit * p.size * sizeof(float), &ws);
        if (rc) return rc;
        p.part = static_cast<float*>(ws);
    }
    if (dry_run()) return ALPHA_OK;
    const dim3 grid((q.rows + kPlaneBM - 1) / kPlaneBM, (q.cols + plan.bn - 1) / plan.bn, p.ksplit);
    launch_planes(p, plan.bn, grid, slice, stream, status);
    note_launch("fc");
    note_plan("fc planes 128x%d ksplit=%d", plan.bn, p.ksplit);
    rc = launched("gemm_planes_kernel");
    return rc || p.ksplit == 1 ? rc : launch_parts<FORM == kFcGlu>(p.part, p.size, p.ksplit, out_rows, q.e, sms, stream);
}

template <int FORM> PlanePlan pick_gathered(const ProductF32& q, int sms, int most = 16)
{
    PlanePlan plan = plan_planes(q.rows, q.cols, q.K, 1, most, static_cast<double>(q.rows) * q.cols, 0, sms);
    plan.time *= 1.2;         // (measured / estimated of 150 products 1.26 in the mean, 10 % about it: both operands are split as they are staged, and come from DRAM)
    return plan;
}
// In any case: without parts where their scratch is refused.
template <int FORM> int run_gathered(const ProductF32& q, int sms, int* status, cudaStream_t stream)
{
    const int rc = launch_gathered<FORM>(q, pick_gathered<FORM>(q, sms), sms, status, stream);
    return rc && scratch_refused(rc) ? launch_gathered<FORM>(q, pick_gathered<FORM>(q, sms, 1), sms, status, stream) : rc;
}

// One or two products by pairs over operands that are split together; 1 where their scratch is refused (nothing has been launched then).
struct PairWork {
    Planes p[3];
    int n = 0;
    size_t parts = 0;          // bytes of the larger of the products' parts
    int sms = 0, *status = nullptr;
    void* part = nullptr;
    uint32_t* seen = nullptr; int seen_n = 0;
    int add(const float* src, int rows, int cols) { p[n] = planes_of(src, rows, cols); return n++; }
    void want(const ProductF32& q, int k) { const size_t bytes = k > 1 ? k * static_cast<size_t>(q.rows) * q.cols * sizeof(float) : 0; if (bytes > parts) parts = bytes; }   // (padding too)
    size_t elements() const { size_t e = 0; for (int i = 0; i < n; ++i) e += static_cast<size_t>(p[i].rows) * p[i].pitch; return e; }
    bool fits() const { return elements() < 4ull << 31; }           // 32-bit indices of words of four
    int split(cudaStream_t stream)
    {
        const size_t seen_bytes = (most_split_ctas(sms) * sizeof(uint32_t) + 255) & ~static_cast<size_t>(255);
        size_t bytes = parts + seen_bytes;
        for (int i = 0; i < n; ++i) bytes += plane_bytes(p[i]);
        void* ws = nullptr;
        const int rc = call_scratch(stream, bytes, &ws);
        if (rc) return scratch_refused(rc) ? 1 : rc;
        if (dry_run()) return ALPHA_OK;
        char* at = static_cast<char*>(ws);
        seen = reinterpret_cast<uint32_t*>(at);
        at += seen_bytes;
        for (int i = 0; i < n; ++i) { p[i].ptr = at; at += plane_bytes(p[i]); }
        part = at;
        const Planes* list[3] = {&p[0], &p[1], &p[2]};
        return launch_split(list, n, seen, &seen_n, sms, stream);
    }
};

// Option FC_TILE: 1 or 11 pairs, 2 never, else where their estimated time is less.
bool pairs_pay(double pair, double other)
{
    const int forced = option_fc_tile();
    return forced == 1 || forced == 11 || (forced != 2 && pair < other);
}

template <int FORM>
int forward_f32(const ProductF32& q, cudaStream_t stream)
{
    PairWork w;
    int rc = device_sms(&w.sms);
    if (!rc) rc = device_status_word(&w.status);
    if (rc) return rc;
    const PairPlan pair = pick_pair(q.rows, 1, q.OC, FORM == kFcGlu, q.K, 1, w.sms);
    const int a = w.add(q.A, q.rows, q.K), b = w.add(q.B, q.halves * q.OC, q.K);
    w.want(q, pair.parts);
    if (w.sms >= 2 && w.fits() && pairs_pay(pair.time + split_time(w.elements()), pick_gathered<FORM>(q, w.sms).time)) {
        rc = w.split(stream);
        if (rc == 0) return dry_run() ? ALPHA_OK : launch_pair<FORM>(q, w.p[a], w.p[b], pair, w.part, w.seen, w.seen_n, w.sms, w.status, stream);
        if (rc < 0) return rc;
    }
    return run_gathered<FORM>(q, w.sms, w.status, stream);
}

// deltaX = dZ W and deltaW = dZ^T X (either may be missing).
int delta_f32(const float* dZ, const float* X, const float* W, float* dX, float* dW, int rows, int OC, int halves, int IC, cudaStream_t stream)
{
    const FcEpilogue plain{nullptr, nullptr, nullptr, nullptr, IC, ALPHA_ACT_NONE, 0.f};
    const int pitch = fc_pitch(OC), wide = halves * pitch;
    ProductF32 x{dZ, W, rows, IC, wide, OC, pitch, halves, wide, IC, plain}, w{dZ, X, wide, IC, rows, OC, pitch, halves, wide, IC, plain};
    x.e.Y = dX; w.e.Y = dW;
    int sms = 0, *status = nullptr;
    int rc = device_sms(&sms);
    if (!rc) rc = device_status_word(&status);
    if (rc) return rc;
    // which of them by pairs: both share the planes of dZ
    const PairPlan px = pick_pair(rows, 1, IC, false, OC, halves, sms), pw = pick_pair(OC, halves, IC, false, rows, 1, sms);
    const double gx = pick_gathered<kFcDeltaX>(x, sms).time, gw = pick_gathered<kFcDeltaW>(w, sms).time;
    PairWork best;
    bool best_x = false, best_w = false;
    double least = 1e300;
    for (int form = 0; form < 4; ++form) {
        const bool bx = form & 1, bw = form & 2;
        if ((bx && !dX) || (bw && !dW) || (form && sms < 2)) continue;
        if ((option_fc_tile() == 1 || option_fc_tile() == 11) && sms >= 2 && (bx != (dX != nullptr) || bw != (dW != nullptr))) continue;
        if (option_fc_tile() == 2 && form) continue;
        PairWork v;
        v.sms = sms; v.status = status;
        if (form) v.add(dZ, rows, wide);
        if (bx) { v.add(W, halves * OC, IC); v.want(x, px.parts); }
        if (bw) { v.add(X, rows, IC); v.want(w, pw.parts); }
        if (!v.fits()) continue;
        const double time = (dX ? (bx ? px.time : gx) : 0.0) + (dW ? (bw ? pw.time : gw) : 0.0) + (form ? split_time(v.elements()) : 0.0);
        if (time < least) { least = time; best = v; best_x = bx; best_w = bw; }
    }
    if (best.n) {
        rc = best.split(stream);
        if (rc < 0) return rc;
        if (rc == 1) best_x = best_w = false;
    }
    rc = ALPHA_OK;
    if (best_x && !dry_run()) rc = launch_pair<kFcDeltaX>(x, best.p[0], best.p[1], px, best.part, best.seen, best.seen_n, sms, status, stream);
    if (!rc && best_w && !dry_run()) rc = launch_pair<kFcDeltaW>(w, best.p[0], best.p[best_x ? 2 : 1], pw, best.part, best.seen, best.seen_n, sms, status, stream);
    if (!rc && dX && !best_x) rc = run_gathered<kFcDeltaX>(x, sms, status, stream);
    if (!rc && dW && !best_w) rc = run_gathered<kFcDeltaW>(w, sms, status, stream);
    return rc;
}

// ---- few rows ---------------------------------------------------------------------------------------------------

constexpr int kSmallRows = 4, kTokenRows = 16;   // fp32, 16-bit

template <bool GLU>
int launch_small(const AlphaFcShape* s, const void* X, const void* W, const void* bias, const void* residual, void* Z, void* Y, cudaStream_t stream)
{
    int sms = 0;
    const int rc = device_sms(&sms);
    if (rc) return rc;
    FcSmall p{s->rows, s->IC, s->OC, fc_pitch(s->OC), 1, 1, s->act, s->k, X, W, bias, residual, Z, Y};
    const int units = GLU ? s->OC : (s->OC + 1) / 2, words = s->IC / 4;
    // 16 warps an SM, each with 64 words of a row at least
    while (p.ks < 8 && static_cast<long long>(units) * p.ks < 16LL * sms && words >= 128 * p.ks) p.ks *= 2;
    const int teams = 8 / p.ks;
    const unsigned blocks = (units + teams - 1) / teams;
    if (s->rows == 1) launch_after(fc_small_kernel<1, GLU>, blocks, 256, 0, stream, p);
    else if (s->rows == 2) launch_after(fc_small_kernel<2, GLU>, blocks, 256, 0, stream, p);
    else launch_after(fc_small_kernel<4, GLU>, blocks, 256, 0, stream, p);
    note_launch("fc_small");
    note_plan("fc small ks=%d", p.ks);
    return launched("fc_small_kernel");
}
template <class T, bool GLU>
int launch_token(const AlphaFcShape* s, const void* X, const void* W, const void* bias, const void* residual, void* Z, void* Y, cudaStream_t stream)
{
    int sms = 0;
    const int rc = device_sms(&sms);
    if (rc) return rc;
    FcSmall p{s->rows, s->IC, s->OC, fc_pitch(s->OC), 1, 1, s->act, s->k, X, W, bias, residual, Z, Y};
    // up to eight warps a row group, each with 4 blocks of 32 steps at least
    while (p.ks < 8 && s->IC >= 256 * p.ks) p.ks *= 2;
    const int teams = 8 / p.ks, groups = (s->OC + 15) / 16;
    const long long blocks = (groups + teams - 1) / teams;
    // row groups that leave SMs to fill are shared, as long as a warp keeps its 32-byte loads of eight rows in flight
    const int pass = 64 * 8 * 4;
    while (p.split < 8 && p.ks == 8 && blocks * p.split * 2 <= 4LL * sms && s->IC >= pass * p.split * 2) p.split *= 2;
    if (blocks * p.split > 2147483647LL) p.split = 1;
    const dim3 grid(static_cast<unsigned>(blocks * p.split));
    const unsigned cluster = p.split > 1 ? p.split : 0;
    if (s->rows <= 8) launch_after_clusters(fc_token_kernel<T, 1, GLU>, grid, 256, cluster, 0, stream, p);
    else launch_after_clusters(fc_token_kernel<T, 2, GLU>, grid, 256, cluster, 0, stream, p);
    note_launch("fc_small");
    note_plan("fc token ks=%d split=%d", p.ks, p.split);
    return launched("fc_token_kernel");
}

int forward(const AlphaFcShape* s, const void* X, const void* W, const void* bias, const void* residual, void* Z, void* Y, bool glu, cudaStream_t stream)
{
    int rc = call_begin(stream);
    if (rc) return rc;
    // Of the gated block from nine rows on only where W is small.  us of bf16, 9 to 16 rows, W from DRAM, this kernel / tiles: 2 x 1024 x 1024 5.4-5.9 / 6.6-7.0, 2 x 2752 x
    // 1024 6.7 / 7.3, 2 x 2048 x 2048 9.6 / 9.5, 2 x 4096 x 2048 11.5 / 10.8, 2 x 5504 x 4096 31 / 20, 2 x 11008 x 4096 49 / 35; without gates 1024 x 1024 3.5 / 6.9, 4096 x
    // 4096 10.9 / 12.9, 5504 x 4096 12 / 15.8, 11008 x 4096 23.0 / 21.4, 8192 x 8192 27 / 28.
    const bool token = s->rows <= 8 || (s->rows <= kTokenRows && (!glu || (long long)s->OC * s->IC <= 4 << 20));
    if ((s->dtype == ALPHA_F32 ? s->rows <= kSmallRows : token) && (!option_fc_tile() || option_fc_tile() == 3)) {
        if (dry_run()) return ALPHA_OK;
        switch (s->dtype) {
        case ALPHA_F32: return glu ? launch_small<true>(s, X, W, bias, residual, Z, Y, stream) : launch_small<false>(s, X, W, bias, residual, Z, Y, stream);
        case ALPHA_BF16:
            return glu ? launch_token<__nv_bfloat16, true>(s, X, W, bias, residual, Z, Y, stream) : launch_token<__nv_bfloat16, false>(s, X, W, bias, residual, Z, Y, stream);
        default: return glu ? launch_token<__half, true>(s, X, W, bias, residual, Z, Y, stream) : launch_token<__half, false>(s, X, W, bias, residual, Z, Y, stream);
        }
    }
    if (s->dtype == ALPHA_F32) {
        const int pitch = fc_pitch(s->OC);
        const FcEpilogue e{static_cast<const float*>(bias), static_cast<const float*>(residual), static_cast<float*>(Z), static_cast<float*>(Y), pitch, s->act, s->k};
        const float *x = static_cast<const float*>(X), *w = static_cast<const float*>(W);
        return glu ? forward_f32<kFcGlu>(ProductF32{x, w, s->rows, 2 * pitch, s->IC, s->OC, pitch, 2, s->IC, s->IC, e}, stream)
                   : forward_f32<kFcForward>(ProductF32{x, w, s->rows, pitch, s->IC, s->OC, pitch, 1, s->IC, s->IC, e}, stream);
    }
    if (dry_run()) return ALPHA_OK;
    const long long IC = s->IC, OC = s->OC;
    return launch_product(Product{s->dtype, s->rows, s->OC, fc_pitch(s->OC), s->IC, 1, 1, glu, Operand{X, false, IC, 1, s->rows, IC, IC}, Operand{W, false, IC, OC, glu ? 2 : 1, IC, OC * IC},
                                  bias, residual, Z, Y, s->act, s->k}, stream);
}

template <class T, bool GLU>
int launch_delta(const AlphaFcShape* s, const void* dY, const void* Z, void* dZ, void* dB, cudaStream_t stream)
{
    int sms = 0;
    int rc = device_sms(&sms);
    if (rc) return rc;
    const int pitch = fc_pitch(s->OC), wide = GLU ? 2 * pitch : pitch, words = pitch / Word16<T>::N;
    const unsigned gy = (words + 31) / 32;
    // one wave of CTAs, four rows of a warp at least
    long long gx = sms * static_cast<long long>(delta_ctas<GLU>()) / gy;
    if (gx < 1) gx = 1;
    const long long by_rows = (s->rows + 31) / 32;
    if (gx > by_rows) gx = by_rows;
    FcDelta p{s->rows, pitch, s->OC, s->act, s->k, dY, Z, dZ, nullptr};
    if (dB) {
        void* ws = nullptr;
        rc = call_scratch(stream, static_cast<size_t>(gx) * wide * sizeof(float), &ws);
        if (rc) return rc;
        p.part = static_cast<float*>(ws);
    }
    if (dry_run()) return ALPHA_OK;
    launch_after(fc_delta_kernel<T, GLU>, dim3(gy, static_cast<unsigned>(gx)), 256, 0, stream, p);
    note_launch("fc_delta");
    rc = launched("fc_delta_kernel");
    if (rc || !dB) return rc;
    launch_after(fc_bias_kernel<T>, (wide + 31) / 32, 256, 0, stream, p.part, static_cast<int>(gx), wide, static_cast<T*>(dB));
    note_launch("fc_delta");
    return launched("fc_bias_kernel");
}

int delta(const char* what, const AlphaFcShape* s, const void* dY, const void* X, const void* W, const void* Z, void* dZ, void* dX, void* dW, void* dB, bool glu,
          cudaStream_t stream)
{
    int rc = check_fc(what, s, glu);
    if (rc) return rc;
    const bool through = glu || s->act != ALPHA_ACT_NONE;           // dZ is not deltaY
    if (!dY || (dX && !W) || (dW && !X)) return fail(ALPHA_E_ARG, "%s: null tensor pointer", what);
    if (!dX && !dW && !dB) return fail(ALPHA_E_ARG, "%s: no gradient asked for", what);
    if (through && (!Z || !dZ)) return fail(ALPHA_E_ARG, "%s: Z of the forward pass and memory for deltaZ are needed (deltaZ may be Z)", what);
    const size_t b = type_bytes(s->dtype), pitch = fc_pitch(s->OC), wide = (glu ? 2 : 1) * pitch, units = (glu ? 2 : 1) * static_cast<size_t>(s->OC), rows = s->rows;
    if (!through) { Z = nullptr; dZ = nullptr; }
    const Span in_z{dZ == Z ? nullptr : Z, rows * wide * b};
    rc = check_spans(what, {{dY, rows * pitch * b}, {dW ? X : nullptr, rows * s->IC * b}, {dX ? W : nullptr, units * s->IC * b}, in_z},
                     {{dZ, rows * wide * b}, {dX, rows * s->IC * b}, {dW, units * s->IC * b}, {dB, wide * b}});
    if (!rc) rc = call_begin(stream);
    if (rc) return rc;
    if (through || dB) {
        switch (s->dtype) {
        case ALPHA_F32: rc = glu ? launch_delta<float, true>(s, dY, Z, dZ, dB, stream) : launch_delta<float, false>(s, dY, Z, dZ, dB, stream); break;
        case ALPHA_BF16: rc = glu ? launch_delta<__nv_bfloat16, true>(s, dY, Z, dZ, dB, stream) : launch_delta<__nv_bfloat16, false>(s, dY, Z, dZ, dB, stream); break;
        default: rc = glu ? launch_delta<__half, true>(s, dY, Z, dZ, dB, stream) : launch_delta<__half, false>(s, dY, Z, dZ, dB, stream);
        }
        if (rc) return rc;
    }
    const void* d = through ? dZ : dY;
    if (s->dtype == ALPHA_F32)
        return delta_f32(static_cast<const float*>(d), static_cast<const float*>(X), static_cast<const float*>(W), static_cast<float*>(dX), static_cast<float*>(dW), s->rows, s->OC,
                         glu ? 2 : 1, s->IC, stream);
    if (dry_run()) return ALPHA_OK;
    const long long IC = s->IC, OC = s->OC, p = pitch, n = s->rows;
    const int halves = glu ? 2 : 1;
    const Product x{s->dtype, s->rows, s->IC, s->IC, s->OC, 1, halves, false, Operand{d, false, OC, halves, n, p, halves * p}, Operand{W, true, IC, OC, halves, IC, OC * IC},
                    nullptr, nullptr, nullptr, dX, ALPHA_ACT_NONE, 0.f};
    const Product w{s->dtype, s->OC, s->IC, s->IC, s->rows, halves, 1, false, Operand{d, true, OC, halves, n, p, halves * p}, Operand{X, true, IC, n, 1, IC, n * IC},
                    nullptr, nullptr, nullptr, dW, ALPHA_ACT_NONE, 0.f};
    if (dX && dW) return launch_products(x, w, stream);
    if (dX) rc = launch_product(x, stream);
    if (dW) rc = launch_product(w, stream);
    return rc;
}

}  // namespace

extern "C" {

int alpha_fullConnect(const AlphaFcShape* s, const void* X, const void* W, const void* bias, const void* residual, void* Z, void* Y, alpha_stream_t stream)
{
    OpRange range("alpha_fullConnect");
    int rc = check_fc("fullConnect", s, false);
    if (rc) return rc;
    if (!X || !W || !Y) return fail(ALPHA_E_ARG, "fullConnect: null tensor pointer");
    const size_t b = type_bytes(s->dtype), pitch = fc_pitch(s->OC), y = s->rows * pitch * b;
    if (reinterpret_cast<uintptr_t>(residual) & 15) return fail(ALPHA_E_ARG, "fullConnect: tensor pointers must be 16-byte aligned");
    rc = check_spans("fullConnect", {{X, static_cast<size_t>(s->rows) * s->IC * b}, {W, static_cast<size_t>(s->OC) * s->IC * b}, {bias, pitch * b}, {residual == Y ? nullptr : residual, y}},
                     {{Y, y}, {Z, y}});
    return rc ? rc : forward(s, X, W, bias, residual, Z, Y, false, static_cast<cudaStream_t>(stream));
}

int alpha_fullConnect_glu(const AlphaFcShape* s, const void* X, const void* W, const void* bias, void* Z, void* Y, alpha_stream_t stream)
{
    OpRange range("alpha_fullConnect_glu");
    int rc = check_fc("fullConnect_glu", s, true);
    if (rc) return rc;
    if (!X || !W || !Y) return fail(ALPHA_E_ARG, "fullConnect_glu: null tensor pointer");
    const size_t b = type_bytes(s->dtype), pitch = fc_pitch(s->OC), y = s->rows * pitch * b;
    rc = check_spans("fullConnect_glu", {{X, static_cast<size_t>(s->rows) * s->IC * b}, {W, 2 * static_cast<size_t>(s->OC) * s->IC * b}, {bias, 2 * pitch * b}}, {{Y, y}, {Z, 2 * y}});
    return rc ? rc : forward(s, X, W, bias, nullptr, Z, Y, true, static_cast<cudaStream_t>(stream));
}

int alpha_fullConnect_delta(const AlphaFcShape* s, const void* deltaY, const void* X, const void* W, const void* Z, void* deltaZ, void* deltaX, void* deltaW, void* deltaB,
                            alpha_stream_t stream)
{
    OpRange range("alpha_fullConnect_delta");
    return delta("fullConnect_delta", s, deltaY, X, W, Z, deltaZ, deltaX, deltaW, deltaB, false, static_cast<cudaStream_t>(stream));
}

int alpha_fullConnect_glu_delta(const AlphaFcShape* s, const void* deltaY, const void* X, const void* W, const void* Z, void* deltaZ, void* deltaX, void* deltaW, void* deltaB,
                                alpha_stream_t stream)
{
    OpRange range("alpha_fullConnect_glu_delta");
    return delta("fullConnect_glu_delta", s, deltaY, X, W, Z, deltaZ, deltaX, deltaW, deltaB, true, static_cast<cudaStream_t>(stream));
}

int alpha_fullConnect_workspace_bytes(const AlphaFcShape* s, int glu, int op, size_t* bytes)
{
    if (!s || !bytes) return fail(ALPHA_E_ARG, "fullConnect_workspace_bytes: null argument");
    if (op != ALPHA_OP_FORWARD && op != ALPHA_OP_DELTAX) return fail(ALPHA_E_ARG, "fullConnect_workspace_bytes: unknown op %d", op);
    // the call itself with launches switched off: what it asks for is what it will ask for (tensors at placeholder addresses far apart)
    auto at = [](int i) { return reinterpret_cast<void*>(static_cast<uintptr_t>(i + 1) << 44); };
    dry_begin();
    int rc;
    if (op == ALPHA_OP_FORWARD) rc = glu ? alpha_fullConnect_glu(s, at(0), at(1), at(2), at(3), at(4), nullptr) : alpha_fullConnect(s, at(0), at(1), at(2), nullptr, at(3), at(4), nullptr);
    else rc = (glu ? alpha_fullConnect_glu_delta : alpha_fullConnect_delta)(s, at(0), at(1), at(2), at(3), at(4), at(5), at(6), at(7), nullptr);
    *bytes = dry_end();
    return rc;
}

}  // extern "C"
