// FullConnect layers of a transformer: products with bias, activation and residual in their epilogue, the gated block, and their gradients.
#include "../../include/alpha_conv_b200.h"
#include "fc_delta.cuh"
#include "fc_f32.cuh"
#include "fc_pair_f32.cuh"
#include "fc_product.cuh"
#include "fc_small.cuh"

using namespace alpha;

namespace {

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

// A product as the kernel of pairs takes it.
struct PairItems { CUtensorMap a, b, y, z; PairF32 p; size_t size; const float* ws; };
template <int FORM>
int prepare_pair(const ProductF32& q, const Planes& A, const Planes& B, const PairPlan& plan, void* part, const uint32_t* seen, int seen_n, int* status, PairItems* out_items)
{
    constexpr bool GLU = FORM == kFcGlu, A_MN = FORM == kFcDeltaW, B_MN = FORM == kFcDeltaX || FORM == kFcDeltaW;
    const bool forward = FORM == kFcForward || FORM == kFcGlu;
    const int bn = plan.bn, parts = plan.parts, out = GLU ? bn / 2 : bn, m_halves = A_MN ? q.halves : 1, k_halves = FORM == kFcDeltaX ? q.halves : 1;
    const int cols = forward ? q.OC : q.cols, steps = FORM == kFcDeltaX ? q.OC : q.K;
    PairF32& p = out_items->p;
    p = PairF32{};
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
    CUtensorMap &a = out_items->a, &b = out_items->b, &y = out_items->y, &z = out_items->z;
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
    out_items->size = size;
    out_items->ws = static_cast<const float*>(ws);
    return rc;
}
template <int FORM>
int launch_pair(const ProductF32& q, const Planes& A, const Planes& B, const PairPlan& plan, void* part, const uint32_t* seen, int seen_n, int sms, int* status, cudaStream_t stream,
                bool join = true)
{
    constexpr bool GLU = FORM == kFcGlu;
    PairItems x;
    int rc = prepare_pair<FORM>(q, A, B, plan, part, seen, seen_n, status, &x);
    if (rc) return rc;
    const int bn = plan.bn, parts = plan.parts;
    const long long items = static_cast<long long>(x.p.m_tiles) * x.p.n_tiles * parts;
    const unsigned pairs = static_cast<unsigned>(items < sms / 2 ? items : sms / 2);
    auto go = [&](auto width) {
        constexpr int BN = decltype(width)::value;
        allow_smem<fc_pair_f32_kernel<GLU, BN>>();
        launch_after_clusters(fc_pair_f32_kernel<GLU, BN>, dim3(2 * pairs), kPairF32Threads, 2, pair_f32_smem(BN), stream, x.a, x.b, x.y, x.z, x.p);
    };
    if (bn == 256) go(std::integral_constant<int, 256>{});
    else go(std::integral_constant<int, 128>{});
    note_launch("fc");
    note_plan("fc planes pair 256x%d parts=%d", bn, parts);
    rc = launched("fc_pair_f32_kernel");
    const int m_halves = FORM == kFcDeltaW ? q.halves : 1;
    return rc || parts == 1 || !join ? rc : launch_parts<GLU>(x.ws, x.size, parts, x.p.rows * m_halves, q.e, sms, stream);
}

// deltaX and deltaW by one launch: its columns, the parts of either, and its time (us).  Their items fill the waves together, and one launch's start is saved
// (softmax cross entropy gradients of 256 x 512 x 1000: 34 us instead of 42 with two; 1024 x 2048 x 1000: 86 instead of 97; 512 x 4096 x 1000: 97 either way).
struct TwoPairs { int bn, x_parts, w_parts; double time; size_t part_bytes; };
TwoPairs pick_two_pairs(int rows, int IC, int OC, int sms)
{
    TwoPairs best{0, 1, 1, 1e300, 0};
    const int pairs = sms / 2, x_windows = (OC + 63) / 64, w_windows = (rows + 63) / 64;
    const double x_size = static_cast<double>(rows) * IC, w_size = static_cast<double>(OC) * IC;
    for (int bn = 256; bn >= 128; bn /= 2) {
        if (option_fc_tile() == (bn == 256 ? 11 : 1)) continue;
        const double window = bn == 256 ? 2.26 : 1.34, tile = bn == 256 ? 2.0 : 1.8;
        const long long xt = static_cast<long long>((rows + 255) / 256) * ((IC + bn - 1) / bn), wt = static_cast<long long>((OC + 255) / 256) * ((IC + bn - 1) / bn);
        for (int xp = 1; xp <= 8 && xp <= x_windows; ++xp) {
            for (int wp = 1; wp <= 8 && wp <= w_windows; ++wp) {
                const int xe = (x_windows + xp - 1) / xp, we = (w_windows + wp - 1) / wp;
                if ((xp - 1) * xe >= x_windows || (wp - 1) * we >= w_windows || xe > 8192 || we > 8192) continue;
                const long long xi = xt * xp, wi = wt * wp;
                // (a pair's items of either: the counts change at the two remainders only)
                double busy = 0.0;
                for (const long long i : {0ll, xi % pairs, (xi + wi) % pairs}) {
                    const long long nx = xi > i ? (xi - i + pairs - 1) / pairs : 0, all = xi + wi > i ? (xi + wi - i + pairs - 1) / pairs : 0;
                    busy = std::max(busy, nx * (xe * window + tile) + (all - nx) * (we * window + tile));
                }
                const double time = 5.0 + busy + (xp > 1 ? 3.0 + x_size * 4e-6 * (2 * xp + 1) / 6.0 : 0.0) + (wp > 1 ? 3.0 + w_size * 4e-6 * (2 * wp + 1) / 6.0 : 0.0);
                if (time < best.time) best = TwoPairs{bn, xp, wp, time, static_cast<size_t>(((xp > 1 ? xp * x_size : 0.0) + (wp > 1 ? wp * w_size : 0.0)) * 4) + 512};
            }
        }
    }
    return best;
}
int launch_two_pairs(const ProductF32& x, const ProductF32& w, const Planes& X, const Planes& W, const Planes& Z, const TwoPairs& plan, void* part, const uint32_t* seen, int seen_n, int sms, int* status,
                     cudaStream_t stream)
{
    const size_t x_bytes = plan.x_parts > 1 ? (plan.x_parts * static_cast<size_t>(x.rows) * x.cols * 4 + 255) & ~static_cast<size_t>(255) : 0;
    PairItems a, b;
    int rc = prepare_pair<kFcDeltaX>(x, Z, W, PairPlan{plan.bn, plan.x_parts, 0.0}, part, seen, seen_n, status, &a);
    if (!rc) rc = prepare_pair<kFcDeltaW>(w, Z, X, PairPlan{plan.bn, plan.w_parts, 0.0}, static_cast<char*>(part) + x_bytes, seen, seen_n, status, &b);
    if (rc) return rc;
    const long long items = static_cast<long long>(a.p.m_tiles) * a.p.n_tiles * plan.x_parts + static_cast<long long>(b.p.m_tiles) * b.p.n_tiles * plan.w_parts;
    const unsigned pairs = static_cast<unsigned>(items < sms / 2 ? items : sms / 2);
    auto go = [&](auto width) {
        constexpr int BN = decltype(width)::value;
        allow_smem<fc_pair_f32_two_kernel<BN>>();
        launch_after_clusters(fc_pair_f32_two_kernel<BN>, dim3(2 * pairs), kPairF32Threads, 2, pair_f32_smem(BN), stream, a.a, a.b, a.y, a.p, b.a, b.b, b.y, b.p);
    };
    if (plan.bn == 256) go(std::integral_constant<int, 256>{});
    else go(std::integral_constant<int, 128>{});
    note_launch("fc");
    note_plan("fc planes two pair 256x%d parts=%d,%d", plan.bn, plan.x_parts, plan.w_parts);
    rc = launched("fc_pair_f32_two_kernel");
    if (!rc && plan.x_parts > 1) rc = launch_parts<false>(a.ws, a.size, plan.x_parts, a.p.rows, x.e, sms, stream);
    if (!rc && plan.w_parts > 1) rc = launch_parts<false>(b.ws, b.size, plan.w_parts, b.p.rows, w.e, sms, stream);
    return rc;
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
    // (the first `now` of them; room for what a second launch sees of the others)
    int split(cudaStream_t stream, int now = 3)
    {
        const size_t seen_bytes = (most_split_ctas(sms) * (now < n ? 2 : 1) * sizeof(uint32_t) + 255) & ~static_cast<size_t>(255);
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
        return launch_split(list, now < n ? now : n, seen, &seen_n, sms, stream);
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

// (of a call that has begun)
int forward(const AlphaFcShape* s, const void* X, const void* W, const void* bias, const void* residual, void* Z, void* Y, bool glu, cudaStream_t stream)
{
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

namespace alpha {

typedef int (*LogitsReady)(void* what, const float* part, int parts);
int fc_logits_f32(const AlphaFcShape* s, const float* X, const float* W, const float* bias, float* Y, cudaStream_t stream)
{
    return forward(s, X, W, bias, nullptr, nullptr, Y, false, stream);
}
int fc_logits_and_gradients_f32(const AlphaFcShape* s, const float* X, const float* W, const float* bias, float* Z, float* dX, float* dW, LogitsReady between, void* what, cudaStream_t stream)
{
    const int rows = s->rows, IC = s->IC, OC = s->OC, pitch = fc_pitch(OC);
    const FcEpilogue of_z{bias, nullptr, nullptr, Z, pitch, ALPHA_ACT_NONE, 0.f}, of_x{nullptr, nullptr, nullptr, dX, IC, ALPHA_ACT_NONE, 0.f}, of_w{nullptr, nullptr, nullptr, dW, IC, ALPHA_ACT_NONE, 0.f};
    const ProductF32 z{X, W, rows, pitch, IC, OC, pitch, 1, IC, IC, of_z}, x{Z, W, rows, IC, pitch, OC, pitch, 1, pitch, IC, of_x}, w{Z, X, pitch, IC, rows, OC, pitch, 1, pitch, IC, of_w};
    PairWork v;
    int rc = device_sms(&v.sms);
    if (!rc) rc = device_status_word(&v.status);
    if (rc) return rc;
    const PairPlan pz = pick_pair(rows, 1, OC, false, IC, 1, v.sms), px = pick_pair(rows, 1, IC, false, OC, 1, v.sms), pw = pick_pair(OC, 1, IC, false, rows, 1, v.sms);
    if (!dX || !dW || v.sms < 2 || rows <= kSmallRows) return 1;
    const int a = v.add(X, rows, IC), b = v.add(W, OC, IC), c = v.add(Z, rows, pitch);
    const TwoPairs both = pick_two_pairs(rows, IC, OC, v.sms);
    const bool two = both.bn && both.time < 0.95 * (px.time + pw.time);      // (within 5 %, which the estimates do not tell apart: two launches)
    v.want(z, pz.parts);
    if (two) v.parts = std::max(v.parts, both.part_bytes);
    else { v.want(x, px.parts); v.want(w, pw.parts); }
    const double pairs = pz.time + (two ? both.time : px.time + pw.time) + split_time(v.elements()) + 2.0;
    const double apart = pick_gathered<kFcForward>(z, v.sms).time + pick_gathered<kFcDeltaX>(x, v.sms).time + pick_gathered<kFcDeltaW>(w, v.sms).time;
    if (!v.fits() || !pairs_pay(pairs, apart)) return 1;
    rc = v.split(stream, 2);                       // X and W
    if (rc) return rc;
    if (dry_run()) return ALPHA_OK;
    rc = launch_pair<kFcForward>(z, v.p[a], v.p[b], pz, v.part, v.seen, v.seen_n, v.sms, v.status, stream, false);
    if (!rc) rc = between(what, pz.parts > 1 ? static_cast<const float*>(v.part) : nullptr, pz.parts);
    const int seen = v.seen_n;
    if (!rc) {
        const Planes* one[1] = {&v.p[c]};
        rc = launch_split(one, 1, v.seen + seen, &v.seen_n, v.sms, stream);
    }
    if (!rc && two) return launch_two_pairs(x, w, v.p[a], v.p[b], v.p[c], both, v.part, v.seen, seen + v.seen_n, v.sms, v.status, stream);
    if (!rc) rc = launch_pair<kFcDeltaX>(x, v.p[c], v.p[b], px, v.part, v.seen, seen + v.seen_n, v.sms, v.status, stream);
    if (!rc) rc = launch_pair<kFcDeltaW>(w, v.p[c], v.p[a], pw, v.part, v.seen, seen + v.seen_n, v.sms, v.status, stream);
    return rc;
}
int fc_gradients_f32(const AlphaFcShape* s, const float* dZ, const float* X, const float* W, float* dX, float* dW, cudaStream_t stream)
{
    return delta_f32(dZ, X, W, dX, dW, s->rows, s->OC, 1, s->IC, stream);
}

}  // namespace alpha

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
    if (!rc) rc = call_begin(static_cast<cudaStream_t>(stream));
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
    if (!rc) rc = call_begin(static_cast<cudaStream_t>(stream));
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
