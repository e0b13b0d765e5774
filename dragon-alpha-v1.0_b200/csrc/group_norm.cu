// Group normalisation with an activation, and its gradients: which kernels a call runs on.
#include "group_norm.cuh"
#include "host_checks.h"

#include <algorithm>
#include <cmath>
#include <numeric>

using namespace alpha;

namespace {

int check_norm(const char* what, const AlphaNormShape* s)
{
    if (!s) return fail(ALPHA_E_ARG, "%s: null shape", what);
    if (s->N <= 0 || s->positions <= 0 || s->C <= 0 || s->groups <= 0) return fail(ALPHA_E_ARG, "%s: non-positive dimension (N=%d positions=%d C=%d groups=%d)", what, s->N, s->positions, s->C, s->groups);
    if (s->C % s->groups) return fail(ALPHA_E_ARG, "%s: %d channels are not %d groups of one size", what, s->C, s->groups);
    // (what a thread or a CTA comes to past a tensor's end is an int too)
    const int most = 2147483647 - (1 << 20);
    if (s->positions > most || s->C > most || static_cast<long long>(s->N) * s->C > most) return fail(ALPHA_E_ARG, "%s: more than %d positions or channels of all samples", what, most);
    if (!known_type(s->dtype)) return fail(ALPHA_E_ARG, "%s: unknown element type %d", what, s->dtype);
    if (s->affine_dtype != s->dtype && s->affine_dtype != ALPHA_F32) return fail(ALPHA_E_ARG, "%s: gamma and beta are of the tensors' type or fp32, not type %d", what, s->affine_dtype);
    if (s->act < ALPHA_ACT_NONE || s->act > ALPHA_ACT_GELU_TANH) return fail(ALPHA_E_ARG, "%s: unknown activation %d", what, s->act);
    if (s->act == ALPHA_ACT_LEAKY_RELU && !(s->k == s->k)) return fail(ALPHA_E_ARG, "%s: slope is NaN", what);
    if (!(s->eps >= 0.f && s->eps <= 3e38f)) return fail(ALPHA_E_ARG, "%s: eps=%g must be finite and not negative", what, s->eps);
    return ALPHA_OK;
}
bool aligned(const void* p, size_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }

Norm norm_of(const AlphaNormShape* s)
{
    Norm p{};
    p.N = s->N; p.R = s->positions; p.C = s->C; p.G = s->groups; p.D = s->C / s->groups;
    p.affine_f32 = s->affine_dtype == ALPHA_F32;
    p.eps = s->eps; p.act = s->act; p.k = s->k;
    return p;
}

// Instructions an element takes: in the passes over shared memory, and in the streamed ones.
double norm_instructions(const Norm& p, int size, bool back, bool streamed)
{
    const bool plain = p.act == ALPHA_ACT_NONE || p.act == ALPHA_ACT_LEAKY_RELU, once = size == 4;         // (once: dz is kept)
    return streamed ? (back ? (plain ? 26.0 : 40.0) : (plain ? 16.0 : 21.0)) : (back ? (once ? (plain ? 14.0 : 22.0) : (plain ? 20.0 : 30.0)) : (plain ? 9.0 : 14.0));
}
// The slab and the cluster of least estimated time (us); false: no slab fits.  A CTA takes of its SM what its bytes take at 43 KB a us (rows of fewer than 64 bytes longer) or its
// instructions at 4100 a us (of a warp), whichever is more, a share of the other and of its loads' latency that is the larger the fewer CTAs an SM holds, and its sums and barriers,
// 0.9 us (backward 1.4), in a cluster 0.2 and 0.1 for each of its CTAs more.  Fitted to all plans of 189 calls; what it takes is 2.4 % above a call's fastest on (geometric)
// average (gradients of 128 x 56 x 56 x 64 fp32: two CTAs of 106 KB to an SM 81 us, one of 204 KB 88).
bool plan_resident(Norm& p, int size, bool back, int sms, size_t* smem, double* least)
{
    const long long unit = static_cast<long long>(p.D) * 4 / std::gcd(p.D, 4);
    *least = 1e300;
    if (unit / 4 > kNormThreads || p.C % 4) return false;
    const int unit_words = static_cast<int>(unit / 4), units = static_cast<int>(p.C / unit);
    for (int each = 1; each <= kNormThreads / unit_words && each <= units; ++each) {
        if (units % each) continue;
        const int words = unit_words * each, slabs = units / each;
        for (int cl = 1; cl <= 8; cl *= 2) {
            const int part = (p.R + cl - 1) / cl;
            const long long ctas = static_cast<long long>(p.N) * slabs * cl;
            if (static_cast<long long>(cl - 1) * part >= p.R || part > (1 << 20) || ctas > 2147483647LL) continue;
            const size_t bytes = norm_smem(back, size, part, words, words * 4 / p.D, cl);
            if (bytes > 224 * 1024) continue;
            const int fit = static_cast<int>(227 * 1024 / (bytes + 1024)), at_once = fit < 4 ? fit : 4;
            const double elements = static_cast<double>(part) * words * 4;
            // (what is there at once runs at once, in whole waves as long as these are few)
            const double waves = static_cast<double>(ctas) / (static_cast<double>(sms) * at_once), rounds = waves <= 1.0 ? 1.0 : waves < 4.0 ? std::ceil(waves) : waves;
            const int on_sm = waves <= 1.0 ? static_cast<int>((ctas + sms - 1) / sms) : at_once;
            const double row = words * 4.0 * size, narrow = row >= 64 ? 1.0 : row >= 32 ? 1.16 : 2.3;
            const double memory = elements * size * (back ? 3 : 2) / 43e3 * narrow, math = elements * norm_instructions(p, size, back, false) / 32 / 4100.0;
            const double alone = on_sm == 1 ? 1.1 : on_sm == 2 ? 0.38 : on_sm == 3 ? 0.09 : 0.0;
            const double each_cta = std::max(memory, math) + alone * (std::min(memory, math) + 1.1) + (back ? 1.4 : 0.9) + 0.1 * cl + (cl > 1 ? 0.2 : 0.0);
            const double time = 2.2 + rounds * on_sm * each_cta;
            if (time < *least) {
                *least = time;
                p.words = words; p.slabs = slabs; p.cluster = cl; p.part = part; p.rows = kNormThreads / words;
                *smem = bytes;
            }
        }
    }
    return *least < 1e300;
}
// Column blocks, of whole groups where one fits, that leave the fewest threads idle (8 x 64 x 64 x 640: blocks of 50 words, the last of 10, 61 us; of 40, 55), and runs of positions
// that fill the SMs once.
void plan_streamed(Norm& p, int V, int size, int sms)
{
    const int words = p.C / V;
    const long long least_words = p.D / std::gcd(p.D, V);            // words of the fewest whole groups
    p.whole = least_words <= 128;
    const int unit = p.whole ? static_cast<int>(least_words) : 1, units = words / unit;
    double best = 0.0;
    for (int each = 1; each <= units && each * unit <= kNormThreads; ++each) {
        const int wide = each * unit, blocks = (units + each - 1) / each, rows = kNormThreads / wide;
        const double used = static_cast<double>(words) / (static_cast<double>(blocks) * wide) * (rows * wide) / kNormThreads, row = static_cast<double>(wide) * V * size;
        // (rows of at least 256 bytes of a tensor at a time, where it has them; four rows of threads for the loads of few positions)
        const double good = used * (row < 256 && blocks > 1 ? 0.7 + row / 853 : 1.0) * (rows < 4 ? 0.97 : 1.0);
        if (good >= best - 1e-9) { best = std::max(best, good); p.words = wide; p.blocks = blocks; p.rows = rows; }
    }
    const long long others = static_cast<long long>(p.N) * p.blocks, least = 8LL * p.rows;        // positions of a run
    long long runs = std::max(1LL, 4LL * sms / others);
    runs = std::min(runs, std::max(1LL, p.R / least));
    p.part = static_cast<int>((p.R + runs - 1) / runs);
    p.runs = (p.R + p.part - 1) / p.part;
}

template <class T, bool BACK> int run_norm(Norm& p, const char* what, void* dgamma, void* dbeta, cudaStream_t stream)
{
    int sms = 0;
    int rc = call_begin(stream);
    if (!rc) rc = device_sms(&sms);
    if (rc) return rc;
    const size_t word = 4 * sizeof(T);
    const bool words = p.C % 4 == 0 && aligned(p.X, word) && aligned(p.out, word) && aligned(p.dY, word);
    // streamed: both passes over the tensors, the second through L2 as far as that holds them, and two more launches
    const double bytes = static_cast<double>(p.N) * p.R * p.C * sizeof(T) * (BACK ? 2 : 1), rate = 43.5e3 * sms;
    const double math = static_cast<double>(p.N) * p.R * p.C * norm_instructions(p, sizeof(T), BACK, true) / 32 / ((BACK ? 3900.0 : 3200.0) * sms);
    const double streamed = (BACK ? 16.0 : 12.0) + std::max(math, bytes / rate + (bytes * (bytes > 80e6 ? 1.0 : 0.5) + bytes / (BACK ? 2 : 1)) / rate);
    size_t smem = 0;
    double least = 0.0;
    const bool resident = words && plan_resident(p, sizeof(T), BACK, sms, &smem, &least) && least < streamed;
    if (!resident) { plan_streamed(p, words ? 4 : 1, sizeof(T), sms); p.cluster = 1; }
    p.by_words = fast_div(p.words); p.by_D = fast_div(p.D);
    if (resident) {
        p.groups = p.words * 4 / p.D;
        p.slots = p.D % 4 == 0 ? 1 : p.D == 2 ? 2 : 4;
        p.span = p.D * p.slots / 4 > 0 ? p.D * p.slots / 4 : 1;
        p.by_slabs = fast_div(p.slabs); p.by_cluster = fast_div(p.cluster); p.by_span = fast_div(p.span);
    }
    void* ws = nullptr;
    auto scratch = [&](size_t bytes) { return rc = rc ? rc : call_scratch(stream, bytes, &ws); };
    if (BACK && !scratch(static_cast<size_t>(p.N) * p.cluster * p.C * sizeof(float2))) p.sums = static_cast<float2*>(ws);
    if (!resident && !scratch(static_cast<size_t>(p.N) * p.G * sizeof(float2))) p.group = static_cast<float2*>(ws);
    if (!resident && !scratch(static_cast<size_t>(p.N) * p.runs * p.C * sizeof(float2))) p.partial = static_cast<float2*>(ws);
    if (rc || dry_run()) return rc;
    if (resident) {
        allow_smem<norm_resident_kernel<T, BACK>>();
        launch_after_clusters(norm_resident_kernel<T, BACK>, dim3(static_cast<unsigned>(p.N) * p.slabs * p.cluster), kNormThreads, p.cluster > 1 ? p.cluster : 0, smem, stream, p);
        note_launch("norm");
        note_plan("norm resident words=%d cluster=%d part=%d", p.words, p.cluster, p.part);
        rc = launched("norm_resident_kernel");
    } else {
        const long long ctas = static_cast<long long>(p.N) * p.runs * p.blocks;
        if (ctas > 2147483647LL) return fail(ALPHA_E_ARG, "%s: more CTAs than a launch takes", what);
        const unsigned grid = static_cast<unsigned>(ctas);
        auto by = [&](auto width) {
            constexpr int V = decltype(width)::value;
            constexpr size_t ring = NormRows<T, V, BACK>::kBytes, sums = 2 * V * kNormThreads * sizeof(float);
            launch_after(norm_sums_kernel<T, V, BACK>, grid, kNormThreads, ring > sums ? ring : sums, stream, p);
        };
        if (words) by(std::integral_constant<int, 4>{});
        else by(std::integral_constant<int, 1>{});
        note_launch("norm");
        rc = launched("norm_sums_kernel");
        if (rc) return rc;
        launch_after(norm_join_kernel<T, BACK>, static_cast<unsigned>(p.N * p.G), kJoinNormThreads, 0, stream, p);
        note_launch("norm");
        rc = launched("norm_join_kernel");
        if (rc) return rc;
        if (words) launch_after(norm_apply_kernel<T, 4, BACK>, grid, kNormThreads, NormRows<T, 4, BACK>::kBytes, stream, p);
        else launch_after(norm_apply_kernel<T, 1, BACK>, grid, kNormThreads, 0, stream, p);
        note_launch("norm");
        note_plan("norm streamed words=%d runs=%d part=%d", p.words, p.runs, p.part);
        rc = launched("norm_apply_kernel");
    }
    if (rc || !dgamma) return rc;
    launch_after(norm_affine_kernel<T>, (p.C + 31) / 32, kAffineThreads, 0, stream, p.sums, p.N * p.cluster, p.C, dgamma, dbeta, p.affine_f32);
    note_launch("norm");
    return launched("norm_affine_kernel");
}

}  // namespace

extern "C" {

int alpha_groupNorm(const AlphaNormShape* s, const void* X, const void* gamma, const void* beta, float* mean, float* rstd, void* Y, alpha_stream_t stream)
{
    OpRange range("alpha_groupNorm");
    int rc = check_norm("groupNorm", s);
    if (rc) return rc;
    if (!X || !Y || !gamma != !beta || !mean != !rstd) return fail(ALPHA_E_ARG, "groupNorm: null tensor pointer");
    const size_t b = type_bytes(s->dtype), a = type_bytes(s->affine_dtype), n = static_cast<size_t>(s->N) * s->positions * s->C * b, g = static_cast<size_t>(s->N) * s->groups * 4;
    if (!aligned(X, b) || !aligned(Y, b) || !aligned(gamma, a) || !aligned(beta, a) || !aligned(mean, 4) || !aligned(rstd, 4)) return fail(ALPHA_E_ARG, "groupNorm: tensors must be aligned to their elements");
    rc = check_overlaps("groupNorm", {{X, n}, {gamma, s->C * a}, {beta, s->C * a}}, {{Y, n}, {mean, g}, {rstd, g}});
    if (rc) return rc;
    Norm p = norm_of(s);
    p.X = X; p.out = Y; p.gamma = gamma; p.beta = beta; p.mean = mean; p.rstd = rstd;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (s->dtype == ALPHA_F32) return run_norm<float, false>(p, "groupNorm", nullptr, nullptr, st);
    if (s->dtype == ALPHA_BF16) return run_norm<__nv_bfloat16, false>(p, "groupNorm", nullptr, nullptr, st);
    return run_norm<__half, false>(p, "groupNorm", nullptr, nullptr, st);
}

int alpha_groupNorm_delta(const AlphaNormShape* s, const void* deltaY, const void* X, const float* mean, const float* rstd, const void* gamma, const void* beta, void* deltaX,
                          void* deltaGamma, void* deltaBeta, alpha_stream_t stream)
{
    OpRange range("alpha_groupNorm_delta");
    int rc = check_norm("groupNorm_delta", s);
    if (rc) return rc;
    if (!deltaY || !X || !mean || !rstd || !deltaX || !gamma != !beta || !deltaGamma != !deltaBeta) return fail(ALPHA_E_ARG, "groupNorm_delta: null tensor pointer");
    const size_t b = type_bytes(s->dtype), a = type_bytes(s->affine_dtype), n = static_cast<size_t>(s->N) * s->positions * s->C * b, g = static_cast<size_t>(s->N) * s->groups * 4, c = s->C * a;
    if (!aligned(X, b) || !aligned(deltaY, b) || !aligned(deltaX, b) || !aligned(gamma, a) || !aligned(beta, a) || !aligned(deltaGamma, a) || !aligned(deltaBeta, a) || !aligned(mean, 4) || !aligned(rstd, 4))
        return fail(ALPHA_E_ARG, "groupNorm_delta: tensors must be aligned to their elements");
    rc = check_overlaps("groupNorm_delta", {{deltaY, n}, {X, n}, {mean, g}, {rstd, g}, {gamma, c}, {beta, c}}, {{deltaX, n}, {deltaGamma, c}, {deltaBeta, c}});
    if (rc) return rc;
    Norm p = norm_of(s);
    p.X = X; p.dY = deltaY; p.out = deltaX; p.gamma = gamma; p.beta = beta; p.mean = const_cast<float*>(mean); p.rstd = const_cast<float*>(rstd);
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (s->dtype == ALPHA_F32) return run_norm<float, true>(p, "groupNorm_delta", deltaGamma, deltaBeta, st);
    if (s->dtype == ALPHA_BF16) return run_norm<__nv_bfloat16, true>(p, "groupNorm_delta", deltaGamma, deltaBeta, st);
    return run_norm<__half, true>(p, "groupNorm_delta", deltaGamma, deltaBeta, st);
}

int alpha_groupNorm_workspace_bytes(const AlphaNormShape* s, int op, size_t* bytes)
{
    if (!s || !bytes) return fail(ALPHA_E_ARG, "groupNorm_workspace_bytes: null argument");
    if (op != ALPHA_OP_FORWARD && op != ALPHA_OP_DELTAX) return fail(ALPHA_E_ARG, "groupNorm_workspace_bytes: unknown op %d", op);
    // the call itself with launches switched off (tensors at placeholder addresses far apart); those of elements that start on no 16-byte boundary need the most
    auto at = [&](int i) { return reinterpret_cast<void*>((static_cast<uintptr_t>(i + 1) << 44) + 4); };
    auto f = [&](int i) { return static_cast<float*>(at(i)); };
    auto words = [&](int i) { return reinterpret_cast<void*>(static_cast<uintptr_t>(i + 1) << 44); };
    size_t most = 0;
    int rc = ALPHA_OK;
    for (int form = 0; form < 2 && !rc; ++form) {
        dry_begin();
        auto t = [&](int i) { return form ? words(i) : at(i); };
        rc = op == ALPHA_OP_FORWARD ? alpha_groupNorm(s, t(0), at(1), at(2), f(3), f(4), t(5), nullptr)
                                    : alpha_groupNorm_delta(s, t(0), t(1), f(2), f(3), at(4), at(5), t(6), at(7), at(8), nullptr);
        most = std::max(most, dry_end());
    }
    *bytes = most;
    return rc;
}

}  // extern "C"
