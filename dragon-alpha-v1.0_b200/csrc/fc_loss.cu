// Softmax cross entropy on top of a FullConnect layer whose logits are not kept, and its gradients.
//
//   z = X W^T + bias,  lse = log sum exp z,  loss = lse - z[label]
//   dz = dL (exp(z - lse) - [label]),  deltaX = dz W,  deltaW = dz^T X,  deltaB = column sums of dz
//
// 16-bit tensors.  Forward: one product whose epilogue reduces each tile's row to its largest logit and the sum of exponentials about it (8 bytes for 128 or fewer logits), and a
// pass that joins them.  Gradients, piece by piece of the classes: logits formed once more, their gradients rounded to the tensors' type into scratch as the epilogue
// of that product, and the two products that read them; deltaX is summed in fp32 over the pieces.  dz is rounded once, as deltaZ of a FullConnect layer is; a dL that all rows share
// is left to the outputs.  In fp16 dz is held times a power of two (the largest |dL| at 2^14 or above), as a probability of 1e-5 over 1e4 rows would not be a normal
// number, and the outputs are scaled back in fp32.
// Bound by the tensor cores: 2 (forward) and 6 (gradients) rows x classes x IC operations; for few rows by reading W.  4096 x 4096 x 128000 in bf16: 3.05 and 9.46 ms, 1.41 and 1.36
// PFLOP/s at the power limit, where cuBLAS sustains 1.39; 4 rows of it 173 us, W at 6.6 TB/s.
//
// fp32 tensors: products at fp32 accuracy as those of the layer, logits of a piece in scratch.  Gradients of 512 x 4096 x 1000: 97 us in a graph, of which the three products take 80.
#include "fc_loss.cuh"
#include "fc_product.cuh"

using namespace alpha;

namespace alpha {
// fp32 products of a call that has begun (fc_api.cu).
int fc_logits_f32(const AlphaFcShape* s, const float* X, const float* W, const float* bias, float* Y, cudaStream_t stream);
int fc_gradients_f32(const AlphaFcShape* s, const float* dZ, const float* X, const float* W, float* dX, float* dW, cudaStream_t stream);
// Z = X W^T + bias, then between(), which makes deltaZ of it in place, then both gradients, the planes of X and W split once; 1 where the products are not all
// best formed from planes, or their scratch is refused (nothing has been launched then).  Where Z was formed in parts it holds nothing yet: they lie in `part`, [part][row][pitch of Z], without the bias.
typedef int (*LogitsReady)(void* what, const float* part, int parts);
int fc_logits_and_gradients_f32(const AlphaFcShape* s, const float* X, const float* W, const float* bias, float* Z, float* dX, float* dW, LogitsReady between, void* what, cudaStream_t stream);
}

namespace {

constexpr size_t kPieceBytes = 256u << 20;       // of logits or their gradients in scratch

struct Loss {
    const AlphaFcShape* s;
    const void *X, *W, *bias, *label;
    int label_bytes;
    cudaStream_t stream;
};

const char* at_class(const void* p, size_t first, size_t row_bytes) { return static_cast<const char*>(p) + first * row_bytes; }

int join(const Loss& c, const float2* part, int slots, int row0, int rows, const float* at_label, float* loss, float* lse)
{
    int across = 1;
    while (across < 32 && across < rows) across *= 2;
    const char* label = at_class(c.label, row0, c.label_bytes);
    launch_after(loss_join_kernel, (rows + across - 1) / across, kJoinThreads, 0, c.stream, part, slots, rows, across, label, c.label_bytes, c.s->OC, at_label, loss ? loss + row0 : nullptr,
                 lse ? lse + row0 : nullptr);
    note_launch("fc_loss");
    return launched("loss_join_kernel");
}

int forward_16(const Loss& c, float* loss, float* lse)
{
    const long long IC = c.s->IC, OC = c.s->OC;
    int sms = 0, *status = nullptr;
    int rc = device_sms(&sms);
    if (!rc) rc = device_status_word(&status);
    if (rc) return rc;
    // runs of rows whose parts take about the size of a piece (a slot for 128 classes, where there are many rows)
    long long run = static_cast<long long>(kPieceBytes / 8) / ((OC + 127) / 128);
    run = std::min<long long>(std::max(4096LL, run / 256 * 256), c.s->rows);
    const ScratchMark mark = call_mark(c.stream);
    for (long long row0 = 0; row0 < c.s->rows; row0 += run) {
        call_rewind(c.stream, mark);
        const int rows = static_cast<int>(std::min<long long>(run, c.s->rows - row0));
        Product q{c.s->dtype, rows, c.s->OC, fc_pitch(c.s->OC), c.s->IC, 1, 1, false, Operand{at_class(c.X, row0, IC * 2), false, IC, 1, rows, IC, IC}, Operand{c.W, false, IC, OC, 1, IC, OC * IC}, c.bias, nullptr, nullptr, nullptr,
                  ALPHA_ACT_NONE, 0.f, FcLoss{}};
        float2 dummy;
        q.loss.part = &dummy;                         // (the plan: nothing is written but parts)
        FcPlan plan = pick_plan(q, sms, nullptr, 1);
        if (!plan.pair) plan.bn = std::min(plan.bn, 128);       // (wider ones can be asked for by option FC_TILE)
        const long long slots = 2 * ((OC + plan.bn - 1) / plan.bn);
        void *part = nullptr, *at_label = nullptr;
        rc = call_scratch(c.stream, static_cast<size_t>(slots) * rows * sizeof(float2), &part);
        if (!rc) rc = call_scratch(c.stream, rows * sizeof(float), &at_label);
        if (rc) return rc;
        if (dry_run()) continue;
        q.loss.label = at_class(c.label, row0, c.label_bytes); q.loss.label_bytes = c.label_bytes; q.loss.classes = c.s->OC;
        q.loss.part = static_cast<float2*>(part); q.loss.at_label = static_cast<float*>(at_label);
        rc = launch_planned<kFcStats>(q, nullptr, plan, sms, status, c.stream);
        if (!rc) rc = join(c, q.loss.part, static_cast<int>(slots), static_cast<int>(row0), rows, q.loss.at_label, loss, lse);
        if (rc) return rc;
    }
    return ALPHA_OK;
}

// deltaB of a piece from its dz.
template <class T> int column_sums(const T* dz, int rows, int pitch, const float* by, float factor, T* dB, int sms, cudaStream_t stream)
{
    if (rows <= 1024 && static_cast<long long>(rows) * pitch <= 1 << 20) {
        // (512 x 1000 fp32: 4 us instead of two launches' 8)
        if (dry_run()) return ALPHA_OK;
        launch_after(loss_few_columns_kernel<T>, (pitch + 31) / 32, 1024, 0, stream, dz, rows, pitch, by, factor, dB);
        note_launch("fc_loss");
        return launched("loss_few_columns_kernel");
    }
    const int blocks = (pitch + 32 * Word16<T>::N - 1) / (32 * Word16<T>::N), most = std::max(1, 8 * sms / blocks), parts = std::min((rows + 31) / 32, most);
    void* part = nullptr;
    int rc = call_scratch(stream, static_cast<size_t>(parts) * pitch * sizeof(float), &part);
    if (rc || dry_run()) return rc;
    launch_after(loss_columns_kernel<T>, dim3(blocks, parts), 256, 0, stream, dz, rows, pitch, static_cast<float*>(part));
    note_launch("fc_loss");
    rc = launched("loss_columns_kernel");
    if (rc) return rc;
    launch_after(loss_bias_kernel<T>, (pitch + 255) / 256, 256, 0, stream, static_cast<const float*>(part), parts, pitch, by, factor, dB);
    note_launch("fc_loss");
    return launched("loss_bias_kernel");
}

// Classes of a piece: all, or as many as fit, in even pieces of multiples of `unit`; 8 KB of a row at least, since each piece adds to all of deltaX (4096 of 16 bits: an eighth of
// the time of its products).
long long piece_classes(long long rows, long long classes, size_t size, long long unit)
{
    const long long fit = std::max<long long>(8192 / size, static_cast<long long>(kPieceBytes / size) / rows / unit * unit), pieces = (classes + fit - 1) / fit;
    return std::min(classes, ((classes + pieces - 1) / pieces + unit - 1) / unit * unit);
}

template <class T> int delta_16(const Loss& c, const float* dL, int dL_step, const float* lse, void* dX, void* dW, void* dB)
{
    const long long rows = c.s->rows, IC = c.s->IC, OC = c.s->OC, piece = piece_classes(rows, OC, 2, 256), pieces = (OC + piece - 1) / piece;
    const int dtype = c.s->dtype, most_pitch = fc_pitch(static_cast<int>(piece));
    int sms = 0, *status = nullptr;
    int rc = device_sms(&sms);
    if (!rc) rc = device_status_word(&status);
    void *dz = nullptr, *sums = nullptr, *scale = nullptr;
    const bool f16 = dtype == ALPHA_F16;
    if (!rc) rc = call_scratch(c.stream, static_cast<size_t>(rows) * most_pitch * 2, &dz);
    if (!rc && dX && pieces > 1) rc = call_scratch(c.stream, static_cast<size_t>(rows) * IC * 4, &sums);
    if (!rc && f16 && dL_step) rc = call_scratch(c.stream, 2 * sizeof(float), &scale);
    if (rc) return rc;
    if (scale && !dry_run()) {
        launch_after(loss_scale_kernel, 1, 1024, 0, c.stream, dL, c.s->rows, c.label, c.label_bytes, c.s->OC, static_cast<float*>(scale));
        note_launch("fc_loss");
        rc = launched("loss_scale_kernel");
        if (rc) return rc;
    }
    // One gradient for all rows stays out of dz, which then is p - [label] (most are 1 or near: they would all be rounded alike) and, in fp16, 2^14 times that.
    const float held = f16 && !dL_step ? 0x1p14f : 1.f;
    const float *out_by = dL_step ? (scale ? static_cast<const float*>(scale) + 1 : nullptr) : dL, out_factor = 1.f / held;
    const ScratchMark mark = call_mark(c.stream);
    for (long long first = 0; first < OC; first += piece) {
        call_rewind(c.stream, mark);
        const long long cols = std::min(piece, OC - first), pitch = fc_pitch(static_cast<int>(cols));
        const T* W = static_cast<const T*>(c.W) + first * IC;
        FcLoss l{};
        l.label = c.label; l.label_bytes = c.label_bytes; l.base = static_cast<int>(first); l.classes = c.s->OC;
        l.lse = lse; l.grad = dL_step ? dL : nullptr; l.scale = static_cast<const float*>(scale); l.held = held;
        FcLoss of_x{}, of_w{};
        of_x.out_by = of_w.out_by = out_by; of_x.out_factor = of_w.out_factor = out_factor;
        of_x.sums = static_cast<float*>(sums); of_x.first = first == 0; of_x.last = first + cols == OC;
        Product x{dtype, c.s->rows, c.s->IC, c.s->IC, static_cast<int>(cols), 1, 1, false, Operand{dz, false, cols, 1, rows, pitch, pitch}, Operand{W, true, IC, cols, 1, IC, cols * IC},
                  nullptr, nullptr, nullptr, dX, ALPHA_ACT_NONE, 0.f, of_x};
        const Product w{dtype, static_cast<int>(cols), c.s->IC, c.s->IC, c.s->rows, 1, 1, false, Operand{dz, true, cols, 1, rows, pitch, pitch}, Operand{c.X, true, IC, rows, 1, IC, rows * IC},
                        nullptr, nullptr, nullptr, dW ? static_cast<T*>(dW) + first * IC : nullptr, ALPHA_ACT_NONE, 0.f, of_w};
        // deltaX in parts of the classes where that is the least
        PartsPlan parts{0, 1, 1e300};
        void* part = nullptr;
        if (dX) {
            double other = 0.0, more = 0.0;
            pick_plan(x, sms, &other);
            if (dW) pick_plan(w, sms, &more);
            parts = pick_parts(x, dW ? &w : nullptr, sms);
            if (parts.parts > 1 && parts.time < 0.93 * (other + more)) {
                rc = call_scratch(c.stream, static_cast<size_t>(parts.parts) * rows * IC * 4, &part);
                if (rc && !scratch_refused(rc)) return rc;
                if (rc) part = nullptr;                      // (without it in one)
            }
        }
        if (!dry_run()) {
            const Product z{dtype, c.s->rows, static_cast<int>(cols), static_cast<int>(pitch), c.s->IC, 1, 1, false, Operand{c.X, false, IC, 1, rows, IC, IC}, Operand{W, false, IC, cols, 1, IC, cols * IC},
                            c.bias ? static_cast<const T*>(c.bias) + first : nullptr, nullptr, nullptr, dz, ALPHA_ACT_NONE, 0.f, l};
            rc = launch_product<kFcSoftmaxDelta>(z, c.stream);
            if (rc) return rc;
            if (part) {
                x.loss.sums = static_cast<float*>(part);
                x.loss.parts = parts.parts;
                rc = launch_planned<kFcSum>(x, dW ? &w : nullptr, FcPlan{true, parts.bn, 1}, sms, status, c.stream);
                if (rc) return rc;
                note_plan("fc loss pair 256x%d parts=%d", parts.bn, parts.parts);
                const size_t words = static_cast<size_t>(rows) * IC / 4;
                launch_after(loss_parts_kernel<T>, static_cast<unsigned>(std::min<size_t>((words + 255) / 256, 8u * sms)), 256, 0, c.stream, static_cast<const float4*>(part), parts.parts, words,
                             static_cast<float4*>(sums), of_x.first, of_x.last, out_by, out_factor, static_cast<uint2*>(dX));
                note_launch("fc_loss");
                rc = launched("loss_parts_kernel");
            } else if (dX && dW) {
                rc = launch_products<kFcSum>(x, w, c.stream);
            } else if (dX) {
                rc = launch_product<kFcSum>(x, c.stream);
            } else if (dW) {
                rc = launch_product<kFcSum>(w, c.stream);
            }
            if (rc) return rc;
        }
        if (dB) rc = column_sums(static_cast<const T*>(dz), c.s->rows, static_cast<int>(pitch), out_by, out_factor, static_cast<T*>(dB) + first, sms, c.stream);
        if (rc) return rc;
    }
    return ALPHA_OK;
}

// CTAs to a row in the passes over fp32 logits: some 512 in all, a thousand logits each at least (13 x 122368: gradients of the logits 78 us by one to a row, 10 by 39).
int row_ctas(long long rows, long long cols) { return static_cast<int>(std::max(1LL, std::min(512 / rows, cols / 1024))); }

int forward_f32(const Loss& c, float* loss, float* lse)
{
    const long long rows = c.s->rows, IC = c.s->IC, OC = c.s->OC, piece = piece_classes(rows, OC, 4, 8), pieces = (OC + piece - 1) / piece;
    const int across = row_ctas(rows, piece);
    const long long slots = pieces * across;
    void *z = nullptr, *part = nullptr, *at_label = nullptr;
    int rc = call_scratch(c.stream, static_cast<size_t>(rows) * fc_pitch(static_cast<int>(piece)) * 4, &z);
    if (!rc && slots > 1) rc = call_scratch(c.stream, static_cast<size_t>(slots) * rows * sizeof(float2), &part);
    if (!rc && slots > 1) rc = call_scratch(c.stream, rows * sizeof(float), &at_label);
    const ScratchMark mark = call_mark(c.stream);
    for (long long first = 0; first < OC && !rc; first += piece) {
        call_rewind(c.stream, mark);
        AlphaFcShape s = *c.s;
        s.OC = static_cast<int>(std::min(piece, OC - first));
        rc = fc_logits_f32(&s, static_cast<const float*>(c.X), static_cast<const float*>(c.W) + first * IC, c.bias ? static_cast<const float*>(c.bias) + first : nullptr, static_cast<float*>(z), c.stream);
        if (rc || dry_run()) continue;
        launch_after(loss_rows_kernel, dim3(static_cast<unsigned>(rows), across), kRowThreads, 0, c.stream, static_cast<const float*>(z), fc_pitch(s.OC), s.OC, static_cast<int>(first), c.s->OC, c.s->rows, c.label,
                     c.label_bytes, part ? static_cast<float2*>(part) + first / piece * across * rows : nullptr, static_cast<float*>(at_label), loss, lse);
        note_launch("fc_loss");
        rc = launched("loss_rows_kernel");
    }
    if (rc || dry_run() || slots == 1) return rc;
    return join(c, static_cast<const float2*>(part), static_cast<int>(slots), 0, c.s->rows, static_cast<const float*>(at_label), loss, lse);
}

int delta_f32(const Loss& c, const float* dL, int dL_step, const float* lse, float* dX, float* dW, float* dB)
{
    const long long rows = c.s->rows, IC = c.s->IC, OC = c.s->OC, piece = piece_classes(rows, OC, 4, 8), pieces = (OC + piece - 1) / piece;
    int sms = 0;
    int rc = device_sms(&sms);
    void *dz = nullptr, *more = nullptr;
    if (!rc) rc = call_scratch(c.stream, static_cast<size_t>(rows) * fc_pitch(static_cast<int>(piece)) * 4, &dz);
    if (!rc && dX && pieces > 1) rc = call_scratch(c.stream, static_cast<size_t>(rows) * IC * 4, &more);
    const ScratchMark mark = call_mark(c.stream);
    for (long long first = 0; first < OC && !rc; first += piece) {
        call_rewind(c.stream, mark);
        AlphaFcShape s = *c.s;
        s.OC = static_cast<int>(std::min(piece, OC - first));
        const float *X = static_cast<const float*>(c.X), *W = static_cast<const float*>(c.W) + first * IC;
        float* z = static_cast<float*>(dz);
        const float* bias = c.bias ? static_cast<const float*>(c.bias) + first : nullptr;
        float* x = dX && first ? static_cast<float*>(more) : dX;
        float* w = dW ? dW + first * IC : nullptr;
        auto softmax = [&](const float* part, int parts) {
            if (dry_run()) return static_cast<int>(ALPHA_OK);
            launch_after(loss_delta_kernel, dim3(static_cast<unsigned>(rows), row_ctas(rows, s.OC)), kRowThreads, 0, c.stream, z, part, parts, part ? bias : nullptr, static_cast<int>(rows), fc_pitch(s.OC), s.OC, static_cast<int>(first),
                         c.s->OC, c.label, c.label_bytes, lse, dL, dL_step);
            note_launch("fc_loss");
            return launched("loss_delta_kernel");
        };
        rc = fc_logits_and_gradients_f32(&s, X, W, bias, z, x, w, [](void* f, const float* part, int parts) { return (*static_cast<decltype(softmax)*>(f))(part, parts); }, &softmax, c.stream);
        if (rc < 0) return rc;
        if (rc == 1) {
            call_rewind(c.stream, mark);
            rc = fc_logits_f32(&s, X, W, bias, z, c.stream);
            if (!rc) rc = softmax(nullptr, 1);
            if (rc) return rc;
            call_rewind(c.stream, mark);                 // (what the logits' product was given)
            if (dX || dW) rc = fc_gradients_f32(&s, z, X, W, x, w, c.stream);
        }
        if (!rc && dX && first && !dry_run()) {
            const size_t words = static_cast<size_t>(rows) * IC / 4;
            launch_after(loss_add_kernel, static_cast<unsigned>(std::min<size_t>((words + 255) / 256, 8u * sms)), 256, 0, c.stream, reinterpret_cast<float4*>(dX), reinterpret_cast<const float4*>(x), words);
            note_launch("fc_loss");
            rc = launched("loss_add_kernel");
        }
        if (!rc && dB) rc = column_sums(z, c.s->rows, fc_pitch(s.OC), nullptr, 1.f, dB + first, sms, c.stream);
    }
    return rc;
}

int check_loss(const char* what, const AlphaFcShape* s, const void* label, int label_bytes)
{
    const int rc = check_fc(what, s, false);
    if (rc) return rc;
    if (s->act != ALPHA_ACT_NONE) return fail(ALPHA_E_ARG, "%s: logits have no activation", what);
    if (!label || (label_bytes != 4 && label_bytes != 8) || reinterpret_cast<uintptr_t>(label) % label_bytes) return fail(ALPHA_E_ARG, "%s: labels are integers of 4 or 8 bytes", what);
    return ALPHA_OK;
}

}  // namespace

extern "C" {

int alpha_fullConnect_softmax_crossEntropy(const AlphaFcShape* s, const void* X, const void* W, const void* bias, const void* label, int label_bytes, float* loss, float* lse,
                                           alpha_stream_t stream)
{
    OpRange range("alpha_fullConnect_softmax_crossEntropy");
    const char* what = "fullConnect_softmax_crossEntropy";
    int rc = check_loss(what, s, label, label_bytes);
    if (rc) return rc;
    if (!X || !W || (!loss && !lse)) return fail(ALPHA_E_ARG, "%s: null tensor pointer", what);
    if ((reinterpret_cast<uintptr_t>(loss) | reinterpret_cast<uintptr_t>(lse)) & 3) return fail(ALPHA_E_ARG, "%s: loss and lse are floats", what);
    const size_t b = type_bytes(s->dtype), rows = s->rows;
    const Span x{X, rows * s->IC * b}, w{W, static_cast<size_t>(s->OC) * s->IC * b}, v{bias, fc_pitch(s->OC) * b};
    rc = check_spans(what, {x, w, v}, {});
    if (!rc) rc = check_overlaps(what, {x, w, v, {label, rows * label_bytes}}, {{loss, rows * 4}, {lse, rows * 4}});
    if (!rc) rc = call_begin(static_cast<cudaStream_t>(stream));
    if (rc) return rc;
    const Loss c{s, X, W, bias, label, label_bytes, static_cast<cudaStream_t>(stream)};
    return s->dtype == ALPHA_F32 ? forward_f32(c, loss, lse) : forward_16(c, loss, lse);
}

int alpha_fullConnect_softmax_crossEntropy_delta(const AlphaFcShape* s, const float* deltaL, int deltaL_step, const void* X, const void* W, const void* bias, const void* label,
                                                 int label_bytes, const float* lse, void* deltaX, void* deltaW, void* deltaB, alpha_stream_t stream)
{
    OpRange range("alpha_fullConnect_softmax_crossEntropy_delta");
    const char* what = "fullConnect_softmax_crossEntropy_delta";
    int rc = check_loss(what, s, label, label_bytes);
    if (rc) return rc;
    if (!deltaL || !X || !W || !lse) return fail(ALPHA_E_ARG, "%s: null tensor pointer", what);
    if (!deltaX && !deltaW && !deltaB) return fail(ALPHA_E_ARG, "%s: no gradient asked for", what);
    if (deltaL_step != 0 && deltaL_step != 1) return fail(ALPHA_E_ARG, "%s: deltaL is one value (step 0) or one for each row (step 1)", what);
    if ((reinterpret_cast<uintptr_t>(deltaL) | reinterpret_cast<uintptr_t>(lse)) & 3) return fail(ALPHA_E_ARG, "%s: deltaL and lse are floats", what);
    const size_t b = type_bytes(s->dtype), rows = s->rows, pitch = fc_pitch(s->OC);
    const Span x{X, rows * s->IC * b}, w{W, static_cast<size_t>(s->OC) * s->IC * b}, v{bias, pitch * b}, dx{deltaX, x.bytes}, dw{deltaW, w.bytes}, db{deltaB, v.bytes};
    rc = check_spans(what, {x, w, v}, {dx, dw, db});
    if (!rc) rc = check_overlaps(what, {{label, rows * label_bytes}, {lse, rows * 4}, {deltaL, deltaL_step ? rows * 4 : 4}}, {dx, dw, db});
    if (!rc) rc = call_begin(static_cast<cudaStream_t>(stream));
    if (rc) return rc;
    const Loss c{s, X, W, bias, label, label_bytes, static_cast<cudaStream_t>(stream)};
    if (s->dtype == ALPHA_F32) return delta_f32(c, deltaL, deltaL_step, lse, static_cast<float*>(deltaX), static_cast<float*>(deltaW), static_cast<float*>(deltaB));
    if (s->dtype == ALPHA_BF16) return delta_16<__nv_bfloat16>(c, deltaL, deltaL_step, lse, deltaX, deltaW, deltaB);
    return delta_16<__half>(c, deltaL, deltaL_step, lse, deltaX, deltaW, deltaB);
}

int alpha_fullConnect_softmax_crossEntropy_workspace_bytes(const AlphaFcShape* s, int op, size_t* bytes)
{
    if (!s || !bytes) return fail(ALPHA_E_ARG, "fullConnect_softmax_crossEntropy_workspace_bytes: null argument");
    if (op != ALPHA_OP_FORWARD && op != ALPHA_OP_DELTAX) return fail(ALPHA_E_ARG, "fullConnect_softmax_crossEntropy_workspace_bytes: unknown op %d", op);
    // the call itself with launches switched off (tensors at placeholder addresses far apart)
    auto at = [](int i) { return reinterpret_cast<void*>(static_cast<uintptr_t>(i + 1) << 44); };
    auto f = [&](int i) { return static_cast<float*>(at(i)); };
    dry_begin();
    const int rc = op == ALPHA_OP_FORWARD ? alpha_fullConnect_softmax_crossEntropy(s, at(0), at(1), at(2), at(3), 8, f(4), f(5), nullptr)
                                          : alpha_fullConnect_softmax_crossEntropy_delta(s, f(0), 1, at(1), at(2), at(3), at(4), 8, f(5), at(6), at(7), at(8), nullptr);
    *bytes = dry_end();
    return rc;
}

}  // extern "C"
