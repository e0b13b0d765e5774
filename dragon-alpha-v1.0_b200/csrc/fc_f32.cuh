// The fp32 products of a FullConnect layer: policies of the kernel that forms them as three bf16 planes at fp32 accuracy.
#pragma once
#include "fc_act.cuh"
#include "gemm_planes.cuh"

namespace alpha {

// What becomes of the sums of a layer: four consecutive columns of a row, glu (gate, up, gate, up) of two units.  Rows are given by
// their place in Y, from which Z and R follow (the same pitch; glu: Z twice).  Parts of sums lie [part][row][column], glu [part][row][gates, ups].
struct FcEpilogue {
    const float *bias, *residual;
    float *Z, *Y;
    int cols, act; float k;         // cols: pitch of Y, and of either half of Z and the bias
};
template <bool GLU> __device__ __noinline__ void fc_finish(const FcEpilogue& e, float* row, int col, float4 o)
{
    const size_t at = row - e.Y;
    if (GLU) {
        const int j = col >> 1;
        float2 g = make_float2(o.x, o.z), u = make_float2(o.y, o.w);
        if (e.bias) {
            g.x += e.bias[j]; g.y += e.bias[j + 1];
            u.x += e.bias[e.cols + j]; u.y += e.bias[e.cols + j + 1];
        }
        if (e.Z) {
            *reinterpret_cast<float2*>(e.Z + 2 * at + j) = g;
            *reinterpret_cast<float2*>(e.Z + 2 * at + e.cols + j) = u;
        }
        with_act(e.act, [&](auto a) {
            g.x = act_value<decltype(a)::value, false>(g.x, e.k) * u.x;
            g.y = act_value<decltype(a)::value, false>(g.y, e.k) * u.y;
        });
        *reinterpret_cast<float2*>(row + j) = g;
        return;
    }
    if (e.bias) {
        const float4 b = *reinterpret_cast<const float4*>(e.bias + col);
        o.x += b.x; o.y += b.y; o.z += b.z; o.w += b.w;
    }
    if (e.Z) *reinterpret_cast<float4*>(e.Z + at + col) = o;
    with_act(e.act, [&](auto a) {
        constexpr int ACT = decltype(a)::value;
        o.x = act_value<ACT, false>(o.x, e.k); o.y = act_value<ACT, false>(o.y, e.k);
        o.z = act_value<ACT, false>(o.z, e.k); o.w = act_value<ACT, false>(o.w, e.k);
    });
    if (e.residual) {
        const float4 r = *reinterpret_cast<const float4*>(e.residual + at + col);
        o.x += r.x; o.y += r.y; o.z += r.z; o.w += r.w;
    }
    *reinterpret_cast<float4*>(row + col) = o;
}

enum FcForm : int { kFcForward, kFcGlu, kFcDeltaX, kFcDeltaW };

// Rows x columns outputs over K steps in `ksplit` parts (bz), each into its own copy of the sums, or finished at once.  Tensors that are OC wide
// have a pitch of `pitch` columns (a half), W and deltaW do not: the padding among rows, columns and steps has no words of W and no outputs.
template <int FORM>
struct PlaneFc {
    static constexpr bool kAk = FORM != kFcDeltaW, kBk = FORM == kFcForward || FORM == kFcGlu, kTail = false, kCopyB = false;
    const float *A, *B;
    int rows, cols, K, OC, pitch, lda, ldb, ksplit;
    float* part; size_t size;       // ksplit > 1
    FcEpilogue e;
    struct Cta { int m0, n0, s0, s1, K; float* out; };

    // Place of a column of Z among the rows of W, -1: padding.
    __device__ int unit_of(int c) const { const int up = c >= pitch ? 1 : 0, j = c - up * pitch; return j < OC ? j + up * OC : -1; }
    __device__ bool cta(Cta& c, int BM, int BN, int bx, int by, int sp) const
    {
        c.m0 = bx * BM; c.n0 = by * BN;
        const int stages = (K + 31) / 32, per = (stages + ksplit - 1) / ksplit;
        c.s0 = sp * per < stages ? sp * per : stages;
        c.s1 = c.s0 + per < stages ? c.s0 + per : stages;
        c.K = K;
        c.out = ksplit > 1 ? part + static_cast<size_t>(sp) * size : e.Y;
        return true;
    }
    __device__ int columns(const Cta& c) const { return cols - c.n0; }
    __device__ const float* a_tensor(const Cta&) const { return A; }
    __device__ const float* b_tensor(const Cta&) const { return B; }
    __device__ PlaneAt a_row(const Cta& c, int m) const { return PlaneAt{static_cast<uint32_t>(kAk ? (c.m0 + m) * lda : c.m0 + m), c.m0 + m < rows ? 1u : 0u}; }
    __device__ PlaneAt b_row(const Cta& c, int col) const
    {
        const int j = c.n0 + col;
        if (!kBk) return PlaneAt{static_cast<uint32_t>(j), j < cols ? 1u : 0u};
        const int unit = FORM == kFcGlu ? j >> 1 : j;                                           // glu: gate and up rows in turn
        return PlaneAt{static_cast<uint32_t>((FORM == kFcGlu ? unit + (j & 1) * OC : unit) * ldb), unit < OC ? 1u : 0u};
    }
    __device__ PlaneAt a_step(const Cta&, int k) const { return PlaneAt{static_cast<uint32_t>(k * (kAk ? 1 : lda)), k < K ? 1u : kNoStep}; }
    __device__ PlaneAt b_step(const Cta&, int k) const
    {
        if (FORM != kFcDeltaX) return PlaneAt{static_cast<uint32_t>(k * (kBk ? 1 : ldb)), k < K ? 1u : kNoStep};
        const int unit = k < K ? unit_of(k) : -1;
        return unit >= 0 ? PlaneAt{static_cast<uint32_t>(unit * ldb), 1u} : PlaneAt{0u, kNoStep};
    }
    __device__ static bool use_a(const PlaneAt& row, const PlaneAt& step) { return plane_meets(row, step); }
    __device__ static bool use_b(const PlaneAt& row, const PlaneAt& step) { return plane_meets(row, step); }
    __device__ float* row_out(const Cta& c, int m) const
    {
        if (c.m0 + m >= rows) return nullptr;
        const int row = FORM == kFcDeltaW ? unit_of(c.m0 + m) : c.m0 + m;
        return row >= 0 ? c.out + static_cast<size_t>(row) * (ksplit > 1 ? cols : e.cols) : nullptr;
    }
    __device__ void store(const Cta& c, float* row, int col, const float4& o) const
    {
        const int j = c.n0 + col;
        if (!row || j >= cols) return;
        if (ksplit > 1 && FORM == kFcGlu) {
            *reinterpret_cast<float2*>(row + (j >> 1)) = make_float2(o.x, o.z);
            *reinterpret_cast<float2*>(row + e.cols + (j >> 1)) = make_float2(o.y, o.w);
        } else if (ksplit > 1 || FORM == kFcDeltaX || FORM == kFcDeltaW) *reinterpret_cast<float4*>(row + j) = o;
        else fc_finish<FORM == kFcGlu>(e, row, j, o);
    }
};

// The parts of a product added in order, then finished: four outputs a thread, glu two.
template <bool GLU>
__global__ void __launch_bounds__(256) fc_parts_kernel(const float* __restrict__ part, size_t size, int parts, FastDiv by_words, size_t words, const __grid_constant__ FcEpilogue e)
{
    grid_dependency_wait();
    grid_dependency_trigger();
    for (size_t i = static_cast<size_t>(blockIdx.x) * 256 + threadIdx.x; i < words; i += static_cast<size_t>(gridDim.x) * 256) {
        unsigned row, q;
        by_words.divmod(static_cast<unsigned>(i), row, q);
        float* out = e.Y + static_cast<size_t>(row) * e.cols;
        if constexpr (GLU) {
            const float* at = part + 2 * static_cast<size_t>(row) * e.cols + 2 * q;
            float2 g = make_float2(0.f, 0.f), u = g;
            for (int s = 0; s < parts; ++s, at += size) {
                const float2 a = __ldg(reinterpret_cast<const float2*>(at)), b = __ldg(reinterpret_cast<const float2*>(at + e.cols));
                g.x += a.x; g.y += a.y; u.x += b.x; u.y += b.y;
            }
            fc_finish<true>(e, out, 4 * q, make_float4(g.x, u.x, g.y, u.y));
        } else {
            const float* at = part + static_cast<size_t>(row) * e.cols + 4 * q;
            float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int r = 0; r < parts; ++r, at += size) {
                const float4 v = __ldg(reinterpret_cast<const float4*>(at));
                s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
            }
            fc_finish<false>(e, out, 4 * q, s);
        }
    }
}

}  // namespace alpha
