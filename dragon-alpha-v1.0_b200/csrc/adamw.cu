// One AdamW step over many tensors.
//
//   g' = c g,  m = b1 m + (1 - b1) g',  v = b2 v + (1 - b2) g'^2
//   p = p (1 - lr wd) - lr / (1 - b1^t) m / (sqrt(v / (1 - b2^t)) + eps)
//
// One pass over every array, one launch for every 128 tensors: bound by HBM, with moments of 8 bits by the instructions as well.  A CTA takes every gridDim.x-th chunk of 2048
// elements of the launch; a thread has 4 elements of each of two rows of 1024, so that all its loads are in flight together and every load of a warp is consecutive.
// 50 million elements, all fp32: 224 us, 6.2 TB/s.  90 million, fp32 weights with bf16 copies and gradients, 8-bit moments: 275 us, 5.3 TB/s (some 70 instructions an element, of which a third are
// the hash and the roundings of the codes).  Chunks of 4096 on three CTAs an SM took 7 and 8 us longer, of 1024 on six 10 and 35.
//
// Moments of 8 bits: an e4m3 code for each element and a power of two for each block of 32, the smallest with which none is above 448, so that scaling is exact
// in both directions.  A code is rounded up or down at random, with the probability that keeps its mean: v moves by one part in 1 / (1 - b2) a step, codes lie 6 to
// 12 % apart, and one rounded to nearest would never fall again.  The random bits are a hash of seed, step, tensor and element: 16 for either
// moment, nothing is kept, and the same call gives the same bits.  The update itself uses the moments before they are rounded.  A v that is not 0 gets a code that is not 0
// (2^-9 of the scale at least): m / sqrt(0) is what would blow up a step.
//
// Moments are formed by separate fp32 products and sums, m = fl(fl(b1 m) + fl((1 - b1) g')): their codes do not depend on how a compiler fuses them.  Quotient
// and root of the update are good to 2 units of 2^-23 of the update.
#include "../../include/alpha_conv_b200.h"
#include "dependent_launch.cuh"
#include "fc_act.cuh"
#include "host_common.h"
#include "pairs.cuh"

#include <cuda_fp8.h>

#include <algorithm>
#include <exception>
#include <vector>

namespace alpha {
namespace {

constexpr int kAdamTensors = 128, kAdamThreads = 256, kAdamRows = 2, kAdamCtas = 4;       // (CTAs of an SM)
constexpr int kAdamRow = 4 * kAdamThreads, kAdamChunk = kAdamRow * kAdamRows, kAdamBlock = 32;
constexpr uint32_t kAdamSeed = 0x243F6A88u;
enum : unsigned char { kNoType = 255 };

struct AdamTensor {
    void* p;
    const void* g;
    void *m, *v;
    uint8_t *m_scale, *v_scale;          // 8 bits
    void* out;
    long long count;
    double weight_decay;
    uint32_t number;                     // of the tensor in the call
    unsigned char type, grad_type, out_type, words;   // words: every array starts on a 16-byte boundary
};
struct AdamTable {
    AdamTensor t[kAdamTensors];
    unsigned first[kAdamTensors + 1];    // first chunk of each tensor; the last: chunks in all
    int n;
};
struct AdamStep {
    double lr, beta1, beta2, max_norm;
    float b1, b1c, b2, b2c, eps;         // beta and 1 - beta
    float size, root;                    // lr / (1 - b1^t), 1 / sqrt(1 - b2^t), where lr and t are the host's
    uint32_t step, seed;                 // (the low 32 bits of the step)
    const float *lr_at, *norm;
    const long long* step_at;
};

__host__ __device__ __forceinline__ uint32_t mix32(uint32_t x)
{
    x = (x ^ (x >> 16)) * 0x9E3779B9u;   // the golden ratio's and e's binary digits
    x = (x ^ (x >> 15)) * 0xB7E15163u;
    return x ^ (x >> 16);
}

// The random bits of an element's codes, 16 each, times 16 (the place where round_e4m3 wants them): the low half of mix32(element ^ key) for m, the high one for v.  Of four neighbours
// (element a multiple of 4) `start` is what mix32 forms first, (element ^ key) ^ (element ^ key) >> 16, which differs in the lowest bits only.
struct Dither { uint32_t m, v; };
__device__ __forceinline__ uint32_t dither_start(uint32_t element, uint32_t key) { const uint32_t x = element ^ key; return x ^ (x >> 16); }
__device__ __forceinline__ Dither dither_of(uint32_t start)
{
    uint32_t x = start * 0x9E3779B9u;
    x = (x ^ (x >> 15)) * 0xB7E15163u;
    const uint32_t high = x >> 12;                 // (x ^ x >> 16 has the high half of x, and the low half xor the high one)
    return Dither{((x << 4) ^ high) & 0xffff0u, high & 0xffff0u};
}

// Four elements at a time, as two pairs of floats.
struct Four { float2 f[2]; };
template <class T> struct FourOf;
template <> struct FourOf<float> {
    using Raw = float4;
    static __device__ Four get(const Raw& r) { return Four{{make_float2(r.x, r.y), make_float2(r.z, r.w)}}; }
    static __device__ Raw put(const Four& v) { return make_float4(v.f[0].x, v.f[0].y, v.f[1].x, v.f[1].y); }
};
template <class T> struct FourOf16 {
    using Raw = uint2;
    static __device__ Four get(const Raw& r)
    {
        Four v;
        unpack16<T>(r.x, v.f[0].x, v.f[0].y);
        unpack16<T>(r.y, v.f[1].x, v.f[1].y);
        return v;
    }
    static __device__ Raw put(const Four& v) { return make_uint2(pack16<T>(v.f[0].x, v.f[0].y), pack16<T>(v.f[1].x, v.f[1].y)); }
};
template <> struct FourOf<__nv_bfloat16> : FourOf16<__nv_bfloat16> {};
template <> struct FourOf<__half> : FourOf16<__half> {};

__device__ __forceinline__ float2 e4m3_pair(uint32_t codes)
{
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(codes), __NV_E4M3);
    return __half22float2(*reinterpret_cast<const __half2*>(&h));
}
__device__ __forceinline__ Four e4m3_get(uint32_t codes) { return Four{{e4m3_pair(codes & 0xffffu), e4m3_pair(codes >> 16)}}; }
__device__ __forceinline__ uint32_t e4m3_put(const Four& v)
{
    return __nv_cvt_float2_to_fp8x2(v.f[0], __NV_SATFINITE, __NV_E4M3) | static_cast<uint32_t>(__nv_cvt_float2_to_fp8x2(v.f[1], __NV_SATFINITE, __NV_E4M3)) << 16;
}
// The value of an exponent byte (0: 2^-127, 255: NaN), and the byte of a block whose largest magnitude is `most`.
__device__ __forceinline__ float scale_of(uint32_t byte) { return __uint_as_float(byte == 0 ? 0x400000u : byte == 255 ? 0x7fc00000u : byte << 23); }
__device__ __forceinline__ uint32_t scale_for(float most)
{
    // the exponent of most / 448, up where its mantissa is above 1.75 (448 = 1.75 * 2^8): adding 2^21 - 1 to the bits carries into it then
    const int e = static_cast<int>((__float_as_uint(most) + 0x1fffffu) >> 23) - 8;
    return static_cast<uint32_t>(e < 1 ? 1 : e);
}
// y, at most 448, to one of the codes beside it; `random` of 16 bits, times 16.  Codes are 2^-9 apart below 2^-6, as they are from there to 2^-5: such a y is moved there
// first.  (The sign is the top bit, which no carry reaches.)  FLOOR: of a y that is not negative, and if it is not 0 nor is its code.
template <bool FLOOR> __device__ __forceinline__ float round_e4m3(float y, uint32_t random)
{
    const float shift = fabsf(y) < 0x1p-6f ? (FLOOR ? 0x1p-6f : copysignf(0x1p-6f, y)) : 0.f;
    const float a = __uint_as_float((__float_as_uint(__fadd_rn(y, shift)) + random) & ~0xfffffu) - shift;
    if (!FLOOR) return a;
    return y > 0.f ? fmaxf(a, 0x1p-9f) : a;
}

// What a launch's elements have in common.
struct AdamUse { float b1, b1c, b2, b2c, eps, size, root, c; };

__device__ __forceinline__ float sqrt_approx(float x) { float y; asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ float rcp_approx(float x) { float y; asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
// Two elements: p is replaced, and m and v, which come times b1 and b2.
__device__ __forceinline__ void adam_pair(const AdamUse& u, float keep, float2& p, float2 g, float2& m, float2& v)
{
    g = mul2(g, twice(u.c));
    // (sums one by one: the assembler fuses a packed product with a packed sum, whatever their rounding)
    const float2 m1 = mul2(g, twice(u.b1c)), v1 = mul2(mul2(g, g), twice(u.b2c));
    m = make_float2(__fadd_rn(m.x, m1.x), __fadd_rn(m.y, m1.y));
    v = make_float2(__fadd_rn(v.x, v1.x), __fadd_rn(v.y, v1.y));
    const float2 by = fma2(make_float2(sqrt_approx(v.x), sqrt_approx(v.y)), twice(u.root), twice(u.eps));
    p = fma2(mul2(m, make_float2(rcp_approx(by.x), rcp_approx(by.y))), twice(-u.size), mul2(p, twice(keep)));
}

template <class F> __device__ __forceinline__ void with_type(int type, F&& f)
{
    if (type == ALPHA_F32) f(float{});
    else if (type == ALPHA_BF16) f(__nv_bfloat16{});
    else f(__half{});
}
__device__ __forceinline__ float get_one(const void* p, long long i, int type)
{
    return type == ALPHA_F32 ? static_cast<const float*>(p)[i] : type == ALPHA_BF16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]) : __half2float(static_cast<const __half*>(p)[i]);
}
__device__ __forceinline__ void put_one(void* p, long long i, int type, float x)
{
    if (type == ALPHA_F32) static_cast<float*>(p)[i] = x;
    else if (type == ALPHA_BF16) static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(x);
    else static_cast<__half*>(p)[i] = __float2half_rn(x);
}

// The rows of an array that a thread has of a chunk; TAIL: of the last one of a tensor, whose words past `count` elements are zeros and whose last word may be a part of one.
template <class T> __device__ __forceinline__ T zero_word() { T z; memset(&z, 0, sizeof z); return z; }
template <class Raw, class T, bool TAIL> __device__ __forceinline__ void get_rows(Raw (&r)[kAdamRows], const void* p, long long first, long long count)
{
    const Raw* at = reinterpret_cast<const Raw*>(p) + first / 4;
#pragma unroll
    for (int i = 0; i < kAdamRows; ++i) {
        if constexpr (TAIL) {
            const long long left = count - first - i * kAdamRow;
            if (left < 4) {
                r[i] = zero_word<Raw>();
                for (int j = 0; j < left; ++j) reinterpret_cast<T*>(&r[i])[j] = static_cast<const T*>(p)[first + i * kAdamRow + j];
                continue;
            }
        }
        r[i] = __ldcs(at + i * kAdamThreads);
    }
}
template <class T, bool TAIL> __device__ __forceinline__ void get_typed(Four (&f)[kAdamRows], const void* p, long long first, long long count)
{
    typename FourOf<T>::Raw r[kAdamRows];
    get_rows<typename FourOf<T>::Raw, T, TAIL>(r, p, first, count);
#pragma unroll
    for (int i = 0; i < kAdamRows; ++i) f[i] = FourOf<T>::get(r[i]);
}
template <class Raw, class T, bool TAIL> __device__ __forceinline__ void put_row(void* p, long long at, long long count, const Raw& r)
{
    if (TAIL && count - at < 4) {
        for (int j = 0; j < count - at; ++j) static_cast<T*>(p)[at + j] = reinterpret_cast<const T*>(&r)[j];
        return;
    }
    __stcs(reinterpret_cast<Raw*>(p) + at / 4, r);
}
template <bool TAIL> __device__ __forceinline__ void put_rows(void* p, long long first, long long count, int type, const Four (&f)[kAdamRows])
{
    with_type(type, [&](auto t) {
        using T = decltype(t);
#pragma unroll
        for (int i = 0; i < kAdamRows; ++i) put_row<typename FourOf<T>::Raw, T, TAIL>(p, first + i * kAdamRow, count, FourOf<T>::put(f[i]));
    });
}

__device__ __forceinline__ float most_of_warp(float x)
{
#pragma unroll
    for (int d = 16; d; d >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
    return x;
}

template <bool EIGHT, bool TAIL>
__device__ __forceinline__ void word_chunk(const AdamTensor& t, const AdamUse& u, float keep, uint32_t key, long long begin)
{
    const long long first = begin + 4 * threadIdx.x;
    Four p[kAdamRows], g[kAdamRows], m[kAdamRows], v[kAdamRows];
    if constexpr (EIGHT) {
        uint32_t mc[kAdamRows], vc[kAdamRows];
        uint8_t ms[kAdamRows], vs[kAdamRows];
        get_rows<uint32_t, uint8_t, TAIL>(mc, t.m, first, t.count);
        get_rows<uint32_t, uint8_t, TAIL>(vc, t.v, first, t.count);
#pragma unroll
        for (int i = 0; i < kAdamRows; ++i) {
            if (TAIL && first + i * kAdamRow >= t.count) { ms[i] = vs[i] = 127; continue; }
            ms[i] = t.m_scale[(first + i * kAdamRow) / kAdamBlock];
            vs[i] = t.v_scale[(first + i * kAdamRow) / kAdamBlock];
        }
        with_type(t.type, [&](auto x) { get_typed<decltype(x), TAIL>(p, t.p, first, t.count); });
        with_type(t.grad_type, [&](auto x) { get_typed<decltype(x), TAIL>(g, t.g, first, t.count); });
#pragma unroll
        for (int i = 0; i < kAdamRows; ++i) {
            m[i] = e4m3_get(mc[i]);
            v[i] = e4m3_get(vc[i]);
            const float a = scale_of(ms[i]) * u.b1, b = scale_of(vs[i]) * u.b2;       // (a power of two: code * (scale * b1) is rounded as (code * scale) * b1 is)
#pragma unroll
            for (int j = 0; j < 2; ++j) { m[i].f[j] = mul2(m[i].f[j], twice(a)); v[i].f[j] = mul2(v[i].f[j], twice(b)); }
        }
    } else {
        get_typed<float, TAIL>(m, t.m, first, t.count);
        get_typed<float, TAIL>(v, t.v, first, t.count);
        with_type(t.type, [&](auto x) { get_typed<decltype(x), TAIL>(p, t.p, first, t.count); });
        with_type(t.grad_type, [&](auto x) { get_typed<decltype(x), TAIL>(g, t.g, first, t.count); });
    }
#pragma unroll
    for (int i = 0; i < kAdamRows; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            if (!EIGHT) { m[i].f[j] = mul2(m[i].f[j], twice(u.b1)); v[i].f[j] = mul2(v[i].f[j], twice(u.b2)); }
            adam_pair(u, keep, p[i].f[j], g[i].f[j], m[i].f[j], v[i].f[j]);
        }
    put_rows<TAIL>(t.p, first, t.count, t.type, p);
    if (t.out_type != kNoType) put_rows<TAIL>(t.out, first, t.count, t.out_type, p);
    if constexpr (!EIGHT) {
        put_rows<TAIL>(t.m, first, t.count, ALPHA_F32, m);
        put_rows<TAIL>(t.v, first, t.count, ALPHA_F32, v);
        return;
    }
    uint8_t *ms = t.m_scale + first / kAdamBlock, *vs = t.v_scale + first / kAdamBlock;
#pragma unroll
    for (int i = 0; i < kAdamRows; ++i) {
        const float mm = fmaxf(fmaxf(fabsf(m[i].f[0].x), fabsf(m[i].f[0].y)), fmaxf(fabsf(m[i].f[1].x), fabsf(m[i].f[1].y)));
        const float vm = fmaxf(fmaxf(v[i].f[0].x, v[i].f[0].y), fmaxf(v[i].f[1].x, v[i].f[1].y));
        // (the byte of the largest is the largest byte: both moments' go through the eight lanes of a block together)
        uint32_t bytes = scale_for(mm) | scale_for(vm) << 16;
#pragma unroll
        for (int d = 4; d; d >>= 1) bytes = __vmaxu2(bytes, __shfl_xor_sync(0xffffffffu, bytes, d));
        const uint32_t a = bytes & 0xffffu, b = bytes >> 16, start = dither_start(static_cast<uint32_t>(first) + i * kAdamRow, key);
        const float2 ai = twice(__uint_as_float((254u - a) << 23)), bi = twice(__uint_as_float((254u - b) << 23));
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const Dither r0 = dither_of(start ^ (2 * j)), r1 = dither_of(start ^ (2 * j + 1));
            const float2 x = mul2(m[i].f[j], ai), y = mul2(v[i].f[j], bi);
            m[i].f[j] = make_float2(round_e4m3<false>(x.x, r0.m), round_e4m3<false>(x.y, r1.m));
            v[i].f[j] = make_float2(round_e4m3<true>(y.x, r0.v), round_e4m3<true>(y.y, r1.v));
        }
        put_row<uint32_t, uint8_t, TAIL>(t.m, first + i * kAdamRow, t.count, e4m3_put(m[i]));
        put_row<uint32_t, uint8_t, TAIL>(t.v, first + i * kAdamRow, t.count, e4m3_put(v[i]));
        if ((threadIdx.x & 7) == 0 && (!TAIL || first + i * kAdamRow < t.count)) {
            ms[i * (kAdamRow / kAdamBlock)] = static_cast<uint8_t>(a);
            vs[i * (kAdamRow / kAdamBlock)] = static_cast<uint8_t>(b);
        }
    }
}

// Element by element, a block of 32 to a warp: arrays that do not start on 16-byte boundaries.
template <bool EIGHT>
__device__ __noinline__ void ragged_chunk(const AdamTensor& t, const AdamUse& u, float keep, uint32_t key, long long begin)
{
    const long long end = begin + kAdamChunk < t.count ? begin + kAdamChunk : t.count;
    for (long long at = begin + (threadIdx.x & ~31u); at < end; at += kAdamThreads) {
        const long long e = at + (threadIdx.x & 31);
        const bool in = e < end;
        float2 p{0.f, 0.f}, m = p, v = p;                    // (the second of each pair is 0 and goes nowhere)
        if (in) {
            if constexpr (EIGHT) {
                m.x = e4m3_pair(static_cast<const uint8_t*>(t.m)[e]).x * scale_of(t.m_scale[e / kAdamBlock]);
                v.x = e4m3_pair(static_cast<const uint8_t*>(t.v)[e]).x * scale_of(t.v_scale[e / kAdamBlock]);
            } else {
                m.x = static_cast<const float*>(t.m)[e];
                v.x = static_cast<const float*>(t.v)[e];
            }
            m.x *= u.b1;
            v.x *= u.b2;
            p.x = get_one(t.p, e, t.type);
            adam_pair(u, keep, p, make_float2(get_one(t.g, e, t.grad_type), 0.f), m, v);
            put_one(t.p, e, t.type, p.x);
            if (t.out_type != kNoType) put_one(t.out, e, t.out_type, p.x);
        }
        if constexpr (!EIGHT) {
            if (in) {
                static_cast<float*>(t.m)[e] = m.x;
                static_cast<float*>(t.v)[e] = v.x;
            }
            continue;
        }
        const uint32_t a = scale_for(most_of_warp(fabsf(m.x))), b = scale_for(most_of_warp(v.x));     // (and a barrier of the warp: the old scales have been read)
        const Dither random = dither_of(dither_start(static_cast<uint32_t>(e), key));
        m.x = round_e4m3<false>(m.x * __uint_as_float((254u - a) << 23), random.m);
        v.x = round_e4m3<true>(v.x * __uint_as_float((254u - b) << 23), random.v);
        if (in) {
            const uint32_t codes = e4m3_put(Four{{make_float2(m.x, v.x), make_float2(0.f, 0.f)}});
            static_cast<uint8_t*>(t.m)[e] = static_cast<uint8_t>(codes);
            static_cast<uint8_t*>(t.v)[e] = static_cast<uint8_t>(codes >> 8);
            if ((threadIdx.x & 31) == 0) {
                t.m_scale[e / kAdamBlock] = static_cast<uint8_t>(a);
                t.v_scale[e / kAdamBlock] = static_cast<uint8_t>(b);
            }
        }
    }
}

template <bool EIGHT>
__device__ __noinline__ void tail_chunk(const AdamTensor& t, const AdamUse& u, float keep, uint32_t key, long long begin) { word_chunk<EIGHT, true>(t, u, keep, key, begin); }

template <bool EIGHT>
__global__ void __launch_bounds__(kAdamThreads, kAdamCtas) adamw_kernel(const __grid_constant__ AdamTable table, const __grid_constant__ AdamStep s)
{
    __shared__ float shared[2];
    grid_dependency_wait();
    grid_dependency_trigger();
    AdamUse u{s.b1, s.b1c, s.b2, s.b2c, s.eps, s.size, s.root, 1.f};
    if (s.norm) {
        const float norm = *s.norm;
        if (!(norm < __int_as_float(0x7f800000))) return;            // NaN or Inf: the step is left out
        const double ratio = s.max_norm / (static_cast<double>(norm) + 1e-6);
        if (ratio < 1.0) u.c = static_cast<float>(ratio);
    }
    const double lr = s.lr_at ? static_cast<double>(*s.lr_at) : s.lr;
    const long long step = s.step_at ? *s.step_at : static_cast<long long>(s.step);
    if (s.lr_at || s.step_at) {
        if (threadIdx.x == 0) {
            shared[0] = static_cast<float>(lr / (1.0 - pow(s.beta1, static_cast<double>(step))));
            shared[1] = static_cast<float>(1.0 / sqrt(1.0 - pow(s.beta2, static_cast<double>(step))));
        }
        __syncthreads();
        u.size = shared[0];
        u.root = shared[1];
    }
    const uint32_t call_key = EIGHT ? mix32(kAdamSeed ^ mix32(s.seed) ^ static_cast<uint32_t>(step)) : 0u;
    for (unsigned chunk = blockIdx.x; chunk < table.first[table.n]; chunk += gridDim.x) {
        int lo = 0, hi = table.n;                // first[lo] <= chunk < first[hi]
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (table.first[mid] <= chunk) lo = mid;
            else hi = mid;
        }
        const AdamTensor& t = table.t[lo];
        const long long begin = static_cast<long long>(chunk - table.first[lo]) * kAdamChunk;
        const float keep = static_cast<float>(1.0 - lr * t.weight_decay);
        uint32_t key = EIGHT ? mix32(call_key ^ t.number) : 0u;
        if (EIGHT && begin >> 32) key = mix32(key ^ static_cast<uint32_t>(begin >> 32));
        if (t.words && begin + kAdamChunk <= t.count) word_chunk<EIGHT, false>(t, u, keep, key, begin);
        else if (t.words) tail_chunk<EIGHT>(t, u, keep, key, begin);
        else ragged_chunk<EIGHT>(t, u, keep, key, begin);
    }
}

int launched(const char* what)
{
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? ALPHA_OK : fail(ALPHA_E_CUDA, "%s launch failed: %s", what, cudaGetErrorString(e));
}
int type_size(int dtype) { return dtype == ALPHA_F32 ? 4 : 2; }

int check_adamw(int n, const AlphaAdamW* list, const AlphaAdamWStep* s)
{
    if (!s || n < 0 || (n && !list)) return fail(ALPHA_E_ARG, "adamW: null argument");
    if (!(s->beta1 >= 0.0 && s->beta1 < 1.0 && s->beta2 >= 0.0 && s->beta2 < 1.0)) return fail(ALPHA_E_ARG, "adamW: beta1=%g beta2=%g must be in [0, 1)", s->beta1, s->beta2);
    if (!(s->eps >= 0.0) || !(s->eps <= 3e38)) return fail(ALPHA_E_ARG, "adamW: eps=%g must be finite and not negative", s->eps);
    if (!s->step_device && s->step < 1) return fail(ALPHA_E_ARG, "adamW: step %lld, the first is 1", static_cast<long long>(s->step));
    if (!s->lr_device && !(s->lr >= 0.0 && s->lr <= 3e38)) return fail(ALPHA_E_ARG, "adamW: lr=%g must be finite and not negative", s->lr);
    if (s->norm && !(s->max_norm >= 0.0)) return fail(ALPHA_E_ARG, "adamW: max_norm must not be negative or NaN");
    if ((reinterpret_cast<uintptr_t>(s->norm) & 3) || (reinterpret_cast<uintptr_t>(s->lr_device) & 3) || (reinterpret_cast<uintptr_t>(s->step_device) & 7))
        return fail(ALPHA_E_ARG, "adamW: norm, lr and step on the device must be aligned to their types");
    struct Range { uintptr_t from, to; bool write; };
    std::vector<Range> ranges;
    try {
        ranges.reserve(7 * static_cast<size_t>(n) + 3);
    } catch (const std::exception&) {
        return fail(ALPHA_E_NOSCRATCH, "adamW: no host memory to check %d tensors", n);
    }
    auto add = [&](const void* p, size_t bytes, bool write) { if (p) ranges.push_back(Range{reinterpret_cast<uintptr_t>(p), reinterpret_cast<uintptr_t>(p) + bytes, write}); };
    add(s->norm, 4, false);
    add(s->lr_device, 4, false);
    add(s->step_device, 8, false);
    auto known = [](int t) { return t == ALPHA_F32 || t == ALPHA_BF16 || t == ALPHA_F16; };
    for (int i = 0; i < n; ++i) {
        const AlphaAdamW& a = list[i];
        if (!known(a.dtype) || !known(a.grad_dtype) || (a.out && !known(a.out_dtype))) return fail(ALPHA_E_ARG, "adamW: unknown element type of tensor %d", i);
        if (a.moment_bits != list[0].moment_bits || (a.moment_bits != 32 && a.moment_bits != 8)) return fail(ALPHA_E_ARG, "adamW: moments of all tensors have 32 bits, or all 8 (tensor %d: %d)", i, a.moment_bits);
        if (a.count < 0 || a.count >= 1LL << 42) return fail(ALPHA_E_ARG, "adamW: tensor %d has %lld elements", i, static_cast<long long>(a.count));
        if (!(a.weight_decay >= 0.0 && a.weight_decay <= 3e38)) return fail(ALPHA_E_ARG, "adamW: weight decay of tensor %d must be finite and not negative", i);
        if (a.count == 0) continue;
        const bool eight = a.moment_bits == 8;
        if (!a.param || !a.grad || !a.m || !a.v || (eight && (!a.m_scale || !a.v_scale))) return fail(ALPHA_E_ARG, "adamW: null pointer of tensor %d", i);
        const size_t ps = type_size(a.dtype), gs = type_size(a.grad_dtype), os = type_size(a.out_dtype), ms = eight ? 1 : 4, scales = (a.count + kAdamBlock - 1) / kAdamBlock;
        auto off = [](const void* p, size_t size) { return reinterpret_cast<uintptr_t>(p) % size != 0; };
        if (off(a.param, ps) || off(a.grad, gs) || off(a.m, ms) || off(a.v, ms) || (a.out && off(a.out, os))) return fail(ALPHA_E_ARG, "adamW: tensor %d is not aligned to its elements", i);
        add(a.param, a.count * ps, true);
        add(a.grad, a.count * gs, false);
        add(a.m, a.count * ms, true);
        add(a.v, a.count * ms, true);
        if (eight) { add(a.m_scale, scales, true); add(a.v_scale, scales, true); }
        add(a.out, a.count * os, true);
    }
    std::sort(ranges.begin(), ranges.end(), [](const Range& a, const Range& b) { return a.from < b.from; });
    uintptr_t read = 0, written = 0;          // ends of the ranges so far
    for (const Range& r : ranges) {
        if (r.from < written || (r.write && r.from < read)) return fail(ALPHA_E_ARG, "adamW: what a step writes overlaps another tensor");
        (r.write ? written : read) = std::max(r.write ? written : read, r.to);
    }
    return ALPHA_OK;
}

int run_adamw(int n, const AlphaAdamW* list, const AlphaAdamWStep* s, cudaStream_t stream)
{
    int rc = check_adamw(n, list, s);
    if (!rc) rc = call_begin(stream);
    int sms = 0;
    if (!rc) rc = device_sms(&sms);
    if (rc || dry_run()) return rc;
    AdamStep a{};
    a.lr = s->lr; a.beta1 = s->beta1; a.beta2 = s->beta2; a.max_norm = s->max_norm;
    a.b1 = static_cast<float>(s->beta1); a.b1c = static_cast<float>(1.0 - s->beta1);
    a.b2 = static_cast<float>(s->beta2); a.b2c = static_cast<float>(1.0 - s->beta2);
    a.eps = static_cast<float>(s->eps);
    a.size = static_cast<float>(s->lr / (1.0 - pow(s->beta1, static_cast<double>(s->step))));
    a.root = static_cast<float>(1.0 / sqrt(1.0 - pow(s->beta2, static_cast<double>(s->step))));
    a.step = static_cast<uint32_t>(s->step); a.seed = s->seed;
    a.lr_at = s->lr_device; a.norm = s->norm; a.step_at = reinterpret_cast<const long long*>(s->step_device);
    AdamTable t;
    t.n = 0;
    long long chunks = 0;
    const bool eight = n && list[0].moment_bits == 8;
    const long long most = sms * static_cast<long long>(kAdamCtas);
    for (int i = 0; i <= n; ++i) {
        long long more = 0;
        if (i < n) {
            if (list[i].count == 0) continue;
            more = (list[i].count + kAdamChunk - 1) / kAdamChunk;
        }
        if (t.n && (i == n || t.n == kAdamTensors || chunks + more > 2147483647LL)) {
            t.first[t.n] = static_cast<unsigned>(chunks);
            const unsigned grid = static_cast<unsigned>(chunks < most ? chunks : most);
            if (eight) launch_after(adamw_kernel<true>, grid, kAdamThreads, 0, stream, t, a);
            else launch_after(adamw_kernel<false>, grid, kAdamThreads, 0, stream, t, a);
            note_launch("adamw");
            rc = launched("adamw_kernel");
            if (rc) return rc;
            t.n = 0;
            chunks = 0;
        }
        if (i == n) break;
        const AlphaAdamW& l = list[i];
        AdamTensor& d = t.t[t.n];
        d = AdamTensor{l.param, l.grad, l.m, l.v, static_cast<uint8_t*>(l.m_scale), static_cast<uint8_t*>(l.v_scale), l.out, l.count, l.weight_decay, static_cast<uint32_t>(i),
                       static_cast<unsigned char>(l.dtype), static_cast<unsigned char>(l.grad_dtype), static_cast<unsigned char>(l.out ? l.out_dtype : kNoType), 0};
        uintptr_t low = 0;
        for (const void* p : {static_cast<const void*>(l.param), l.grad, static_cast<const void*>(l.m), static_cast<const void*>(l.v), static_cast<const void*>(l.out)}) low |= reinterpret_cast<uintptr_t>(p);
        d.words = low % 16 == 0;
        t.first[t.n++] = static_cast<unsigned>(chunks);
        chunks += more;
    }
    return ALPHA_OK;
}

}  // namespace
}  // namespace alpha

extern "C" int alpha_adamW(int n, const AlphaAdamW* tensors, const AlphaAdamWStep* step, alpha_stream_t stream)
{
    alpha::OpRange range("alpha_adamW");
    return alpha::run_adamw(n, tensors, step, static_cast<cudaStream_t>(stream));
}
