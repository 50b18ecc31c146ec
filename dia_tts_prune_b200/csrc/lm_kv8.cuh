// lm_kv8.cuh - what the kernels of the cache in 8 bits share: codes and their numbers, and what is left of a row's softmax between two kernels.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "lm_kv8.h"

namespace lm {
namespace {

template <int TYPE> struct ElementOf { using type = float; };
template <> struct ElementOf<kTypeBf16> { using type = __nv_bfloat16; };
template <> struct ElementOf<kTypeF16> { using type = __half; };
template <int TYPE> using Element = typename ElementOf<TYPE>::type;

__device__ __forceinline__ float widen(float v) { return v; }
__device__ __forceinline__ float widen(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float widen(__half v) { return __half2float(v); }
template <typename E> __device__ __forceinline__ E narrow(float v);
template <> __device__ __forceinline__ float narrow<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 narrow<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half narrow<__half>(float v) { return __float2half_rn(v); }

// Four codes as two pairs of fp16, which holds both formats' numbers as they are.
template <int FORMAT>
__device__ __forceinline__ void decode4(uint32_t w, uint32_t& lo, uint32_t& hi) {
    if constexpr (FORMAT == kKvE4m3) {
        asm("{\n\t.reg .b16 a, b;\n\t"
            "mov.b32 {a, b}, %2;\n\t"
            "cvt.rn.f16x2.e4m3x2 %0, a;\n\t"
            "cvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
            : "=r"(lo), "=r"(hi) : "r"(w));
    } else {
        const uint32_t u = w ^ 0x80808080u;                    // code + 128; with 0x64 above it, 1152 + code in fp16
        const __half2 bias = __half2half2(__ushort_as_half(0x6480));
        uint32_t x = __byte_perm(u, 0x64646464u, 0x4140), y = __byte_perm(u, 0x64646464u, 0x4342);
        __half2 p = __hsub2(*reinterpret_cast<__half2*>(&x), bias), q = __hsub2(*reinterpret_cast<__half2*>(&y), bias);
        lo = *reinterpret_cast<uint32_t*>(&p);
        hi = *reinterpret_cast<uint32_t*>(&q);
    }
}
template <int FORMAT>
__device__ __forceinline__ float4 values4(uint32_t w, float scale) {
    uint32_t lo, hi;
    decode4<FORMAT>(w, lo, hi);
    const float2 a = __half22float2(*reinterpret_cast<__half2*>(&lo)), b = __half22float2(*reinterpret_cast<__half2*>(&hi));
    return make_float4(a.x * scale, a.y * scale, b.x * scale, b.y * scale);
}

constexpr float kLog2e = 1.4426950408889634f, kWeightBits = 14.f;

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack_half(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// (reference of the weights, reference with value scales, sum) of a row in a part of its tokens, as they are left for whoever joins them
struct RowStats {
    float m, w, l;
};

__device__ __forceinline__ void store_out(const Kv8Attention& a, size_t at, float v) {
    if (a.type == kTypeF32) reinterpret_cast<float*>(a.out)[at] = v;
    else if (a.type == kTypeBf16) reinterpret_cast<__nv_bfloat16*>(a.out)[at] = __float2bfloat16_rn(v);
    else reinterpret_cast<__half*>(a.out)[at] = __float2half_rn(v);
}
__device__ __forceinline__ float load_q(const Kv8Attention& a, long long at) {
    if (a.type == kTypeF32) return reinterpret_cast<const float*>(a.q.x)[at];
    if (a.type == kTypeBf16) return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(a.q.x)[at]);
    return __half2float(reinterpret_cast<const __half*>(a.q.x)[at]);
}
// what the sums of a row are times to be its output
__device__ __forceinline__ float row_factor(const Kv8Attention& a, int head, float m, float w, float l) {
    float sink = a.sinks ? a.sinks[head] : -INFINITY;
    sink = sink < INFINITY ? fminf(sink * kLog2e, 0x1.fffffep+127f) : sink * kLog2e;     // (a finite one stays finite: infinity less itself is no number)
    if (sink != -INFINITY) {
        const float top = fmaxf(m, a.type == kTypeF32 ? floorf(sink) : sink);       // (whole, as the references of fp32 rows are)
        l = (m == -INFINITY ? l : l * exp2_fast(m - top)) + exp2_fast(sink - top);
        m = top;
    }
    if (l == 0.f || w == -INFINITY) return l != l ? l : 0.f;    // nothing was seen (or what was seen is NaN)
    return exp2_fast(w - m - kWeightBits) / l;
}
__device__ __forceinline__ float lower_to(float from, float to) { return from == -INFINITY ? 0.f : exp2_fast(from - to); }      // 2^(from - to)

// rows that no sequence has (all of `threads`, who know which they are)
__device__ __forceinline__ void zero_rows_of_none(const Kv8Step& s, const Kv8Attention& a, int dim, long long thread, long long threads) {
    if (!s.first) return;
    const int begin = min(max(s.first[0], 0), s.rows), end = min(max(s.first[s.sequences], begin), s.rows), width = a.heads * dim;
    for (long long i = thread; i < (long long)(begin + s.rows - end) * width; i += threads)
        store_out(a, i < (long long)begin * width ? i : i + (long long)(end - begin) * width, 0.f);
}

}  // namespace
}  // namespace lm
