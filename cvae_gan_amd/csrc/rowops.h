// Helpers shared by the group-norm, linear and distillation kernels.
#pragma once
#include <initializer_list>
#include "common.h"

// ---- activations (CVG_ACT_*) --------------------------------------------------------------------------------
// SiLU and the tanh form of GELU are both v * sigmoid(a(v)): a = v, and a = 2 sqrt(2/pi) (v + 0.044715 v^3) because
// 0.5 (1 + tanh u) = sigmoid(2u).  The bf16 form takes v_exp_f32 and v_rcp_f32 as they are: their errors, and the
// rounding of a log2(e), sit sixteen bits below the rounding to bf16 that follows; in the f32 sums of the parameters'
// gradients, which nothing rounds, they leave 1e-7 to 3e-7 of the norm (65536 terms a channel).  The f32 form (EXACT) adds the low part of
// a log2(e) to first order and one Newton step of the reciprocal: 19 operations where expf and a division take 45, at an
// error of about an ulp.  Beyond |a| = 87 the sigmoid is 0 or 1 to the last bit of f32.
template <bool EXACT> __device__ __forceinline__ float fast_sigmoid(float a) {
    constexpr float L = -1.4426950408889634f, LLO = -1.9259629911266175e-8f;          // -log2(e) = L + LLO
    if (!EXACT) return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(a * L));
    const float x = __builtin_amdgcn_fmed3f(a, -87.f, 87.f);
    const float t = x * L, lo = fmaf(x, LLO, fmaf(x, L, -t));
    float e = __builtin_amdgcn_exp2f(t);
    e = fmaf(e, lo * 0.6931471805599453f, e);
    const float d = 1.0f + e, r = __builtin_amdgcn_rcpf(d);
    const float p = fmaf(fmaf(-d, r, 1.0f), r, r);
    return a < -87.f ? 0.f : p;
}
#define GELU_A 1.5957691216057308f       // 2 sqrt(2 / pi)
#define GELU_B 0.044715f
template <bool EXACT> __device__ __forceinline__ float act_value(float v, int act) {
    switch (act) {
        case CVG_ACT_LRELU: return v > 0.f ? v : LRELU_SLOPE * v;
        case CVG_ACT_SILU: return v * fast_sigmoid<EXACT>(v);
        case CVG_ACT_GELU: return v * fast_sigmoid<EXACT>(GELU_A * (v + GELU_B * v * v * v));
        default: return v;
    }
}
template <bool EXACT> __device__ __forceinline__ float act_slope(float v, int act) {
    switch (act) {
        case CVG_ACT_LRELU: return v > 0.f ? 1.f : LRELU_SLOPE;
        case CVG_ACT_SILU: {
            const float p = fast_sigmoid<EXACT>(v);
            return p * (1.f + v * (1.f - p));
        }
        case CVG_ACT_GELU: {
            // beyond |v| = 16 the slope is 0 or 1 to the last bit; the clamp keeps 0 * inf out of it (NaN passes: the
            // comparisons are false for it)
            const float c = v > 16.f ? 16.f : (v < -16.f ? -16.f : v);
            const float p = fast_sigmoid<EXACT>(GELU_A * (c + GELU_B * c * c * c));
            return p * (1.f + c * (1.f - p) * GELU_A * (1.f + 3.f * GELU_B * c * c));
        }
        default: return 1.f;
    }
}
// eight values at once: the activation is chosen once, outside the loop
template <bool EXACT, int ACT> __device__ __forceinline__ void act_value8_(float (&v)[8]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = act_value<EXACT>(v[j], ACT);
}
template <bool EXACT, int ACT> __device__ __forceinline__ void act_slope8_(float (&v)[8]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = act_slope<EXACT>(v[j], ACT);
}
template <bool EXACT> __device__ __forceinline__ void act_value8(float (&v)[8], int act) {
    if (act == CVG_ACT_LRELU) act_value8_<EXACT, CVG_ACT_LRELU>(v);
    else if (act == CVG_ACT_SILU) act_value8_<EXACT, CVG_ACT_SILU>(v);
    else if (act == CVG_ACT_GELU) act_value8_<EXACT, CVG_ACT_GELU>(v);
}
template <bool EXACT> __device__ __forceinline__ void act_slope8(float (&v)[8], int act) {
    if (act == CVG_ACT_LRELU) act_slope8_<EXACT, CVG_ACT_LRELU>(v);
    else if (act == CVG_ACT_SILU) act_slope8_<EXACT, CVG_ACT_SILU>(v);
    else if (act == CVG_ACT_GELU) act_slope8_<EXACT, CVG_ACT_GELU>(v);
    else act_slope8_<EXACT, CVG_ACT_NONE>(v);
}
static inline bool act_known(int act) { return act >= CVG_ACT_NONE && act <= CVG_ACT_GELU; }

// a barrier for LDS only: global loads and stores stay in flight across it
__device__ __forceinline__ void lds_barrier() {
    asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" : : : "memory");
}

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
    return v;
}
// none of the outputs (null: absent) is one of the inputs or another output
static inline bool apart(std::initializer_list<const void*> outs, std::initializer_list<const void*> ins) {
    for (auto o = outs.begin(); o != outs.end(); ++o) {
        if (!*o) continue;
        for (const void* i : ins) if (*o == i) return false;
        for (auto q = outs.begin(); q != o; ++q) if (*q == *o) return false;
    }
    return true;
}
static inline bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

// 8 elements as they lie in memory (registers that hold a tile between two passes)
template <typename T> struct Raw8;
template <> struct Raw8<bf16> { u32x4 a; };
template <> struct Raw8<float> { u32x4 a, b; };
__device__ __forceinline__ void raw_load(Raw8<bf16>& r, const bf16* p) { r.a = *(const u32x4*)p; }
__device__ __forceinline__ void raw_load(Raw8<float>& r, const float* p) { r.a = *(const u32x4*)p; r.b = *(const u32x4*)(p + 4); }
__device__ __forceinline__ void raw_zero(Raw8<bf16>& r) { r.a = u32x4{0, 0, 0, 0}; }
__device__ __forceinline__ void raw_zero(Raw8<float>& r) { r.a = u32x4{0, 0, 0, 0}; r.b = r.a; }
__device__ __forceinline__ void raw_f32(const Raw8<bf16>& r, float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(r.a[i] << 16);
        v[2 * i + 1] = __uint_as_float(r.a[i] & 0xffff0000u);
    }
}
__device__ __forceinline__ void raw_f32(const Raw8<float>& r, float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) { v[i] = __uint_as_float(r.a[i]); v[4 + i] = __uint_as_float(r.b[i]); }
}
// (exact for values that came from such elements)
__device__ __forceinline__ void raw_pack(Raw8<bf16>& r, const float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) r.a[i] = (__float_as_uint(v[2 * i]) >> 16) | (__float_as_uint(v[2 * i + 1]) & 0xffff0000u);
}
__device__ __forceinline__ void raw_pack(Raw8<float>& r, const float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) { r.a[i] = __float_as_uint(v[i]); r.b[i] = __float_as_uint(v[4 + i]); }
}
// keeps the unpacking of registers where it is written: hoisted above a branch, it would wait for every load at once
__device__ __forceinline__ void pin(Raw8<bf16>& r) { asm volatile("" : "+v"(r.a)); }
__device__ __forceinline__ void pin(Raw8<float>& r) { asm volatile("" : "+v"(r.a), "+v"(r.b)); }
// keeps values in registers: where they come from LDS the compiler would rather read them again at every use
__device__ __forceinline__ void pin(float (&v)[8]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) asm volatile("" : "+v"(v[j]));
}
