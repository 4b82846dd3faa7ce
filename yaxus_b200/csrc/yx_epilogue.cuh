// What follows the sums of a matrix product: bias, activation and residual, or the statistics of a softmax over the
// product's columns.  Shared by the kernels that finish a product in registers.
#pragma once

#include <math.h>

#include "yx_device.cuh"

namespace yx {

namespace dev {

__device__ __forceinline__ float load_as_f32(const void *p, int dtype, size_t i) {
    if (dtype == YX_F32) return ((const float *)p)[i];
    if (dtype == YX_F16) return __half2float(((const __half *)p)[i]);
    return __bfloat162float(((const __nv_bfloat16 *)p)[i]);
}
__device__ __forceinline__ void store_from_f32(void *p, int dtype, size_t i, float v) {
    if (dtype == YX_F32) ((float *)p)[i] = v;
    else if (dtype == YX_F16) ((__half *)p)[i] = __float2half_rn(v);
    else ((__nv_bfloat16 *)p)[i] = __float2bfloat16_rn(v);
}

// y times the logistic function of u.  The hardware's 2^x and 1 / x (two units and one in the last place): where their
// error counts, y's own is as large.
__device__ __forceinline__ float logistic(float y, float u) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + fast_exp2(-1.4426950408889634f * u)));
    return y * r;
}
// y times the normal distribution's share below it, for y < 0 as the tail it is: 0.5 y (1 + erf(y / sqrt 2)) cancels there (4 % off
// at y = -5, 0 from -5.5 on).  The share beyond a = |y| is exp(-a^2 / 2) t q(t) with t = 1 / (1 + 0.35 a); the coefficients of q are a
// fit to that for a of 0 to 14, 3.2e-8 off at most, 3.4e-7 with f32's roundings up to a = 1 and a^2 half units beyond, the exponent's
// argument.  (Two units of the hardware's and thirteen operations: 2048 bf16 rows x [8192, 1024] to bf16 83 us, with erff
// 91, with erfcf 106; [14336, 4096] 209, 228 and 254.)
__device__ __forceinline__ float gelu(float y) {
    float t;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(t) : "f"(fmaf(0.35f, fabsf(y), 1.0f)));
    float q = -0.0291457232f;
    q = fmaf(q, t, 0.143970788f);
    q = fmaf(q, t, -0.255712599f);
    q = fmaf(q, t, 0.159172505f);
    q = fmaf(q, t, -0.0231088512f);
    q = fmaf(q, t, 0.105507649f);
    q = fmaf(q, t, 0.119832940f);
    q = fmaf(q, t, 0.139861867f);
    q = fmaf(q, t, 0.139621407f);
    const float beyond = q * t * fast_exp2(-0.721347520f * (y * y));
    return y * (y < 0.0f ? beyond : 1.0f - beyond);
}
__device__ __forceinline__ float activate(float y, int act) {
    switch (act) {
    case YX_ACT_RELU: return y < 0.0f ? 0.0f : y;
    case YX_ACT_GELU: return gelu(y);
    // 0.5 (1 + tanh u) is the logistic function of 2 u: no cancellation where tanh is near -1.
    case YX_ACT_GELU_TANH: return logistic(y, 1.5957691216057308f * (y + 0.044715f * y * y * y));
    case YX_ACT_SILU: return logistic(y, y);
    default: return y;
    }
}
__device__ __forceinline__ float4 activate4(float4 y, int act) {   // (the choice once for four, whose exponentials then overlap)
#define YX_FOUR(A) make_float4(activate(y.x, A), activate(y.y, A), activate(y.z, A), activate(y.w, A))
    if (act == YX_ACT_NONE) return y;
    if (act == YX_ACT_SILU) return YX_FOUR(YX_ACT_SILU);
    if (act == YX_ACT_GELU_TANH) return YX_FOUR(YX_ACT_GELU_TANH);
    if (act == YX_ACT_GELU) return YX_FOUR(YX_ACT_GELU);
    return YX_FOUR(YX_ACT_RELU);
#undef YX_FOUR
}

// A softmax's statistics over some of a row's logits l: the largest m, s = sum exp(l - m), t = sum exp(l - m) (l - m).
// log sum exp = m + log s, and the entropy is log s - t / s.  A logit that is no number counts as -inf, +inf as the
// largest f32: `clean` sees to that.  Distances below -150 weigh nothing in f32 (exp(-150) is far below the smallest
// subnormal); cutting them there, which also takes in -inf - -inf, keeps 0 * inf out of t.
constexpr float LEAST_DISTANCE = -150.0f;
constexpr float LOG2_E = 1.4426950408889634f, LARGEST = 3.402823466e38f;
struct RowStats {
    float m, s, t;
};
__device__ __forceinline__ RowStats no_stats() { return RowStats{-INFINITY, 0.0f, 0.0f}; }
__device__ __forceinline__ float clean(float l) { return fminf(fmaxf(l, -INFINITY), LARGEST); }
// (fmaxf passes over an operand that is no number)
__device__ __forceinline__ float distance(float l, float m) { return fmaxf(l - m, LEAST_DISTANCE); }
__device__ __forceinline__ RowStats merge(RowStats a, RowStats b) {
    RowStats r;
    r.m = fmaxf(a.m, b.m);
    const float da = distance(a.m, r.m), db = distance(b.m, r.m);
    const float ca = fast_exp2(da * LOG2_E), cb = fast_exp2(db * LOG2_E);
    r.s = a.s * ca + b.s * cb;
    r.t = ca * (a.t + da * a.s) + cb * (b.t + db * b.s);
    return r;
}
// Two f32 at a time (add.f32x2 and the like: half the issue slots).
struct F2 {
    uint64_t bits;
};
__device__ __forceinline__ F2 f2(float a, float b) {
    F2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r.bits) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void split(F2 v, float &a, float &b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v.bits)); }
__device__ __forceinline__ F2 operator+(F2 a, F2 b) {
    F2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.bits) : "l"(a.bits), "l"(b.bits));
    return r;
}
__device__ __forceinline__ F2 operator*(F2 a, F2 b) {
    F2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.bits) : "l"(a.bits), "l"(b.bits));
    return r;
}
__device__ __forceinline__ F2 fma(F2 a, F2 b, F2 c) {
    F2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.bits) : "l"(a.bits), "l"(b.bits), "l"(c.bits));
    return r;
}

// Adds exp(x - m) to s and exp(x - m) (x - m) to t, for N values.
template <int N>
__device__ __forceinline__ void add_up(const float (&x)[N], float m, F2 &s, F2 &t) {
    const F2 minus_m = f2(-m, -m), log2_e = f2(LOG2_E, LOG2_E);
#pragma unroll
    for (int j = 0; j < N; j += 2) {
        float d0, d1, y0, y1;
        split(f2(x[j], x[j + 1]) + minus_m, d0, d1);
        const F2 d = f2(fmaxf(d0, LEAST_DISTANCE), fmaxf(d1, LEAST_DISTANCE));   // (see distance())
        split(d * log2_e, y0, y1);
        const F2 e = f2(fast_exp2(y0), fast_exp2(y1));
        s = s + e;
        t = fma(e, d, t);
    }
}

// The log probability of a logit under the row's statistics; -inf in a row with nothing left.
__device__ __forceinline__ float log_prob(float l, float m, float log_s) { return m == -INFINITY ? -INFINITY : clean(l) - m - log_s; }
__device__ __forceinline__ float entropy(RowStats r) { return r.m == -INFINITY ? 0.0f : logf(r.s) - r.t / r.s; }

}  // namespace dev
}  // namespace yx
