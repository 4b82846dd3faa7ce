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

__device__ __forceinline__ float activate(float y, int act) {
    switch (act) {
    case YX_ACT_RELU: return y < 0.0f ? 0.0f : y;
    case YX_ACT_GELU: return 0.5f * y * (1.0f + erff(y * 0.70710678118654752f));
    // 0.5 (1 + tanh u) = 1 / (1 + exp(-2 u)): one exponential, and no cancellation where tanh is near -1.
    case YX_ACT_GELU_TANH: return y / (1.0f + expf(-1.5957691216057308f * (y + 0.044715f * y * y * y)));
    case YX_ACT_SILU: return y / (1.0f + expf(-y));
    default: return y;
    }
}

// (out of line: a tile's epilogue is unrolled over up to 128 results, and five activations in each would not fit the
// instruction cache; four at a time, the call costs less than the exponentials)
static __device__ __noinline__ float4 activate4(float4 y, int act) {
    return make_float4(activate(y.x, act), activate(y.y, act), activate(y.z, act), activate(y.w, act));
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
// The log probability of a logit under the row's statistics; -inf in a row with nothing left.
__device__ __forceinline__ float log_prob(float l, float m, float log_s) { return m == -INFINITY ? -INFINITY : clean(l) - m - log_s; }
__device__ __forceinline__ float entropy(RowStats r) { return r.m == -INFINITY ? 0.0f : logf(r.s) - r.t / r.s; }

}  // namespace dev
}  // namespace yx
