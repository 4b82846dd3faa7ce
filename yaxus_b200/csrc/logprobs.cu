// Log probabilities under the softmax of rows of logits: of given tokens, the entropy, the most probable tokens
// (yx_logprob_rows).  No counterpart in the reference, which samples on the host; its neighbour here is yx_argmax_rows.
#include <string.h>

#include <algorithm>

#include "yx_epilogue.cuh"

namespace yx {
namespace {

using namespace dev;

// Given tokens on their way to the device: in kernel-parameter space, which is copied with the call, so that nothing on the
// host has to outlive it and a recorded call keeps its own.
constexpr uint32_t IDS_A_LAUNCH = 1000;
struct Ids {
    uint32_t v[IDS_A_LAUNCH];
};
__global__ void __launch_bounds__(256) put_ids_kernel(const __grid_constant__ Ids ids, uint32_t n, uint32_t *__restrict__ out) {
    dependent_entry();
    for (uint32_t i = threadIdx.x; i < n; i += blockDim.x) out[i] = ids.v[i];
}

// A logit and its token as one whole number, larger for a larger logit and, between equal ones, for the smaller token.
__device__ __forceinline__ uint64_t key_of(float l, uint32_t token) {
    const uint32_t b = __float_as_uint(clean(l) + 0.0f);   // (-0 equals 0)
    return (uint64_t)(b & 0x80000000u ? ~b : b | 0x80000000u) << 32 | (uint32_t)~token;
}
__device__ __forceinline__ uint32_t key_token(uint64_t k) { return ~(uint32_t)k; }
__device__ __forceinline__ float key_logit(uint64_t k) {
    const uint32_t b = (uint32_t)(k >> 32);
    return __uint_as_float(b & 0x80000000u ? b & 0x7fffffffu : ~b);
}

__device__ __forceinline__ RowStats merge_warp(RowStats r) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1)
        r = merge(r, RowStats{__shfl_xor_sync(0xffffffffu, r.m, d), __shfl_xor_sync(0xffffffffu, r.s, d), __shfl_xor_sync(0xffffffffu, r.t, d)});
    return r;
}

struct RowsArgs {
    const void *logits;
    int dtype;
    uint32_t cols;
    size_t stride;
    const uint32_t *ids;
    uint32_t n_ids, n_top;
    float *logprob, *entropy;
    uint32_t *top_ids;
    float *top_logprob;
};

// One CTA a row: the statistics in one pass, then a pass for every alternative.
__global__ void __launch_bounds__(256) logprob_rows_kernel(const RowsArgs a) {
    __shared__ RowStats part[8];
    __shared__ uint64_t best[2][8];
    dependent_entry();
    const size_t row = blockIdx.x, base = row * a.stride;
    RowStats r = no_stats();
    for (uint32_t c = threadIdx.x; c < a.cols; c += blockDim.x) r = merge(r, RowStats{clean(load_as_f32(a.logits, a.dtype, base + c)), 1.0f, 0.0f});
    r = merge_warp(r);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = r;
    __syncthreads();
    r = part[0];
    for (int i = 1; i < 8; i++) r = merge(r, part[i]);
    const float log_s = logf(r.s);
    for (uint32_t i = threadIdx.x; i < a.n_ids; i += blockDim.x)
        a.logprob[row * a.n_ids + i] = log_prob(load_as_f32(a.logits, a.dtype, base + a.ids[row * a.n_ids + i]), r.m, log_s);
    if (threadIdx.x == 0 && a.entropy) a.entropy[row] = entropy(r);
    uint64_t below = ~0ull;
    for (uint32_t k = 0; k < a.n_top; k++) {
        uint64_t b = 0;
        for (uint32_t c = threadIdx.x; c < a.cols; c += blockDim.x) {
            const uint64_t key = key_of(load_as_f32(a.logits, a.dtype, base + c), c);
            if (key < below && key > b) b = key;
        }
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) b = max(b, __shfl_xor_sync(0xffffffffu, b, d));
        if ((threadIdx.x & 31) == 0) best[k & 1][threadIdx.x >> 5] = b;
        __syncthreads();
        for (int i = 0; i < 8; i++) b = max(b, best[k & 1][i]);
        below = b;
        if (threadIdx.x == 0) {
            a.top_ids[row * a.n_top + k] = key_token(b);
            a.top_logprob[row * a.n_top + k] = log_prob(key_logit(b), r.m, log_s);
        }
    }
}

// The statistics of a row's blocks of columns, merged; one CTA a row.
__global__ void __launch_bounds__(128) logprob_blocks_kernel(const float4 *__restrict__ stats, uint32_t blocks, const float *__restrict__ picked,
                                                             float *__restrict__ logprob, float *__restrict__ out_entropy) {
    __shared__ RowStats part[4];
    dependent_entry();
    const size_t row = blockIdx.x;
    RowStats r = no_stats();
    for (uint32_t b = threadIdx.x; b < blocks; b += blockDim.x) {
        const float4 f = stats[row * blocks + b];
        r = merge(r, RowStats{f.x, f.y, f.z});
    }
    r = merge_warp(r);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = r;
    __syncthreads();
    if (threadIdx.x != 0) return;
    r = merge(merge(part[0], part[1]), merge(part[2], part[3]));
    logprob[row] = log_prob(picked[row], r.m, logf(r.s));
    if (out_entropy) out_entropy[row] = entropy(r);
}

}  // namespace

int put_ids(yx_ctx *ctx, const uint32_t *host, size_t n, const uint32_t **out) {
    if (int rc = grow(ctx, ctx->lp_ids, n * 4)) return rc;
    *out = (const uint32_t *)ctx->lp_ids.dev;
    ctx->last_launch = yx_ctx::LAST_OTHER;
    Ids ids;
    for (size_t i = 0; i < n; i += IDS_A_LAUNCH) {
        const uint32_t m = (uint32_t)std::min<size_t>(IDS_A_LAUNCH, n - i);
        memcpy(ids.v, host + i, (size_t)m * 4);
        if (int rc = launch_dependent(ctx, "token id kernel launch", put_ids_kernel, dim3(1), dim3(256), 0, ids, m, (uint32_t *)ctx->lp_ids.dev + i)) return rc;
    }
    return YX_OK;
}

int launch_logprob_blocks(yx_ctx *ctx, const void *stats, uint32_t blocks, const float *picked, uint32_t rows, float *logprob, float *entropy) {
    ctx->last_launch = yx_ctx::LAST_OTHER;
    return launch_dependent(ctx, "logprob_blocks kernel launch", logprob_blocks_kernel, dim3(rows), dim3(128), 0, (const float4 *)stats, blocks, picked, logprob, entropy);
}

int launch_logprob_rows(yx_ctx *ctx, const void *logits, int dtype, uint32_t rows, uint32_t cols, size_t stride, const uint32_t *ids_host,
                        uint32_t n_ids, uint32_t n_top, float *logprob, float *entropy, uint32_t *top_ids, float *top_logprob) {
    RowsArgs a{logits, dtype, cols, stride, nullptr, n_ids, n_top, logprob, entropy, top_ids, top_logprob};
    if (n_ids > 0)
        if (int rc = put_ids(ctx, ids_host, (size_t)rows * n_ids, &a.ids)) return rc;
    ctx->last_launch = yx_ctx::LAST_OTHER;
    return launch_dependent(ctx, "logprob_rows kernel launch", logprob_rows_kernel, dim3(rows), dim3(256), 0, a);
}

}  // namespace yx

using namespace yx;

extern "C" int yx_logprob_rows(yx_ctx *ctx, const void *logits_dev, int dtype, uint32_t rows, uint32_t cols, size_t stride,
                               const uint32_t *ids_host, uint32_t n_ids, uint32_t n_top, float *logprob_dev, float *entropy_dev,
                               uint32_t *top_ids_dev, float *top_logprob_dev) {
    if (!ctx) return YX_ERR_INVALID;
    if (ctx->status != YX_OK) return ctx->status;
    if (dtype != YX_F32 && dtype != YX_F16 && dtype != YX_BF16) return fail(ctx, YX_ERR_INVALID, "logprob_rows: bad dtype");
    if (rows == 0) return YX_OK;
    if (!logits_dev || cols == 0) return fail(ctx, YX_ERR_INVALID, "logprob_rows: null tensor or no columns");
    if (stride < cols) return fail(ctx, YX_ERR_INVALID, "logprob_rows: rows lie over one another");
    if (rows > 0x7fffffffu) return fail(ctx, YX_ERR_INVALID, "logprob_rows: too many rows");
    if (((uintptr_t)logits_dev & (dtype == YX_F32 ? 3u : 1u)) != 0 ||
        (((uintptr_t)logprob_dev | (uintptr_t)entropy_dev | (uintptr_t)top_ids_dev | (uintptr_t)top_logprob_dev) & 3u) != 0)
        return fail(ctx, YX_ERR_INVALID, "logprob_rows: a tensor off its type's alignment");
    if (n_top > YX_TOP_MAX || n_top > cols) return fail(ctx, YX_ERR_INVALID, "logprob_rows: more alternatives than YX_TOP_MAX or than there are columns");
    if ((n_ids > 0) != (logprob_dev != nullptr) || (n_ids > 0 && !ids_host)) return fail(ctx, YX_ERR_INVALID, "logprob_rows: given tokens and their result go together");
    if ((n_top > 0) != (top_ids_dev != nullptr) || (n_top > 0) != (top_logprob_dev != nullptr))
        return fail(ctx, YX_ERR_INVALID, "logprob_rows: alternatives and their results go together");
    for (size_t i = 0; i < (size_t)rows * n_ids; i++)
        if (ids_host[i] >= cols) return fail(ctx, YX_ERR_INVALID, "logprob_rows: a token id is outside the vocabulary");
    if (n_ids == 0 && n_top == 0 && !entropy_dev) return YX_OK;
    int prev = -1;
    cudaGetDevice(&prev);
    if (prev != ctx->device) cudaSetDevice(ctx->device);
    const int rc = launch_logprob_rows(ctx, logits_dev, dtype, rows, cols, stride, ids_host, n_ids, n_top, logprob_dev, entropy_dev, top_ids_dev,
                                       top_logprob_dev);
    if (prev >= 0 && prev != ctx->device) cudaSetDevice(prev);
    return rc;
}
