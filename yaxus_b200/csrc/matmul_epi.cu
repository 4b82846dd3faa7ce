// Matrix products that end in something other than themselves: bias, activation and residual (yx_matmul_epilogue), or
// the log probabilities of a softmax over the product's columns (yx_matmul_logprobs).  No counterpart in the reference,
// whose models have projections without bias and a gated MLP; the products are those of yx_matmul.
#include <algorithm>

#include "yx_epilogue.cuh"

namespace yx {
namespace {

using namespace dev;

// Any shape: a warp per output, pass rows in the grid's y extent.
__global__ void matmul_epilogue_any_kernel(const void *__restrict__ x, int x_dtype, const __nv_bfloat16 *__restrict__ w, uint32_t N, uint32_t K,
                                           const Epilogue e, void *out) {
    const uint32_t n = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5), t = blockIdx.y, lane = threadIdx.x & 31;
    if (n >= N) return;
    float s = 0.0f;
    for (uint32_t k = lane; k < K; k += 32) s += __bfloat162float(w[(size_t)n * K + k]) * load_as_f32(x, x_dtype, (size_t)t * K + k);
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
    if (lane != 0) return;
    const size_t at = (size_t)t * N + n;
    float y = activate(e.bias ? s + e.bias[n] : s, e.act);
    if (e.residual) y += load_as_f32(e.residual, e.out_dtype, at);
    store_from_f32(out, e.out_dtype, at, y);
}

size_t size_of(int dtype) { return dtype == YX_F32 ? 4 : 2; }
bool valid(int dtype) { return dtype == YX_F32 || dtype == YX_F16 || dtype == YX_BF16; }
bool overlap(const void *a, size_t an, const void *b, size_t bn) {
    return a && b && (uintptr_t)a < (uintptr_t)b + bn && (uintptr_t)b < (uintptr_t)a + an;
}

constexpr uint32_t MOST = 0x7fffffffu;   // rows, columns, inner size: coordinates of copies are signed
bool aligned(const void *p, size_t size) { return ((uintptr_t)p & (size - 1)) == 0; }

struct Guard {
    int prev = -1;
    explicit Guard(int dev) {
        cudaGetDevice(&prev);
        if (prev != dev) cudaSetDevice(dev);
        else prev = -1;
    }
    ~Guard() {
        if (prev >= 0) cudaSetDevice(prev);
    }
};

int matmul_any(yx_ctx *ctx, const Product &p, int x_dtype) {
    const size_t xs = size_of(x_dtype), os = size_of(p.e.out_dtype);
    for (uint32_t t0 = 0; t0 < p.T; t0 += 65535u) {   // (the y extent's end)
        Epilogue e = p.e;
        if (e.residual) e.residual = (const char *)e.residual + (size_t)t0 * p.N * os;
        matmul_epilogue_any_kernel<<<dim3((p.N - 1) / 8 + 1, std::min(p.T - t0, 65535u)), 256, 0, ctx->stream>>>(
            (const char *)p.x + (size_t)t0 * p.K * xs, x_dtype, (const __nv_bfloat16 *)p.w, p.N, p.K, e, (char *)p.out + (size_t)t0 * p.N * os);
        ctx->launches++;
        ctx->last_launch = yx_ctx::LAST_OTHER;
        if (int rc = check_cuda(ctx, cudaGetLastError(), "matmul kernel (any shape)")) return rc;
    }
    return YX_OK;
}

// Rows that are taken at a time where a row needs `each` bytes of scratch: all of them within 256 MB (10000 f32 rows of 4096,
// 14000 rows of 128256 columns' statistics, past which reading the weights once more is nothing), else even slices.
constexpr size_t MOST_SCRATCH = (size_t)256 << 20;
uint32_t rows_at_once(uint32_t rows, size_t each) {
    const size_t most = std::max<size_t>(1, MOST_SCRATCH / std::max<size_t>(each, 1));
    if (rows <= most) return rows;
    const uint32_t even = (uint32_t)((rows + ((rows - 1) / most)) / ((rows - 1) / most + 1));
    return most < 256 ? even : (uint32_t)std::min<size_t>(most / 256 * 256, ((size_t)even + 255) / 256 * 256);
}

Product product(const void *x, int x_dtype, const void *w, uint32_t T, uint32_t N, uint32_t K) {
    Product p{};
    p.x = x;
    p.w = w;
    p.T = T;
    p.N = N;
    p.K = K;
    p.parts = x_dtype == YX_BF16 ? 1 : x_dtype == YX_F16 ? 2 : 3;
    p.e.out_dtype = YX_F32;
    return p;
}

}  // namespace
}  // namespace yx

using namespace yx;

extern "C" {

int yx_matmul_epilogue(yx_ctx *ctx, const void *x_dev, int x_dtype, const void *w_bf16_dev, const float *bias_dev, int activation,
                       const void *residual_dev, uint32_t rows, uint32_t n, uint32_t k, void *out_dev, int out_dtype) {
    if (!ctx) return YX_ERR_INVALID;
    if (ctx->status != YX_OK) return ctx->status;
    if (!valid(x_dtype) || !valid(out_dtype)) return fail(ctx, YX_ERR_INVALID, "matmul_epilogue: bad dtype");
    if (activation < YX_ACT_NONE || activation > YX_ACT_SILU) return fail(ctx, YX_ERR_INVALID, "matmul_epilogue: unknown activation");
    if (rows == 0 || n == 0) return YX_OK;
    if (!x_dev || !w_bf16_dev || !out_dev || k == 0) return fail(ctx, YX_ERR_INVALID, "matmul_epilogue: null tensor or empty inner dimension");
    if (rows > MOST || n > MOST || k > MOST) return fail(ctx, YX_ERR_INVALID, "matmul_epilogue: a size of 2^31 or more");
    if (!aligned(x_dev, size_of(x_dtype)) || !aligned(w_bf16_dev, 2) || !aligned(bias_dev, 4) || !aligned(residual_dev, size_of(out_dtype)) ||
        !aligned(out_dev, size_of(out_dtype)))
        return fail(ctx, YX_ERR_INVALID, "matmul_epilogue: a tensor off its type's alignment");
    const size_t x_bytes = (size_t)rows * k * size_of(x_dtype), out_bytes = (size_t)rows * n * size_of(out_dtype);
    if (overlap(out_dev, out_bytes, w_bf16_dev, (size_t)n * k * 2) || overlap(out_dev, out_bytes, bias_dev, (size_t)n * 4))
        return fail(ctx, YX_ERR_INVALID, "matmul_epilogue: the result lies over the weight or the bias");
    if (out_dev != residual_dev && overlap(out_dev, out_bytes, residual_dev, out_bytes))
        return fail(ctx, YX_ERR_INVALID, "matmul_epilogue: the result lies over part of the residual");
    Guard guard(ctx->device);
    Product p = product(x_dev, x_dtype, w_bf16_dev, rows, n, k);
    p.out = out_dev;
    const size_t quad = 4 * size_of(out_dtype);
    p.e = Epilogue{bias_dev, residual_dev, activation, out_dtype, n % 4 == 0 && aligned(bias_dev, 16) && aligned(residual_dev, quad) && aligned(out_dev, quad)};
    const bool tensor = exact_tc_takes(p);
    // Other CTAs still read the rows when a result is written: a result over its own rows takes them from a copy.
    if ((!tensor || exact_tc_reads_rows_late(p)) && overlap(out_dev, out_bytes, x_dev, x_bytes)) {
        if (int rc = grow(ctx, ctx->ep_rows, x_bytes)) return rc;
        if (int rc = check_cuda(ctx, cudaMemcpyAsync(ctx->ep_rows.dev, x_dev, x_bytes, cudaMemcpyDeviceToDevice, ctx->stream), "matmul_epilogue: rows under the result"))
            return rc;
        ctx->last_launch = yx_ctx::LAST_OTHER;
        p.x = ctx->ep_rows.dev;
    }
    if (!tensor) return matmul_any(ctx, p, x_dtype);
    // (a result over rows that are cut into parts waits for all of them to be)
    const bool scratch = exact_tc_copies_rows(p);
    const uint32_t step = scratch && !overlap(out_dev, out_bytes, x_dev, x_bytes) ? rows_at_once(rows, (size_t)k * 2 * p.parts) : rows;
    for (uint32_t r = 0; r < rows; r += step) {
        Product s = p;
        s.x = (const char *)p.x + (size_t)r * k * size_of(x_dtype);
        s.T = std::min(step, rows - r);
        s.out = (char *)out_dev + (size_t)r * n * size_of(out_dtype);
        if (residual_dev) s.e.residual = (const char *)residual_dev + (size_t)r * n * size_of(out_dtype);
        if (int rc = launch_matmul_epilogue_tc(ctx, s)) return rc;
    }
    return YX_OK;
}

int yx_matmul_logprobs(yx_ctx *ctx, const void *x_dev, int x_dtype, const void *w_bf16_dev, uint32_t rows, uint32_t n, uint32_t k,
                       const uint32_t *ids_host, float *logprob_dev, float *entropy_dev) {
    if (!ctx) return YX_ERR_INVALID;
    if (ctx->status != YX_OK) return ctx->status;
    if (!valid(x_dtype)) return fail(ctx, YX_ERR_INVALID, "matmul_logprobs: bad dtype");
    if (rows == 0) return YX_OK;
    if (!x_dev || !w_bf16_dev || !ids_host || !logprob_dev || n == 0 || k == 0)
        return fail(ctx, YX_ERR_INVALID, "matmul_logprobs: null tensor, no columns or empty inner dimension");
    if (rows > MOST || n > MOST || k > MOST) return fail(ctx, YX_ERR_INVALID, "matmul_logprobs: a size of 2^31 or more");
    if (!aligned(x_dev, size_of(x_dtype)) || !aligned(w_bf16_dev, 2) || !aligned(logprob_dev, 4) || !aligned(entropy_dev, 4))
        return fail(ctx, YX_ERR_INVALID, "matmul_logprobs: a tensor off its type's alignment");
    const size_t x_bytes = (size_t)rows * k * size_of(x_dtype), w_bytes = (size_t)n * k * 2, results = (size_t)rows * 4;
    if (overlap(logprob_dev, results, x_dev, x_bytes) || overlap(logprob_dev, results, w_bf16_dev, w_bytes) || overlap(entropy_dev, results, x_dev, x_bytes) ||
        overlap(entropy_dev, results, w_bf16_dev, w_bytes))
        return fail(ctx, YX_ERR_INVALID, "matmul_logprobs: a result lies over the rows or the weight");
    if (overlap(logprob_dev, results, entropy_dev, results)) return fail(ctx, YX_ERR_INVALID, "matmul_logprobs: the results lie over one another");
    for (uint32_t r = 0; r < rows; r++)
        if (ids_host[r] >= n) return fail(ctx, YX_ERR_INVALID, "matmul_logprobs: a token id is outside the vocabulary");
    Guard guard(ctx->device);
    Product p = product(x_dev, x_dtype, w_bf16_dev, rows, n, k);
    if (exact_tc_takes(p)) {
        // (the statistics, then the given tokens' logits)
        const size_t row_stats = (size_t)most_logprob_blocks(ctx, p) * 16;
        const uint32_t step = rows_at_once(rows, std::max(row_stats, exact_tc_copies_rows(p) ? (size_t)k * 2 * p.parts : (size_t)0));
        if (int rc = grow(ctx, ctx->lp_stats, step * (row_stats + 4))) return rc;
        p.stats = ctx->lp_stats.dev;
        p.picked = (float *)(ctx->lp_stats.dev + step * row_stats);
        const uint32_t *ids_dev = nullptr;
        if (rows > 32)
            if (int rc = put_ids(ctx, ids_host, rows, &ids_dev)) return rc;
        for (uint32_t r = 0; r < rows; r += step) {
            Product s = p;
            s.x = (const char *)x_dev + (size_t)r * k * size_of(x_dtype);
            s.T = std::min(step, rows - r);
            s.ids_host = ids_host + r;
            s.ids_dev = ids_dev ? ids_dev + r : nullptr;
            if (int rc = launch_matmul_logprobs_tc(ctx, s)) return rc;
            if (int rc = launch_logprob_blocks(ctx, s.stats, s.blocks, s.picked, s.T, logprob_dev + r, entropy_dev ? entropy_dev + r : nullptr)) return rc;
        }
        return YX_OK;
    }
    // Logits of as many rows as 64 MB hold, then their log probabilities.
    const uint32_t step = (uint32_t)std::max<size_t>(1, std::min<size_t>(rows, ((size_t)64 << 20) / ((size_t)n * 4)));
    if (int rc = grow(ctx, ctx->lp_logits, (size_t)step * n * 4)) return rc;
    p.out = ctx->lp_logits.dev;
    for (uint32_t r = 0; r < rows; r += step) {
        p.x = (const char *)x_dev + (size_t)r * k * size_of(x_dtype);
        p.T = std::min(step, rows - r);
        if (int rc = matmul_any(ctx, p, x_dtype)) return rc;
        if (int rc = launch_logprob_rows(ctx, p.out, YX_F32, p.T, n, n, ids_host + r, 1, 0, logprob_dev + r, entropy_dev ? entropy_dev + r : nullptr,
                                         nullptr, nullptr))
            return rc;
    }
    return YX_OK;
}

}  // extern "C"
