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

// ---- rows of logits ---------------------------------------------------------------------------------------
//
// One pass over the logits.  A row is cut into parts, a CTA each (one part where there are rows enough to fill the chip), and a
// part into tiles of 16 logits a thread, the next tile's loads in flight while one is worked on.  A thread keeps the
// statistics (m, s, t) of what it has seen and moves m only when a tile exceeds it.
//
// The best tokens: whatever exceeds the n-th best found so far goes to a list in shared memory, and the list is cut back
// to its n best, in order, when it has grown.  The first tile has no n-th best: the n-th largest of 32 groups' largest serves
// (n numbers are at least that, one of each group), which some n to 4 n logits pass.  Keys of logit and token are all
// different, so that a row of equal logits passes no more.  The parts' lists and statistics meet in the row's last CTA.
constexpr int THREADS = 256, WARPS = THREADS / 32;
constexpr int PER_THREAD = 16;                              // logits of a tile
constexpr int TILE = THREADS * PER_THREAD;
constexpr uint32_t MAX_PARTS = 128;                         // of a row: TILE of their best tokens
constexpr uint32_t MAX_SHARED = 2048;                       // parts of all rows that have more than one
constexpr int LIST_AGAIN = 64;                              // threads that have added to the list, after which it is cut back
constexpr uint32_t IDS_PARAM = 512;                         // given tokens that ride in kernel-parameter space
static_assert(MAX_PARTS * YX_TOP_MAX <= TILE, "the last CTA holds the parts' best tokens as one tile");

struct RowsArgs {
    const void *logits;
    uint32_t cols, parts, n_ids, n_top;
    size_t stride;
    const uint32_t *ids_dev;                                // null: ids
    float *logprob, *entropy;
    uint32_t *top_ids;
    float *top_logprob;
    float4 *part_stats;                                     // [rows][parts]
    uint64_t *part_best;                                    // [rows][parts][n_top]
    uint32_t *arrived;                                      // [rows], zero between launches
    uint32_t ids[IDS_PARAM];
};

struct List {
    uint64_t key[YX_TOP_MAX + (LIST_AGAIN + THREADS) * PER_THREAD];   // the best, what has come since, and one more tile
    uint64_t group[WARPS][32];
    uint64_t warp_best[2][WARPS];
    uint32_t count;
};

// The n-th largest of 32 groups' largest keys; a group is a lane of every warp.  All threads get it.
__device__ __forceinline__ uint64_t nth_of_groups(List &list, uint64_t best, uint32_t n) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    list.group[warp][lane] = best;
    __syncthreads();
    uint64_t g = list.group[0][lane];
#pragma unroll
    for (int w = 1; w < WARPS; w++) g = max(g, list.group[w][lane]);
    uint32_t larger = 0;
#pragma unroll 8
    for (int i = 0; i < 32; i++) {
        const uint64_t other = __shfl_sync(0xffffffffu, g, i);
        larger += other > g || (other == g && i < lane);   // (groups without a token share key 0)
    }
    return __shfl_sync(0xffffffffu, g, __ffs(__ballot_sync(0xffffffffu, larger == n - 1)) - 1);
}

// Adds this thread's key to the list if `in`; all lanes of a warp call it together.
__device__ __forceinline__ void add_to_list(List &list, bool in, uint64_t key) {
    const uint32_t mask = __ballot_sync(0xffffffffu, in);
    if (mask == 0) return;
    const int lane = threadIdx.x & 31;
    uint32_t at = 0;
    if (lane == 0) at = atomicAdd(&list.count, (uint32_t)__popc(mask));
    at = __shfl_sync(0xffffffffu, at, 0) + __popc(mask & ((1u << lane) - 1));
    if (in) list.key[at] = key;
}

// Cuts the list back to its n best, in order; after a barrier, and ends in one.  Returns how many there are.
__device__ __forceinline__ uint32_t cut_list(List &list, uint32_t n) {
    const uint32_t count = list.count;
    if (count <= 2 * THREADS) {
        // A key's place is the number of keys above it.
        uint64_t key[2];
        uint32_t place[2] = {0, 0};
#pragma unroll
        for (int j = 0; j < 2; j++) key[j] = threadIdx.x + j * THREADS < count ? list.key[threadIdx.x + j * THREADS] : 0;
        for (uint32_t i = 0; i < count; i++) {
            const uint64_t other = list.key[i];
#pragma unroll
            for (int j = 0; j < 2; j++) place[j] += other > key[j];
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 2; j++)
            if (key[j] != 0 && place[j] < n) list.key[place[j]] = key[j];
    } else {
        // (a row whose logits rise: nearly all of a tile is on the list)
        uint64_t below = ~0ull, mine = 0;
        for (uint32_t k = 0; k < n; k++) {
            uint64_t b = 0;
            for (uint32_t i = threadIdx.x; i < count; i += THREADS) {
                const uint64_t key = list.key[i];
                if (key < below && key > b) b = key;
            }
#pragma unroll
            for (int d = 16; d > 0; d >>= 1) b = max(b, __shfl_xor_sync(0xffffffffu, b, d));
            if ((threadIdx.x & 31) == 0) list.warp_best[k & 1][threadIdx.x >> 5] = b;
            __syncthreads();
            b = list.warp_best[k & 1][0];
#pragma unroll
            for (int w = 1; w < WARPS; w++) b = max(b, list.warp_best[k & 1][w]);
            below = b;
            if (threadIdx.x == k) mine = b;
        }
        __syncthreads();
        if (threadIdx.x < n) list.key[threadIdx.x] = mine;
    }
    if (threadIdx.x == 0) list.count = min(count, n);
    __syncthreads();
    return min(count, n);
}

// The statistics of all of the CTA's threads, in all of them; `scratch` is the caller's alone.
__device__ __forceinline__ RowStats merge_cta(RowStats r, RowStats *scratch) {
    r = merge_warp(r);
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = r;
    __syncthreads();
    r = scratch[0];
#pragma unroll
    for (int i = 1; i < WARPS; i++) r = merge(r, scratch[i]);
    return r;
}

template <int DTYPE>
struct Tile {
    static constexpr int WIDE = DTYPE == YX_F32 ? 4 : 8;   // logits in 16 bytes
    static constexpr int VECS = PER_THREAD / WIDE;
    uint4 v[VECS];

    // Vectors first, first + THREADS, ... of a row whose logit 0 is element `shift` of vector 0; what lies before the row, behind
    // it, or at or behind vector `end` counts as forbidden.
    __device__ __forceinline__ void load(const char *base, uint32_t shift, uint32_t cols, uint64_t first, uint64_t end) {
#pragma unroll
        for (int i = 0; i < VECS; i++) {
            const uint64_t vec = first + (uint64_t)i * THREADS, c = vec * WIDE;
            constexpr uint32_t none = DTYPE == YX_F32 ? 0xff800000u : DTYPE == YX_F16 ? 0xfc00fc00u : 0xff80ff80u;
            v[i] = make_uint4(none, none, none, none);
            if (vec >= end) continue;
            if (c >= shift && c + WIDE <= (uint64_t)shift + cols) {
                v[i] = __ldcs((const uint4 *)(base + vec * 16));
            } else {
                uint32_t w[4] = {none, none, none, none};
#pragma unroll
                for (int e = 0; e < WIDE; e++) {
                    if (c + e < shift || c + e >= (uint64_t)shift + cols) continue;
                    if constexpr (DTYPE == YX_F32) w[e] = *(const uint32_t *)(base + vec * 16 + e * 4);
                    else w[e / 2] = (w[e / 2] & (e & 1 ? 0xffffu : 0xffff0000u)) | (uint32_t)*(const uint16_t *)(base + vec * 16 + e * 2) << (e & 1 ? 16 : 0);
                }
                v[i] = make_uint4(w[0], w[1], w[2], w[3]);
            }
        }
    }
    __device__ __forceinline__ void unpack(float (&x)[PER_THREAD]) const {
#pragma unroll
        for (int i = 0; i < VECS; i++) {
            const uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
            for (int e = 0; e < 4; e++) {
                if constexpr (DTYPE == YX_F32) {
                    x[4 * i + e] = __uint_as_float(w[e]);
                } else {
                    const float2 f = unpack2<DTYPE == YX_BF16>(w[e]);
                    x[8 * i + 2 * e] = f.x;
                    x[8 * i + 2 * e + 1] = f.y;
                }
            }
        }
    }
    // The token of element j; past any vocabulary before the row and at or behind vector `end`.
    static __device__ __forceinline__ uint32_t token(uint64_t first, int j, uint32_t shift, uint64_t end) {
        const uint64_t vec = first + (uint64_t)(j / WIDE) * THREADS;
        return vec < end ? (uint32_t)(vec * WIDE) + j % WIDE - shift : 0xffffffffu;
    }
};

template <int DTYPE, bool TOP>
__global__ void __launch_bounds__(THREADS, 4) logprob_rows_kernel(const __grid_constant__ RowsArgs a) {
    __shared__ List list;
    __shared__ RowStats scratch[2][WARPS];
    __shared__ bool last;
    using T = Tile<DTYPE>;
    dependent_entry();
    const uint32_t row = blockIdx.x / a.parts, part = blockIdx.x - row * a.parts;
    constexpr int ES = DTYPE == YX_F32 ? 4 : 2;
    const char *logits = (const char *)a.logits + (size_t)row * a.stride * ES;
    const uint32_t shift = (uint32_t)((uintptr_t)logits & 15u) / ES;
    const char *base = logits - shift * ES;
    const uint64_t vecs = ((uint64_t)shift + a.cols + T::WIDE - 1) / T::WIDE;
    const uint64_t v0 = vecs * part / a.parts, v1 = vecs * (part + 1) / a.parts;
    if (TOP && threadIdx.x == 0) list.count = 0;

    RowStats r = no_stats();
    float least = -INFINITY;   // the n-th best logit found, once there are n
    int added = 0;
    T next;
    next.load(base, shift, a.cols, v0 + threadIdx.x, v1);
    for (uint64_t v = v0; v < v1; v += T::VECS * THREADS) {
        const T tile = next;
        next.load(base, shift, a.cols, v + T::VECS * THREADS + threadIdx.x, v1);
        float x[PER_THREAD];
        tile.unpack(x);
        float most = x[0];
#pragma unroll
        for (int j = 1; j < PER_THREAD; j++) most = fmaxf(most, x[j]);
        if (most > r.m) {
            if (most == INFINITY) {
#pragma unroll
                for (int j = 0; j < PER_THREAD; j++) x[j] = clean(x[j]);
                most = clean(most);
            }
            const float d = distance(r.m, most), c = fast_exp2(d * LOG2_E);
            r.t = c * (r.t + d * r.s);
            r.s *= c;
            r.m = most;
        }
#pragma unroll
        for (int j = 0; j < PER_THREAD; j++) {
            const float d = distance(x[j], r.m), e = fast_exp2(d * LOG2_E);
            r.s += e;
            r.t += e * d;
        }
        if constexpr (TOP) {
            if (v == v0) {
                uint64_t best = 0;
#pragma unroll
                for (int j = PER_THREAD - 1; j >= 0; j--) {
                    const uint32_t token = T::token(v + threadIdx.x, j, shift, v1);
                    if (token < a.cols) best = max(best, key_of(x[j], token));
                }
                const uint64_t least_key = nth_of_groups(list, best, a.n_top);
#pragma unroll
                for (int j = 0; j < PER_THREAD; j++) {
                    const uint32_t token = T::token(v + threadIdx.x, j, shift, v1);
                    const uint64_t key = token < a.cols ? key_of(x[j], token) : 0;
                    add_to_list(list, key != 0 && key >= least_key, key);
                }
            } else if (__any_sync(0xffffffffu, most > least)) {
                // (tokens come in order: an equal one later is no better)
#pragma unroll
                for (int j = 0; j < PER_THREAD; j++) add_to_list(list, x[j] > least, key_of(x[j], T::token(v + threadIdx.x, j, shift, v1)));
            }
            // (counted by the barrier itself: the list's own count may be moving again when the last thread reads it)
            added += __syncthreads_count(v == v0 || most > least);
            if (added > LIST_AGAIN) {
                added = 0;
                if (cut_list(list, a.n_top) == a.n_top) least = key_logit(list.key[a.n_top - 1]);
                __syncthreads();
            }
        }
    }
    uint32_t found = 0;
    if constexpr (TOP) {
        __syncthreads();
        found = cut_list(list, a.n_top);
    }
    r = merge_cta(r, scratch[0]);
    if (a.parts > 1) {
        const size_t mine = (size_t)row * a.parts + part;
        if constexpr (TOP)
            if (threadIdx.x < a.n_top) __stcg(a.part_best + mine * a.n_top + threadIdx.x, threadIdx.x < found ? list.key[threadIdx.x] : 0ull);
        if (threadIdx.x == 0) __stcg(a.part_stats + mine, make_float4(r.m, r.s, r.t, 0.0f));
        __threadfence();
        __syncthreads();
        if (threadIdx.x == 0) {
            last = atomicAdd(a.arrived + row, 1u) + 1 == a.parts;
            if (last) a.arrived[row] = 0u;
        }
        __syncthreads();
        if (!last) return;
        __threadfence();
        r = no_stats();
        if (threadIdx.x < a.parts) {
            const float4 f = __ldcg(a.part_stats + (size_t)row * a.parts + threadIdx.x);
            r = RowStats{f.x, f.y, f.z};
        }
        if constexpr (TOP) {
            const uint32_t keys = a.parts * a.n_top;
            const uint64_t *from = a.part_best + (size_t)row * keys;
            uint64_t key[PER_THREAD], best = 0;
#pragma unroll
            for (int j = 0; j < PER_THREAD; j++) {
                const uint32_t i = threadIdx.x + j * THREADS;
                key[j] = i < keys ? __ldcg(from + i) : 0;
                best = max(best, key[j]);
            }
            if (threadIdx.x == 0) list.count = 0;
            const uint64_t least_key = nth_of_groups(list, best, a.n_top);
#pragma unroll
            for (int j = 0; j < PER_THREAD; j++) {
                if (j * THREADS >= keys) break;
                add_to_list(list, key[j] != 0 && key[j] >= least_key, key[j]);
            }
            __syncthreads();
            cut_list(list, a.n_top);
        }
        r = merge_cta(r, scratch[1]);
    }
    const float log_s = logf(r.s);
    const uint32_t *ids = a.ids_dev ? a.ids_dev : a.ids;
    for (uint32_t i = threadIdx.x; i < a.n_ids; i += THREADS)
        a.logprob[(size_t)row * a.n_ids + i] = log_prob(load_as_f32(logits, DTYPE, ids[(size_t)row * a.n_ids + i]), r.m, log_s);
    if (threadIdx.x == 0 && a.entropy) a.entropy[row] = entropy(r);
    if constexpr (TOP) {
        if (threadIdx.x < a.n_top) {
            const uint64_t key = list.key[threadIdx.x];
            a.top_ids[(size_t)row * a.n_top + threadIdx.x] = key_token(key);
            a.top_logprob[(size_t)row * a.n_top + threadIdx.x] = log_prob(key_logit(key), r.m, log_s);
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
    RowsArgs a;
    a.logits = logits;
    a.cols = cols;
    a.stride = stride;
    a.n_ids = n_ids;
    a.n_top = n_top;
    a.ids_dev = nullptr;
    a.logprob = logprob;
    a.entropy = entropy;
    a.top_ids = top_ids;
    a.top_logprob = top_logprob;
    // Rows that fill the chip by themselves are a CTA each; fewer are cut into parts of a tile or more.
    const uint32_t tiles = (uint32_t)(((uint64_t)cols + TILE - 1) / TILE), want = 4 * (uint32_t)ctx->sm_count;
    a.parts = rows >= want / 2 ? 1 : std::min({tiles, MAX_PARTS, (want + rows - 1) / rows, MAX_SHARED / rows});
    // (at the most any call needs, for recordings)
    const size_t stats = MAX_SHARED * sizeof(float4), best = (size_t)MAX_SHARED * YX_TOP_MAX * sizeof(uint64_t);
    char *before = ctx->lp_parts.dev;
    if (int rc = grow(ctx, ctx->lp_parts, stats + best + MAX_SHARED * sizeof(uint32_t))) return rc;
    a.part_stats = (float4 *)ctx->lp_parts.dev;
    a.part_best = (uint64_t *)(ctx->lp_parts.dev + stats);
    a.arrived = (uint32_t *)(ctx->lp_parts.dev + stats + best);
    if (ctx->lp_parts.dev != before)
        if (int rc = check_cuda(ctx, cudaMemsetAsync(a.arrived, 0, MAX_SHARED * sizeof(uint32_t), ctx->stream), "logprob_rows: counters")) return rc;
    const size_t given = (size_t)rows * n_ids;
    if (given > IDS_PARAM) {
        if (int rc = put_ids(ctx, ids_host, given, &a.ids_dev)) return rc;
    } else if (given > 0) {
        memcpy(a.ids, ids_host, given * 4);
    }
    ctx->last_launch = yx_ctx::LAST_OTHER;
    auto go = [&](auto kernel) { return launch_dependent(ctx, "logprob_rows kernel launch", kernel, dim3(rows * a.parts), dim3(THREADS), 0, a); };
    if (dtype == YX_F32) return n_top > 0 ? go(logprob_rows_kernel<YX_F32, true>) : go(logprob_rows_kernel<YX_F32, false>);
    if (dtype == YX_F16) return n_top > 0 ? go(logprob_rows_kernel<YX_F16, true>) : go(logprob_rows_kernel<YX_F16, false>);
    return n_top > 0 ? go(logprob_rows_kernel<YX_BF16, true>) : go(logprob_rows_kernel<YX_BF16, false>);
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
    if (rows > 0x7fffffffu || cols > 0x7fffffffu) return fail(ctx, YX_ERR_INVALID, "logprob_rows: more than 2^31 rows or columns");
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
