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
// (Two sizes: a launch takes longer with 32 KB of parameters than with four, and three launches longer than that.)
template <uint32_t N>
struct Ids {
    uint32_t v[N];
};
constexpr uint32_t IDS_CTA = 256;   // (an SM reads parameters one thread's after another: 8000 tokens by one CTA took 10 us)
template <uint32_t N>
__global__ void __launch_bounds__(IDS_CTA) put_ids_kernel(const __grid_constant__ Ids<N> ids, uint32_t n, uint32_t *__restrict__ out) {
    dependent_entry();
    const uint32_t i = blockIdx.x * IDS_CTA + threadIdx.x;
    if (i < n) out[i] = ids.v[i];
}
template <uint32_t N>
int put_ids_launch(yx_ctx *ctx, const uint32_t *host, uint32_t n, uint32_t *out) {
    Ids<N> ids;
    memcpy(ids.v, host, (size_t)n * 4);
    return launch_dependent(ctx, "token id kernel launch", put_ids_kernel<N>, dim3((n + IDS_CTA - 1) / IDS_CTA), dim3(IDS_CTA), 0, ids, n, out);
}
constexpr uint32_t FEW_IDS = 1000, MANY_IDS = 8000;

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
// statistics (m, s, t) of what it has seen, m its warp's largest logit so far, and notes the tile that has its largest and the
// largest outside that tile.
//
// The n best tokens of a part come from that: of 32 or 64 groups of threads, the n-th largest of the groups' best is a bound that n
// tokens reach, and only the n or so threads whose best reaches it can hold others that do.  Of most of those the best tile alone
// can, whose logits are read once more; of the few whose others may all are, a warp to a thread's (2048 rows of 50257 f32 with
// five and 20 tokens 76.2 and 79.4 us; all logits of all of them 76.0 and 94.2, as what is read is 16 bytes in every 4096).  What reaches
// the bound (n to some 2 n tokens) is put in order.  Where too many logits equal it the bound is a key of logit and
// token, which are all different.  (With a list that grew as the logits went by, and a barrier a tile for it, five tokens took
// 170 us.)  The parts' tokens and statistics meet in the row's last CTA.
constexpr int THREADS = 256, WARPS = THREADS / 32;
constexpr int PER_THREAD = 16;                              // logits of a tile
constexpr int TILE = THREADS * PER_THREAD;
constexpr uint32_t MAX_PARTS = 128;                         // of a row
constexpr uint32_t MAX_SHARED = 2048;                       // parts of all rows that have more than one
constexpr uint32_t LIST = 512;                              // tokens put in order by counting
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
    uint64_t *part_best;                                    // [rows][n_top][parts]
    uint32_t *arrived;                                      // [rows], zero between launches
    uint32_t ids[IDS_PARAM];
};

struct Best {
    uint64_t key[LIST];
    uint64_t group[WARPS][32];
    uint64_t warp_best[2][WARPS];
    uint64_t least;
    uint32_t count, threads, tiles;
    uint8_t thread[THREADS];     // whose all have to be looked at
    uint2 tile[THREADS];         // a tile and a thread
};

// The n-th largest of the largest keys of 32 groups of threads, lanes of every warp, or of 64 where n is near 32: the least of 32
// groups is reached by some 130 keys, the 32nd of 64 by 44 (16 rows of 32000 bf16 with 32 tokens 17.6 and 9.8 us, with 20 tokens 8.0 and
// 8.2).  All threads get it, after two barriers.
__device__ __forceinline__ uint64_t nth_of_groups(Best &b, uint64_t best, uint32_t n) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    b.group[warp][lane] = best;
    __syncthreads();
    if (warp == 0) {
        uint64_t g = best;
        if (n <= 20) {
#pragma unroll
            for (int w = 1; w < WARPS; w++) g = max(g, b.group[w][lane]);
            uint32_t above = 0;   // (groups without a token share key 0)
#pragma unroll
            for (int i = 0; i < 32; i++) {
                const uint64_t other = __shfl_sync(0xffffffffu, g, i);
                above += other > g || (other == g && i < lane);
            }
            if (above == n - 1) b.least = g;
        } else {
            // (the list has nothing on it yet, and lends its room)
#pragma unroll
            for (int w = 2; w < WARPS; w += 2) g = max(g, b.group[w][lane]);
            b.key[lane] = g;
            g = b.group[1][lane];
#pragma unroll
            for (int w = 3; w < WARPS; w += 2) g = max(g, b.group[w][lane]);
            b.key[32 + lane] = g;
            __syncwarp();
#pragma unroll 1
            for (int j = lane; j < 64; j += 32) {
                g = b.key[j];
                uint32_t above = 0;
#pragma unroll 8
                for (int i = 0; i < 64; i++) above += b.key[i] > g || (b.key[i] == g && i < j);
                if (above == n - 1) b.least = g;
            }
        }
    }
    __syncthreads();
    return b.least;
}

// Adds this thread's key to the list if `in`; all lanes of a warp call it together.  The list's end is not passed, but
// counted on.
__device__ __forceinline__ void add_to_list(Best &b, bool in, uint64_t key) {
    const uint32_t mask = __ballot_sync(0xffffffffu, in);
    if (mask == 0) return;
    const int lane = threadIdx.x & 31;
    uint32_t at = 0;
    if (lane == 0) at = atomicAdd(&b.count, (uint32_t)__popc(mask));
    at = __shfl_sync(0xffffffffu, at, 0) + __popc(mask & ((1u << lane) - 1));
    if (in && at < LIST) b.key[at] = key;
}

// The n best of the list, in order, to its front; after a barrier, and ends in one.  If more than LIST have been added, the n
// best of `source(0 .. size - 1)` instead, a pass over all of it for each (rows made for it: most of the largest logits in one
// of 32 places of every 128 or 256).
template <typename F>
__device__ __forceinline__ void order_list(Best &b, uint32_t n, uint32_t size, F source) {
    const uint32_t count = b.count;
    if (count <= LIST) {
        // A key's place is the number of keys above it.
        constexpr int EACH = LIST / THREADS;
        uint64_t key[EACH];
        uint32_t place[EACH] = {};
#pragma unroll
        for (int j = 0; j < EACH; j++) key[j] = threadIdx.x + j * THREADS < count ? b.key[threadIdx.x + j * THREADS] : 0;
        if (threadIdx.x < count) {
#pragma unroll 4
            for (uint32_t i = 0; i < count; i++) {
                const uint64_t other = b.key[i];
#pragma unroll
                for (int j = 0; j < EACH; j++) place[j] += other > key[j];
            }
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < EACH; j++)
            if (key[j] != 0 && place[j] < n) b.key[place[j]] = key[j];
    } else {
        uint64_t below = ~0ull, mine = 0;
        for (uint32_t k = 0; k < n; k++) {
            uint64_t best = 0;
            for (uint32_t i = threadIdx.x; i < size; i += THREADS) {
                const uint64_t key = source(i);
                if (key < below && key > best) best = key;
            }
#pragma unroll
            for (int d = 16; d > 0; d >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, d));
            if ((threadIdx.x & 31) == 0) b.warp_best[k & 1][threadIdx.x >> 5] = best;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < WARPS; w++) best = max(best, b.warp_best[k & 1][w]);
            below = best;
            if (threadIdx.x == k) mine = best;
        }
        if (threadIdx.x < n) b.key[threadIdx.x] = mine;   // (all have read the list's count; nobody reads its keys)
    }
    __syncthreads();
}

__device__ __forceinline__ float warp_max(float v) {   // (passes over what is no number)
    float r;
    asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
    return r;
}
// (s, t) of statistics under another m
__device__ __forceinline__ RowStats moved(RowStats r, float m) {
    const float d = distance(r.m, m), c = fast_exp2(d * LOG2_E);
    return RowStats{m, c * r.s, c * (r.t + d * r.s)};
}
template <int LANES>
__device__ __forceinline__ RowStats warp_sum(RowStats r) {
    r = moved(r, warp_max(r.m));
#pragma unroll
    for (int d = LANES / 2; d > 0; d >>= 1) {
        r.s += __shfl_xor_sync(0xffffffffu, r.s, d);
        r.t += __shfl_xor_sync(0xffffffffu, r.t, d);
    }
    return r;
}
// The statistics of all of the CTA's threads: share_stats by all, a barrier, all_stats.
__device__ __forceinline__ void share_stats(RowStats r, RowStats *scratch) {
    r = warp_sum<32>(r);
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = r;
}
__device__ __forceinline__ RowStats all_stats(const RowStats *scratch) { return warp_sum<WARPS>(scratch[threadIdx.x & (WARPS - 1)]); }

template <int DTYPE, int N = PER_THREAD>
struct Tile {
    static constexpr int WIDE = DTYPE == YX_F32 ? 4 : 8;   // logits in 16 bytes
    static constexpr int VECS = N / WIDE;
    uint4 v[VECS];

    // Vectors first, first + step, ... , all inside the row.
    __device__ __forceinline__ void load_inside(const char *base, uint32_t first, uint32_t step) {
        const uint4 *p = (const uint4 *)base + first;
#pragma unroll
        for (int i = 0; i < VECS; i++) v[i] = p[(size_t)i * step];
    }
    // The same of a row whose logit 0 is element `shift` of vector 0: what lies before the row, behind it, or at or behind
    // vector `end` counts as forbidden.
    __device__ __forceinline__ void load(const char *base, uint32_t shift, uint32_t cols, uint32_t first, uint32_t step, uint32_t end) {
#pragma unroll
        for (int i = 0; i < VECS; i++) {
            const uint32_t vec = first + i * step;
            const uint64_t c = (uint64_t)vec * WIDE;
            constexpr uint32_t none = DTYPE == YX_F32 ? 0xff800000u : DTYPE == YX_F16 ? 0xfc00fc00u : 0xff80ff80u;
            v[i] = make_uint4(none, none, none, none);
            if (vec >= end) continue;
            if (c >= shift && c + WIDE <= (uint64_t)shift + cols) {
                v[i] = *((const uint4 *)base + vec);
            } else {
                uint32_t w[4] = {none, none, none, none};
#pragma unroll
                for (int e = 0; e < WIDE; e++) {
                    if (c + e < shift || c + e >= (uint64_t)shift + cols) continue;
                    if constexpr (DTYPE == YX_F32) w[e] = *((const uint32_t *)base + c + e);
                    else w[e / 2] = (w[e / 2] & (e & 1 ? 0xffffu : 0xffff0000u)) | (uint32_t)*((const uint16_t *)base + c + e) << (e & 1 ? 16 : 0);
                }
                v[i] = make_uint4(w[0], w[1], w[2], w[3]);
            }
        }
    }
    __device__ __forceinline__ void unpack(float (&x)[N]) const {
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
    static __device__ __forceinline__ uint32_t first_token(uint32_t vec, uint32_t shift) { return vec > 0 ? vec * WIDE - shift : 0u; }
};

// Five CTAs an SM: 48 registers a thread, which is tight (2048 rows of 50257 bf16 with five tokens then 58 us; four CTAs 64, three
// 73, six with half the logits in flight each 69; with the given token's logit in shared memory, which leaves next to no spills, 55).
template <int DTYPE, bool TOP>
__global__ void __launch_bounds__(THREADS, 5) logprob_rows_kernel(const __grid_constant__ RowsArgs a) {
    __shared__ Best b;
    __shared__ RowStats scratch[2][WARPS];
    __shared__ bool last;
    __shared__ float given_s[THREADS];
    using T = Tile<DTYPE>;
    dependent_entry();
    const uint32_t row = blockIdx.x / a.parts, part = blockIdx.x - row * a.parts;
    constexpr int ES = DTYPE == YX_F32 ? 4 : 2;
    const char *logits = (const char *)a.logits + (size_t)row * a.stride * ES;
    const uint32_t shift = (uint32_t)((uintptr_t)logits & 15u) / ES;
    const char *base = logits - shift * ES;
    const uint32_t vecs = (uint32_t)(((uint64_t)shift + a.cols + T::WIDE - 1) / T::WIDE);
    const uint32_t v0 = (uint32_t)((uint64_t)vecs * part / a.parts), v1 = (uint32_t)((uint64_t)vecs * (part + 1) / a.parts);
    // Tiles that begin in [in0, in1) lie inside the row and the part.
    constexpr uint32_t STEP = T::VECS * THREADS;
    const uint32_t in0 = shift > 0 && part == 0 ? 1 : v0, inside = min(v1, (uint32_t)(((uint64_t)shift + a.cols) / T::WIDE));
    const uint32_t in1 = inside >= STEP - 1 ? inside - (STEP - 1) : 0;

    // The first given token's logit is asked for at once: behind the sums it would be one more trip to memory.
    const uint32_t *ids = (a.ids_dev ? a.ids_dev : a.ids) + (size_t)row * a.n_ids;
    const float given = threadIdx.x < a.n_ids ? load_as_f32(logits, DTYPE, ids[threadIdx.x]) : 0.0f;

    RowStats r = no_stats();
    F2 s2 = f2(0.0f, 0.0f), t2 = s2;
    float best = -INFINITY;
    float second = -INFINITY;         // the largest outside that tile
    uint32_t best_at = 0xffffffffu;   // the tile of the first of this thread's largest logits
    T next;
    auto load = [&](uint32_t v) {
        if (v >= in0 && v < in1) next.load_inside(base, v + threadIdx.x, THREADS);
        else next.load(base, shift, a.cols, v + threadIdx.x, THREADS, v1);
    };
    load(v0);
    if (threadIdx.x < a.n_ids) given_s[threadIdx.x] = given;   // (a register is worth more)
    for (uint32_t v = v0; v < v1; v += STEP) {
        const T tile = next;
        if (v + STEP < v1) load(v + STEP);
        float x[PER_THREAD];
        tile.unpack(x);
        float most = x[0];
#pragma unroll
        for (int j = 1; j < PER_THREAD; j++) most = fmaxf(most, x[j]);
        if constexpr (TOP) {
            const float c = clean(most);
            second = fmaxf(second, fminf(best, c));
            if (c > best) {
                best = c;
                best_at = v;
            }
        }
        // m is never below a logit that has been added: where one token has nearly all the weight, log s and l - m are then near 0 and
        // not near 8 and -8 with their last places to lose, s >= 1 and t <= 0, and no probability exceeds 1.  One m for a warp takes
        // one instruction, and moves in the first tiles and with the few logits that stand out of a row.
        most = warp_max(most);
        if (most > r.m) {
            if (most == INFINITY) {
#pragma unroll
                for (int j = 0; j < PER_THREAD; j++) x[j] = clean(x[j]);
                most = clean(most);
            }
            const float d = distance(r.m, most), c = fast_exp2(d * LOG2_E);
            t2 = f2(c, c) * fma(f2(d, d), s2, t2);
            s2 = f2(c, c) * s2;
            r.m = most;
        }
        add_up(x, r.m, s2, t2);
    }
    {
        float x, y;
        split(s2, x, y);
        r.s = x + y;
        split(t2, x, y);
        r.t = x + y;
    }
    share_stats(r, scratch[0]);
    if constexpr (TOP) {
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
        // Puts on the list what `reaches` of the logits of the threads that are `in`, or of their best tile if that is `one`; between
        // barriers.
        auto look_again = [&](bool in, bool one, auto reaches) {
            if (in) {
                if (one) b.tile[atomicAdd(&b.tiles, 1u)] = make_uint2(best_at, threadIdx.x);
                else b.thread[atomicAdd(&b.threads, 1u)] = (uint8_t)threadIdx.x;
            }
            __syncthreads();
            auto look = [&](uint32_t own) {
                Tile<DTYPE, T::WIDE> again;
                again.load(base, shift, a.cols, own, 0, v1);
                float x[T::WIDE];
                again.unpack(x);
#pragma unroll
                for (int e = 0; e < T::WIDE; e++) {
                    const uint32_t t = own * T::WIDE + e - shift;
                    if (!(own < v1 && t < a.cols && reaches(x[e], t))) continue;
                    const uint32_t at = atomicAdd(&b.count, 1u);   // (few are: a vote for each logit takes longer)
                    if (at < LIST) b.key[at] = key_of(x[e], t);
                }
            };
            for (uint32_t i = threadIdx.x; i < b.tiles * T::VECS; i += THREADS) {
                const uint2 at = b.tile[i / T::VECS];
                look(at.x + at.y + i % T::VECS * THREADS);
            }
            for (uint32_t i = warp; i < b.threads; i += WARPS) {
                for (uint32_t v = v0 + b.thread[i]; v < v1; v += 32 * THREADS) {
                    if (__any_sync(0xffffffffu, *(volatile uint32_t *)&b.count > LIST)) break;
                    look(v + lane * THREADS);
                }
            }
            __syncthreads();
        };
        if (threadIdx.x == 0) b.count = b.threads = b.tiles = 0;
        // The bound is a logit; only where too many equal it (or it is the forbidden's) is it a logit and a token.
        const uint64_t bound = nth_of_groups(b, v0 + threadIdx.x < v1 ? key_of(best, 0) : 0, a.n_top);
        const float least = key_logit(bound);
        bool precise = bound == 0 || least == -INFINITY;
        if (!precise) {
            look_again(best >= least, second < least, [&](float x, uint32_t) { return x >= least; });
            precise = b.count > LIST;
            __syncthreads();
        }
        if (precise) {
            uint32_t token = T::first_token(v0 + threadIdx.x, shift);   // (all of them -inf or no number)
            if (best_at != 0xffffffffu) {
                next.load(base, shift, a.cols, best_at + threadIdx.x, THREADS, v1);
                float x[PER_THREAD];
                next.unpack(x);
                int at = 0;
#pragma unroll
                for (int j = PER_THREAD - 1; j >= 0; j--)
                    if (clean(x[j]) == best) at = j;
                token = (best_at + threadIdx.x + at / T::WIDE * THREADS) * T::WIDE + at % T::WIDE - shift;
            }
            if (threadIdx.x == 0) b.count = b.threads = b.tiles = 0;
            const uint64_t mine = v0 + threadIdx.x < v1 ? key_of(best, token) : 0;
            const uint64_t reached = nth_of_groups(b, mine, a.n_top);
            look_again(mine != 0 && mine >= reached, false, [&](float x, uint32_t t) { return key_of(x, t) >= reached; });
        }
        const uint32_t t0 = T::first_token(v0, shift), t1 = min(a.cols, v1 * T::WIDE - shift);
        order_list(b, a.n_top, t1 - t0, [&](uint32_t i) { return key_of(load_as_f32(logits, DTYPE, t0 + i), t0 + i); });
    } else {
        __syncthreads();
    }
    r = all_stats(scratch[0]);
    if (a.parts > 1) {
        if constexpr (TOP)   // (a part of fewer than n_top tokens has them all on the list)
            if (threadIdx.x < a.n_top) __stcg(a.part_best + ((size_t)row * a.n_top + threadIdx.x) * a.parts + part, threadIdx.x < b.count ? b.key[threadIdx.x] : 0ull);
        if (threadIdx.x == 0) __stcg(a.part_stats + (size_t)row * a.parts + part, make_float4(r.m, r.s, r.t, 0.0f));
        __syncthreads();
        if (threadIdx.x == 0) {
            __threadfence();   // (for all of the CTA's stores, which the barrier puts before it)
            last = atomicAdd(a.arrived + row, 1u) + 1 == a.parts;
            if (last) a.arrived[row] = 0u;
            b.count = 0;
        }
        __syncthreads();
        if (!last) return;
        __threadfence();
        r = no_stats();
        if (threadIdx.x < a.parts) {
            const float4 f = __ldcg(a.part_stats + (size_t)row * a.parts + threadIdx.x);
            r = RowStats{f.x, f.y, f.z};
        }
        share_stats(r, scratch[1]);
        if constexpr (TOP) {
            // (best ones first, so that the groups' largest are the parts' first few)
            const uint32_t keys = a.parts * a.n_top;
            const uint64_t *from = a.part_best + (size_t)row * keys;
            uint64_t key[PER_THREAD], best = 0;
#pragma unroll
            for (int j = 0; j < PER_THREAD; j++) {
                const uint32_t i = threadIdx.x + j * THREADS;
                key[j] = i < keys ? __ldcg(from + i) : 0;
                best = max(best, key[j]);
            }
            const uint64_t least = nth_of_groups(b, best, a.n_top);
#pragma unroll
            for (int j = 0; j < PER_THREAD; j++) {
                if (j * THREADS >= keys) break;
                add_to_list(b, key[j] != 0 && key[j] >= least, key[j]);
            }
            __syncthreads();
            order_list(b, a.n_top, keys, [&](uint32_t i) { return __ldcg(from + i); });
        } else {
            __syncthreads();
        }
        r = all_stats(scratch[1]);
    }
    const float log_s = logf(r.s);
    if (threadIdx.x < a.n_ids) a.logprob[(size_t)row * a.n_ids + threadIdx.x] = log_prob(given_s[threadIdx.x], r.m, log_s);
    for (uint32_t i = threadIdx.x + THREADS; i < a.n_ids; i += THREADS)
        a.logprob[(size_t)row * a.n_ids + i] = log_prob(load_as_f32(logits, DTYPE, ids[i]), r.m, log_s);
    if (threadIdx.x == 0 && a.entropy) a.entropy[row] = entropy(r);
    if constexpr (TOP) {
        if (threadIdx.x < a.n_top) {
            const uint64_t key = b.key[threadIdx.x];
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
    // (all asked for before the first is used: one trip to memory for up to 512 blocks; a row and a head of [128256, 1024] 46.1 us, with
    // a block at a time 47.6)
    const float given = threadIdx.x == 0 ? picked[row] : 0.0f;
    RowStats r = no_stats();
    for (uint32_t b = threadIdx.x; b < blocks; b += 4 * 128) {
        float4 f[4];
#pragma unroll
        for (int j = 0; j < 4; j++) f[j] = b + 128 * j < blocks ? stats[row * blocks + b + 128 * j] : make_float4(-INFINITY, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int j = 0; j < 4; j++) r = merge(r, RowStats{f[j].x, f[j].y, f[j].z});
    }
    r = merge_warp(r);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = r;
    __syncthreads();
    if (threadIdx.x != 0) return;
    r = merge(merge(part[0], part[1]), merge(part[2], part[3]));
    logprob[row] = log_prob(given, r.m, logf(r.s));
    if (out_entropy) out_entropy[row] = entropy(r);
}

}  // namespace

int put_ids(yx_ctx *ctx, const uint32_t *host, size_t n, const uint32_t **out) {
    if (int rc = grow(ctx, ctx->lp_ids, n * 4)) return rc;
    *out = (const uint32_t *)ctx->lp_ids.dev;
    ctx->last_launch = yx_ctx::LAST_OTHER;
    for (size_t i = 0; i < n; i += MANY_IDS) {
        const uint32_t m = (uint32_t)std::min<size_t>(MANY_IDS, n - i);
        uint32_t *to = (uint32_t *)ctx->lp_ids.dev + i;
        if (int rc = m <= FEW_IDS ? put_ids_launch<FEW_IDS>(ctx, host + i, m, to) : put_ids_launch<MANY_IDS>(ctx, host + i, m, to)) return rc;
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
    // A CTA a row, unless there are few rows and long ones: a CTA takes 48 bytes a nanosecond, and parts meeting in a last
    // CTA cost 3 us (one row of 50257 f32 with five tokens 8.5 us whole and 7.6 in 13 parts, of 150000 16.9 and 8.2; 100
    // rows of 50257 9.5 whole, 11.7 in two parts, more in more).
    const uint32_t tiles = (uint32_t)(((uint64_t)cols + TILE - 1) / TILE);
    const uint32_t most = std::min({tiles, MAX_PARTS, (uint32_t)ctx->sm_count / rows, MAX_SHARED / rows});
    const uint64_t bytes = (uint64_t)cols * (dtype == YX_F32 ? 4 : 2);
    a.parts = most > 1 && bytes - bytes / most > 144 * 1024 ? most : 1;
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
    // Rows are read while others' results are written.
    const size_t read = (((size_t)rows - 1) * stride + cols) * (dtype == YX_F32 ? 4 : 2);
    auto over = [&](const void *p, size_t each) {
        return p && (uintptr_t)p < (uintptr_t)logits_dev + read && (uintptr_t)logits_dev < (uintptr_t)p + (size_t)rows * each * 4;
    };
    if (over(logprob_dev, n_ids) || over(entropy_dev, 1) || over(top_ids_dev, n_top) || over(top_logprob_dev, n_top))
        return fail(ctx, YX_ERR_INVALID, "logprob_rows: a result lies over the logits");
    const struct {
        const void *p;
        size_t each;
    } results[] = {{logprob_dev, n_ids}, {entropy_dev, 1}, {top_ids_dev, n_top}, {top_logprob_dev, n_top}};
    for (int i = 0; i < 4; i++)
        for (int j = 0; j < i; j++)
            if (results[i].p && results[j].p && (uintptr_t)results[i].p < (uintptr_t)results[j].p + (size_t)rows * results[j].each * 4 &&
                (uintptr_t)results[j].p < (uintptr_t)results[i].p + (size_t)rows * results[i].each * 4)
                return fail(ctx, YX_ERR_INVALID, "logprob_rows: results lie over one another");
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
