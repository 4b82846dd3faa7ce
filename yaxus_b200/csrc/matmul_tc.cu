// out [T, N] f32 = x [T, K] f32 . w [N, K]^T (bf16) for passes of many rows, on the fifth-generation
// tensor cores, and the same with silu(gate) * up taken in the epilogue (crates/yaxus-model/src/lib.rs:128,164-168).
// Two more kinds of the kernels take their rows exactly and end in something else (yx_matmul_epilogue, yx_matmul_logprobs): see Kind.
//
// Activations keep 16 bits of mantissa: x = hi + lo, two bf16 matrices, and every weight tile that reaches
// shared memory is multiplied by both, into one f32 accumulator in tensor memory.  The arithmetic is twice
// that of a plain bf16 product; what a tile costs in weight traffic, accumulator reads and stores is not.
//
// The products are taken transposed, out^T = w x^T, by pairs of CTAs (cta_group::2): a tile is 256 weight
// rows (128 in each CTA) by up to 256 pass rows (half of them in each CTA), so a lane of tensor memory is a
// weight row, a warp's store of one pass row is one 128-byte line, and a pass of 33 rows fills the 256-row
// side as well as one of 2048 does.  A k step of 64 costs a CTA 16 KiB of weights and up to 32 KiB of
// activations for 2 x 256 x 256 x 64 multiply-adds: 32 bytes a clock and SM, half of what L2 delivers.
//
// Tiles are dealt to the pairs in whole rounds, pass rows fastest, so that the pairs that run together share
// weight rows and activations in L2.  What is left after the last whole round is cut along k into one equal
// share a pair (stream-K): such a share's sums go to scratch, and the CTA that comes last at a tile adds them
// up in order.  The shares come first in a pair's work, so that the adding up hides under whole tiles.  Adding up
// is a chain of L2 latencies: with one warp to a lane quarter and one share at a time it took 15 to 20 us.
//
// Large passes are bound by the tensor cores: 2048 rows on 4096 -> 28672 (gate and up) take 608 us, 1.58 PFLOP/s
// of bf16 products; 80 rows by the weights' way into shared memory: 235 MB in 64 us.  Against two
// library products (high part, then low part added to it) and a SwiGLU kernel, whole steps of one layer went from
// 2151 to 1509 us (2048 rows) and from 1244 to 358 us (80 rows).
//
// Warps 0-7 epilogue (two to each 32 lanes of tensor memory, taking turns at 32 pass rows), warp 8 TMA, warp 9
// issues the MMAs (first CTA of the pair).  All waits are bounded; on expiry the CTA records where, stops waiting
// anywhere, frees its tensor memory together with its partner and returns.
#include <cuda.h>

#include <algorithm>

#include "yx_epilogue.cuh"
#include "yx_tcgen05.cuh"

namespace yx {
namespace {

using namespace dev;

constexpr uint32_t TC_M = 256;              // weight rows of a pair's tile
constexpr uint32_t TC_KSTEP = 64;           // k of a stage: one 128-byte swizzled row
constexpr uint32_t TC_MAX_BT = 256;         // pass rows of a tile
constexpr int TC_MAX_STAGES = 12;
constexpr int TC_THREADS = 10 * 32;
constexpr int TC_TMA_WARP = 8, TC_MMA_WARP = 9;
constexpr uint32_t W_BYTES = 128 * 128;     // a CTA's share of a stage's weights
constexpr uint32_t TC_SMEM_BUDGET = 220 * 1024;
// k steps summed in tensor memory before the epilogue takes them over into its own f32 sums: the tensor core drops what
// lies below its accumulator's last place at each of a step's eight additions (see ROWS_CHAIN below).  Whole rounds of tiles of
// more than 128 rows and 32 k steps or more take chains of 16.  Error of the result against 64-bit products, 512 rows x
// [28672, 4096] with a GLU: one chain 1.9e-5, two library products 0.97e-5, chains of 16 0.64e-5; there, a piece begins with
// a longer chain where only two accumulators fit: it is what the tensor cores have to do while the epilogue stores the
// piece before (2048 rows x [28672, 4096]: 608 us, with chains of eight throughout 665, without chains 590).
// Everything else takes chains that lose no more than two library products would, whose accumulators take half the
// additions (one part each) and which cut k for small results: eight steps, half of the k steps where there are fewer than
// 16 of them, six where every tile is cut along k.  Errors with chains of 16, now, and the library's (2.44e-6 of each is
// the activations' two parts'): 275 rows x [34914, 1152] 3.19, 2.67 and 2.70e-6; 262 x [1460, 6784] 3.27, 2.60 and 2.60e-6;
// 558 x [41408, 1024] with a GLU 5.70, 4.22 and 4.09e-6.  Over 110 shapes of 33 to 900 rows at most 1.05 times the
// library's (1.39 before).  It costs 1 % in the mean, 6 % where it costs most (the last of these: 90 and 96 us); a step of
// 80 rows pays 19 us of 399 for chains of eight in place of 16.
constexpr uint32_t TC_CHAIN = 16, TC_FIRST_CHAIN = 32, TC_SHORT_CHAIN = 8, TC_CUT_CHAIN = 6, TC_LEAST_CHAIN = 4;
constexpr int TC_MAX_BUFS = 4;
constexpr uint32_t MAX_CLUSTER = 4;         // pairs of a cluster (eight CTAs: the most that any chip of this kind places)
// The same for rows taken exactly (EPILOGUE, LOGPROBS), by their parts: what keeps the result well within a millionth (2-norm
// of the error over the result's, 2048 x [14336, 4096]: one part in chains of 8, 12 and 16 steps 4.7, 7.1 and 9.9e-7 and in short runs 235, 225
// and 216 us, two of 4, 6 and 8 4.7, 7.2 and 10.1e-7 and 369, 356 and 348 us, three of 2, 3 and 4 3.4, 5.5 and 7.7e-7 and 547, 514 and 505 us; a library's
// f32 products 6 to 12e-7, yx_matmul 27e-7).  Results of 16 bits take chains that lose 4 to 7e-6: half a step of bf16 is 500
// times that.  2048 bf16 rows x [14336, 4096], call after call, in chains of 64 steps (a whole tile's), 32, 16 and 12: 206, 219, 249 and
// 256 us, and 0.23, 0.13, 0.07 and 0.05 % of the results are not the correctly rounded value but its neighbour (of a library's f32
// sums 0.04 %); the same of f16 rows and results, in chains of 48, 24, 12 and 6, 359, 366, 381 and 412 us and 2.2, 1.2, 0.7 and 0.35 % (0.41 %).
constexpr uint32_t EXACT_CHAIN[3] = {12, 6, 4}, NARROW_CHAIN[3] = {64, 48, 32};
constexpr uint32_t GLU_GROUP = 16;          // gate and up rows alternate in a tile sixteen by sixteen: a warp holds both

// What becomes of a product.
//  PLAIN, GLU: f32 rows in two bf16 parts (yx_matmul, yx_matmul_glu).
//  EPILOGUE: bias, activation and residual; LOGPROBS: softmax statistics of 128 columns at a time.  Both take the rows exactly, in
//  as many bf16 parts as their type has bits for: bf16 one, f16 (11 bits) two, f32 (24 bits) three.
enum Kind { PLAIN, GLU, EPILOGUE, LOGPROBS };
constexpr int kind_parts(int kind, int parts) { return kind < EPILOGUE ? 2 : parts; }

// Where the LOGPROBS kinds leave the statistics of a pass row t over 128 columns: [T][blocks] of (m, s, t, -), and the
// logit of the row's given token.
struct StatsOut {
    float4 *stats;
    uint32_t blocks;
    float *picked;          // [T]
};

struct PairArgs {
    uint32_t T, cols;                 // pass rows; columns of the result
    uint32_t parts;                   // bf16 parts of a pass row (EPILOGUE, LOGPROBS)
    uint32_t cluster;                 // pairs that share a tile as one cluster (EPILOGUE, LOGPROBS; 1: none)
    bool early_w;                     // what wrote the weights is complete when this kernel starts
    uint32_t bt, t_tiles;             // pass rows of a tile (multiple of 32), tiles of them
    uint32_t ksteps;
    uint32_t pairs;                   // CTA pairs of the grid
    uint32_t rounds;                  // whole rounds of tiles
    uint32_t rest_units, rest_pairs;  // k steps of the tiles after them, and the pairs that share those
    uint32_t stages;
    uint32_t bufs, buf_columns;       // accumulators in tensor memory
    uint32_t chain, long_first;       // k steps summed in one of them; whether a piece begins with more
    float *out;
    Epilogue e;                       // EPILOGUE (`out` is of its type)
    StatsOut so;                      // LOGPROBS
    const uint32_t *ids;              // LOGPROBS: given tokens [T]
    float *part;                      // [2 * rest_pairs shares][2 CTAs][bt][128]
    uint32_t *counters;               // [tiles left over][2 CTAs], zero between launches
    yx_dev_status *status;
};

// One stretch of k steps of one tile.
struct Piece {
    uint32_t tile, k0, k1;
    bool whole;
};

__device__ __forceinline__ uint32_t rest_begin(const PairArgs &a, uint32_t p) { return (uint32_t)((uint64_t)p * a.rest_units / a.rest_pairs); }
// The pair whose share holds unit u.
__device__ __forceinline__ uint32_t rest_owner(const PairArgs &a, uint32_t u) {
    return (uint32_t)((((uint64_t)u + 1) * a.rest_pairs - 1) / a.rest_units);
}

// Walks a pair's pieces: its share of the left-over tiles (at most two pieces), then its whole tiles.  In a cluster of several
// pairs there is one piece: the pair's share of the cluster's tile.
struct Walk {
    uint32_t u, u_end, round;
    __device__ __forceinline__ Walk(const PairArgs &a, uint32_t pair) : u(0), u_end(0), round(0) {
        if (a.cluster > 1) {
            const uint32_t tile = pair / a.cluster, at = pair - tile * a.cluster;
            u = tile * a.ksteps + at * a.ksteps / a.cluster;
            u_end = tile * a.ksteps + (at + 1) * a.ksteps / a.cluster;
        } else if (pair < a.rest_pairs) {
            u = rest_begin(a, pair);
            u_end = rest_begin(a, pair + 1);
        }
    }
    __device__ __forceinline__ bool next(const PairArgs &a, uint32_t pair, Piece &p) {
        if (u < u_end) {
            const uint32_t tile = u / a.ksteps;
            p.k0 = u - tile * a.ksteps;
            p.k1 = min(a.ksteps, p.k0 + (u_end - u));
            u += p.k1 - p.k0;
            p.tile = a.rounds * a.pairs + tile;
            p.whole = p.k1 - p.k0 == a.ksteps;
            return true;
        }
        if (round >= a.rounds) return false;
        p = Piece{round * a.pairs + pair, 0, a.ksteps, true};
        round++;
        return true;
    }
};

// Where the chain of k steps that begins at k ends.
__device__ __forceinline__ uint32_t chain_end(const PairArgs &a, const Piece &p, uint32_t k) {
    const uint32_t n = k == p.k0 && a.long_first ? min(TC_FIRST_CHAIN, max(a.chain, (p.k1 - p.k0) * 3 / 8)) : a.chain;
    return min(p.k1, k + n);
}
// Accumulators in turn, and the parity of the current round of them.
struct AccTurn {
    uint32_t buf = 0, round = 0;
    __device__ __forceinline__ void next(uint32_t bufs) {
        if (++buf == bufs) {
            buf = 0;
            round++;
        }
    }
};

__device__ __forceinline__ uint32_t mapa(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ float4 load_cluster(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
}

// ---- a warp's 32 columns by N pass rows change places -----------------------------------------------------
//
// A lane holds a column.  What follows a product wants a pass row's columns side by side: through shared memory, a pass row's
// 128 bytes in 16-byte chunks at chunk ^ (row & 7), which meets no bank twice either way.
template <int N, int V>
__device__ __forceinline__ void stage(const float (&v)[V], int first, float *staged, int lane) {
    __syncwarp();
#pragma unroll
    for (int i = 0; i < N; i++) staged[i * 32 + (((lane >> 2) ^ (i & 7)) << 2) + (lane & 3)] = v[first + i];
    __syncwarp();
}
__device__ __forceinline__ uint32_t staged_at(uint32_t row, uint32_t column) { return row * 32 + (((column >> 2) ^ (row & 7)) << 2) + (column & 3); }

// Bias, activation and residual of N staged pass rows, t0 and on, by the 32 columns from col0, as far as `end`.  All residuals are asked
// for before the first is used, and what follows is a loop, whose registers move up: unrolled over a thread's up to 128 results
// the code does not fit the instruction cache, and out of line every sum still in a register goes through local memory
// (2048 x [14336, 4096] bf16: 220 us plain, 386 onto a residual with a type looked up for each; out of line 296 and 392).
template <int N>
__device__ __forceinline__ void finish_staged(const Epilogue &e, void *out, uint32_t T, uint32_t cols, uint32_t end, const float *staged, uint32_t t0, uint32_t col0, int lane) {
    if (t0 >= T) return;
    const uint32_t rows = min((uint32_t)N, T - t0);
    constexpr int R = N / 4;
    const float4 zero = make_float4(0.f, 0.f, 0.f, 0.f);
    float4 res[R];
    auto ask = [&](auto load) {   // load(type, i): the residuals of turn i
        if (!e.residual) {
#pragma unroll
            for (int i = 0; i < R; i++) res[i] = zero;
        } else if (e.out_dtype == YX_F32) {
#pragma unroll
            for (int i = 0; i < R; i++) res[i] = load(YX_F32, i);
        } else if (e.out_dtype == YX_F16) {
#pragma unroll
            for (int i = 0; i < R; i++) res[i] = load(YX_F16, i);
        } else {
#pragma unroll
            for (int i = 0; i < R; i++) res[i] = load(YX_BF16, i);
        }
    };
    auto next = [&](float4 y) {
        y = activate4(y, e.act);
        if (e.residual) y = make_float4(y.x + res[0].x, y.y + res[0].y, y.z + res[0].z, y.w + res[0].w);
#pragma unroll
        for (int i = 0; i + 1 < R; i++) res[i] = res[i + 1];
        return y;
    };
    if (e.quads) {
        // A turn: four columns a lane, four pass rows a warp.
        const uint32_t q = 4 * (lane & 7), col = col0 + q, r0 = lane >> 3;
        if (col >= end) return;
        size_t at = (size_t)(t0 + r0) * cols + col;
        const float4 bias = e.bias ? *(const float4 *)(e.bias + col) : zero;
        ask([&](int dtype, int i) { return r0 + 4 * i < rows ? load4_as_f32(e.residual, dtype, at + (size_t)(4 * i) * cols) : zero; });
#pragma unroll 1
        for (uint32_t r = r0; r < rows; r += 4, at += (size_t)4 * cols) {
            const float4 y = *(const float4 *)(staged + staged_at(r, q));
            store4(out, e.out_dtype, at, next(make_float4(y.x + bias.x, y.y + bias.y, y.z + bias.z, y.w + bias.w)));
        }
    } else {
        // A turn: a column a lane, four pass rows.
        const uint32_t col = col0 + lane;
        if (col >= end) return;
        size_t at = (size_t)t0 * cols + col;
        const float bias = e.bias ? e.bias[col] : 0.0f;
        ask([&](int dtype, int i) {
            float v[4];
#pragma unroll
            for (int k = 0; k < 4; k++) v[k] = 4 * i + k < (int)rows ? load_as_f32(e.residual, dtype, at + (size_t)(4 * i + k) * cols) : 0.0f;
            return make_float4(v[0], v[1], v[2], v[3]);
        });
#pragma unroll 1
        for (uint32_t r = 0; r < rows; r += 4) {
            const float4 y = next(make_float4(staged[staged_at(r, lane)] + bias, staged[staged_at(r + 1, lane)] + bias, staged[staged_at(r + 2, lane)] + bias,
                                              staged[staged_at(r + 3, lane)] + bias));
            const float z[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
            for (int k = 0; k < 4; k++, at += cols)
                if (r + k < rows) store_from_f32(out, e.out_dtype, at, z[k]);
        }
    }
}

// ---- softmax statistics of a warp's 32 columns for each of its pass rows --------------------------------
//
// Sixteen pass rows at a time change places with the columns, after which a lane has half a pass row's: 1.25
// shared-memory accesses for a logit's six or so instructions, where summing across lanes would take three shuffles.
constexpr int STATS_SCRATCH = 16 * 32;   // floats a warp

// Statistics of pass rows 0..15 of v over this warp's 32 columns, in lanes r and r + 16 for row r.  `want`: the row's given
// token, counted from the warp's first column (past 31: not here); `logit`: set to its logit.
template <int N>
__device__ __forceinline__ RowStats stats_of_16(const float (&v)[N], int first, bool column, float *scratch, int lane, uint32_t want, float &logit) {
    __syncwarp();
#pragma unroll
    for (int i = 0; i < (N < 16 ? N : 16); i++) scratch[staged_at(i, lane)] = column ? v[first + i] : -INFINITY;
    __syncwarp();
    const int r = lane & 15;
    float q[16];
#pragma unroll
    for (int c = 0; c < 4; c++) *(float4 *)(q + 4 * c) = *(const float4 *)(scratch + staged_at(r, ((lane >> 4) * 4 + c) * 4));
    if (want < 32u) logit = scratch[staged_at(r, want)];
    float m = q[0];
#pragma unroll
    for (int i = 1; i < 16; i++) m = fmaxf(m, q[i]);
    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
    if (!(m < INFINITY)) {   // an infinity (or nothing but no numbers)
#pragma unroll
        for (int i = 0; i < 16; i++) q[i] = clean(q[i]);
        m = clean(m);
    }
    F2 s2 = f2(0.0f, 0.0f), t2 = s2;
    add_up(q, m, s2, t2);
    float s, t, s1, t1;
    split(s2, s, s1);
    split(t2, t, t1);
    s += s1;
    t += t1;
    return RowStats{m, s + __shfl_xor_sync(0xffffffffu, s, 16), t + __shfl_xor_sync(0xffffffffu, t, 16)};
}

// Of N pass rows from t0 on: this warp's 32 columns as far as `end`, lane i row t0 + i, and the given tokens' logits where they are among them.
template <int N>
__device__ __forceinline__ float4 stats_of(const StatsOut &so, uint32_t T, uint32_t end, const float (&v)[N], uint32_t t0, uint32_t row, const uint32_t *ids,
                                           float *scratch, int lane) {
    const uint32_t t = t0 + lane;
    const uint32_t id = lane < N && t < T ? ids[t] : 0xffffffffu, want = id < end ? id - (row - lane) : 0xffffffffu;
    float logit = 0.0f;
    RowStats st = stats_of_16(v, 0, row < end, scratch, lane, lane < 16 ? want : 0xffffffffu, logit);
    if constexpr (N > 16) {
        const RowStats hi = stats_of_16(v, 16, row < end, scratch, lane, lane < 16 ? 0xffffffffu : want, logit);
        if (lane >= 16) st = hi;
    }
    if (want < 32u) so.picked[t] = logit;
    return make_float4(st.m, st.s, st.t, 0.0f);
}
// Four warps' statistics of the same pass rows as one.
__device__ __forceinline__ float4 merge_four(const float4 (&f)[4]) {
    const float m = fmaxf(fmaxf(f[0].x, f[1].x), fmaxf(f[2].x, f[3].x));
    float s = 0.0f, t = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float d = distance(f[i].x, m), c = fast_exp2(d * LOG2_E);
        s += c * f[i].y;
        t += c * (f[i].z + d * f[i].y);
    }
    return make_float4(m, s, t, 0.0f);
}

// 32 pass rows from `t0` on of this lane's weight row.
template <bool GLU>
__device__ __forceinline__ void store_rows(const PairArgs &a, const float (&v)[32], uint32_t t0, uint32_t row, int lane) {
    if constexpr (!GLU) {
        if (row >= a.cols) return;
        float *dst = a.out + (size_t)t0 * a.cols + row;
        if (t0 + 32 <= a.T) {
#pragma unroll
            for (int i = 0; i < 32; i++) dst[(size_t)i * a.cols] = v[i];
        } else {
#pragma unroll
            for (int i = 0; i < 32; i++)
                if (t0 + i < a.T) dst[(size_t)i * a.cols] = v[i];
        }
    } else {
        // Lanes 0-15 hold gate rows, lanes 16-31 the same rows' up: the lower half finishes the first sixteen
        // pass rows, the upper half the others.  `row` counts both kinds, so its 32 are 16 columns.
        const uint32_t col = (row >> 5) * GLU_GROUP + (lane & 15), t = t0 + (lane & 16);
        float *dst = a.out + (size_t)t * a.cols + col;
#pragma unroll
        for (int i = 0; i < 16; i++) {
            const float other = __shfl_xor_sync(0xffffffffu, lane < 16 ? v[16 + i] : v[i], 16);
            const float g = lane < 16 ? v[i] : other, u = lane < 16 ? other : v[16 + i];
            if (col < a.cols && t + i < a.T) dst[(size_t)i * a.cols] = g / (1.0f + expf(-g)) * u;
        }
    }
}

// CHUNKS: 64-row chunks of a tile, what an epilogue thread keeps in registers (two for up to
// 128 pass rows, three for up to 192: before the chains of eight above, steps of 80 and of 311 rows took 391 and 453 us with
// room for four, 382 and 437 so; with them 399 and 440).
template <int KIND, int CHUNKS>
__device__ __forceinline__ void pair_body(const CUtensorMap &w_map, const CUtensorMap &x_map, const PairArgs &a) {
    extern __shared__ __align__(1024) unsigned char smem[];
    __shared__ __align__(8) uint64_t bar_store[2 * TC_MAX_STAGES + 2 * TC_MAX_BUFS];
    __shared__ uint32_t tmem_base_s;
    __shared__ int abort_flag;
    __shared__ int last_s;
    constexpr int SCRATCH = KIND == EPILOGUE ? 32 * 32 : KIND == LOGPROBS ? STATS_SCRATCH : 1;   // floats a warp
    __shared__ __align__(16) float scratch_s[8 * SCRATCH];
    float *scratch = scratch_s + ((threadIdx.x >> 5) & 7) * SCRATCH;
    __shared__ float4 stats_s[KIND == LOGPROBS ? CHUNKS : 1][8][KIND == LOGPROBS ? 32 : 1];   // of a tile, by chunks and warps
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const uint32_t rank = blockIdx.x & 1u, pair = blockIdx.x >> 1;
    const uint32_t first = KIND < EPILOGUE ? 0u : cluster_rank() & ~1u;   // the pair's first CTA
    const uint32_t parts = KIND < EPILOGUE ? 2u : a.parts;
    const uint32_t S = a.stages, x_bytes = parts * a.bt * 64u, stage_bytes = W_BYTES + x_bytes;   // x: bt / 2 rows, the high part first
    const uint32_t base = smem_u32(smem);
    const uint32_t b_full = smem_u32(bar_store), b_empty = b_full + 8 * TC_MAX_STAGES;
    const uint32_t b_acc_full = b_empty + 8 * TC_MAX_STAGES, b_acc_empty = b_acc_full + 8 * TC_MAX_BUFS;
    volatile int *abortp = &abort_flag;

    if (threadIdx.x == 0) {
        abort_flag = 0;
        for (uint32_t s = 0; s < S; s++) {
            mbar_init(b_full + 8 * s, 1);
            mbar_init(b_empty + 8 * s, 1);
        }
        for (int b = 0; b < TC_MAX_BUFS; b++) {
            mbar_init(b_acc_full + 8 * b, 1);
            mbar_init(b_acc_empty + 8 * b, 16);   // a warp's arrival each, from both CTAs
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == TC_TMA_WARP && elect()) {
        prefetch_tensormap(&w_map);
        prefetch_tensormap(&x_map);
    }
    if (warp == TC_MMA_WARP) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base_s)), "n"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync();
    tc_fence_after();
    const uint32_t tmem = tmem_base_s;

    if (warp == TC_TMA_WARP) {
        if (elect()) {
            // ---- producer -------------------------------------------------------------------------
            // One thread issues every copy: nothing is computed in the loops that does not change there, and the thread is
            // elected (see elect).  80 rows bf16 x [14336, 4096]: 34.7 us, without the divisions and the flag 31.8, elected 28.4.
            const uint32_t full0 = mapa(b_full, first);   // the first CTA's barriers count both CTAs' bytes
            struct Place {
                int row, group, x;   // weight row (PLAIN) or group of them (GLU), pass row
            };
            auto place = [&](const Piece &p) {
                const uint32_t at = p.tile / a.t_tiles, m0 = at * TC_M + rank * 128u;
                return Place{KIND == GLU ? 0 : (int)m0, KIND == GLU ? (int)(m0 / (2 * GLU_GROUP)) : 0, (int)((p.tile - at * a.t_tiles) * a.bt + rank * (a.bt / 2))};
            };
            auto load_w = [&](uint32_t s, const Place &at, uint32_t k) {
                if (rank == 0) mbar_expect_tx(b_full + 8 * s, 2 * stage_bytes);
                tma_load_4d_pair(base + s * stage_bytes, &w_map, (int)(k * TC_KSTEP), at.row, 0, at.group, full0 + 8 * s);
            };
            auto load_x = [&](uint32_t s, const Place &at, uint32_t k) {
                tma_load_3d_pair(base + s * stage_bytes + W_BYTES, &x_map, (int)(k * TC_KSTEP), at.x, 0, full0 + 8 * s);
            };
            // The kernel ahead (the split of the activations) let this one start only after its own wait, so nothing
            // that may still run writes the weights: the ring's first weights are on their way before the wait.  (Rows that are
            // bf16 already have no split ahead of them.)
            uint32_t ahead = 0;
            if (KIND < EPILOGUE || a.early_w) {
                Walk walk(a, pair);
                Piece p;
                while (ahead < S && walk.next(a, pair, p)) {
                    const Place at = place(p);
                    for (uint32_t k = p.k0; k < p.k1 && ahead < S; k++) load_w(ahead++, at, k);
                }
            }
            asm volatile("griddepcontrol.wait;" ::: "memory");
            asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
            Walk walk(a, pair);
            Piece p;
            uint32_t it = 0, s = 0, phase = 0;
            bool gone = false;
            while (!gone && walk.next(a, pair, p)) {
                const Place at = place(p);
                for (uint32_t k = p.k0; k < p.k1; k++, it++) {
                    if (it >= ahead) {
                        if (!mbar_try(b_empty + 8 * s, phase ^ 1u)) {
                            mbar_wait_slow(b_empty + 8 * s, phase ^ 1u, abortp, a.status, 501);
                            gone = *abortp;
                            if (gone) break;
                        }
                        load_w(s, at, k);
                    }
                    load_x(s, at, k);
                    if (++s == S) {
                        s = 0;
                        phase ^= 1u;
                    }
                }
            }
        }
    } else if (warp == TC_MMA_WARP) {
        if (rank == 0 && elect()) {
            // ---- MMA issuer -----------------------------------------------------------------------
            const uint32_t idesc = f16_instr_desc(true, false, TC_M, a.bt);
            Walk walk(a, pair);
            Piece p;
            uint32_t s = 0, phase = 0;
            AccTurn turn;
            while (!*abortp && walk.next(a, pair, p)) {
                for (uint32_t k0 = p.k0; k0 < p.k1 && !*abortp; turn.next(a.bufs)) {
                    const uint32_t acc = tmem + turn.buf * a.buf_columns, k_end = chain_end(a, p, k0);
                    if (turn.round > 0) mbar_wait(b_acc_empty + 8 * turn.buf, (turn.round - 1) & 1u, abortp, a.status, 502);
                    tc_fence_after();
                    for (uint32_t k = k0; k < k_end; k++) {
                        if (!mbar_try(b_full + 8 * s, phase)) {
                            mbar_wait_slow(b_full + 8 * s, phase, abortp, a.status, 503);
                            if (*abortp) break;
                        }
                        tc_fence_after();
                        const uint32_t w_lo = desc_lo(base + s * stage_bytes, 0), h_lo = w_lo + W_BYTES / 16;
                        if constexpr (KIND < EPILOGUE) {
#pragma unroll
                            for (uint32_t kk = 0; kk < 4; kk++) umma2_ss_lo(acc, w_lo + 2 * kk, h_lo + 2 * kk, idesc, k > k0 || kk > 0);
#pragma unroll
                            for (uint32_t kk = 0; kk < 4; kk++) umma2_ss_lo(acc, w_lo + 2 * kk, h_lo + a.bt * 4u + 2 * kk, idesc, 1);
                        } else {
                            // The smallest part first: in a chain's first step the large sum is not there yet to drop its bits.
                            for (uint32_t part = parts; part-- > 0;) {
                                const uint32_t x_lo = h_lo + part * (a.bt * 4u);
                                const bool fresh = k == k0 && part == parts - 1;
#pragma unroll
                                for (uint32_t kk = 0; kk < 4; kk++) umma2_ss_lo(acc, w_lo + 2 * kk, x_lo + 2 * kk, idesc, !fresh || kk > 0);
                            }
                        }
                        umma2_commit(b_empty + 8 * s, first);
                        if (++s == S) {
                            s = 0;
                            phase ^= 1u;
                        }
                    }
                    umma2_commit(b_acc_full + 8 * turn.buf, first);
                    k0 = k_end;
                }
            }
        }
    } else if (warp < 8) {
        // ---- epilogue -------------------------------------------------------------------------
        // (it reads what the kernels ahead wrote, residuals and given tokens, with loads of its own)
        if constexpr (KIND >= EPILOGUE) asm volatile("griddepcontrol.wait;" ::: "memory");
        Walk walk(a, pair);
        Piece p;
        AccTurn turn;
        auto finish = [&](const auto &v, uint32_t t, uint32_t row, uint32_t chunk) {
            constexpr int N = sizeof(v) / sizeof(float);
            if constexpr (KIND < EPILOGUE) store_rows<KIND == GLU>(a, v, t, row, lane);
            else if constexpr (KIND == EPILOGUE) {
                stage<N>(v, 0, scratch, lane);
                finish_staged<N>(a.e, a.out, a.T, a.cols, a.cols, scratch, t, row - lane, lane);
            } else {
                stats_s[chunk][warp][lane] = stats_of(a.so, a.T, a.cols, v, t, row, a.ids, scratch, lane);
            }
        };
        // A tile's statistics: the four warps of the same pass rows each take a chunk of them.
        auto finish_stats = [&](uint32_t t0, uint32_t c0, uint32_t row) {
            asm volatile("bar.sync %0, 128;" ::"r"(2 + (warp >> 2)) : "memory");
            const uint32_t chunk = warp & 3, t = t0 + c0 + 64 * chunk + lane;
            if (chunk < CHUNKS && c0 + 64 * chunk < a.bt && t < a.T) {
                const int g = warp & 4;
                const float4 four[4] = {stats_s[chunk][g][lane], stats_s[chunk][g + 1][lane], stats_s[chunk][g + 2][lane], stats_s[chunk][g + 3][lane]};
                a.so.stats[(size_t)t * a.so.blocks + (row >> 7)] = merge_four(four);
            }
            asm volatile("bar.sync %0, 128;" ::"r"(2 + (warp >> 2)) : "memory");
        };
        while (walk.next(a, pair, p)) {
            const uint32_t wr = (warp & 3) * 32 + lane;   // weight row of this CTA's 128
            const uint32_t row = (p.tile / a.t_tiles) * TC_M + rank * 128u + wr, t0 = (p.tile % a.t_tiles) * a.bt;
            const uint32_t rest = p.whole ? 0u : p.tile - a.rounds * a.pairs;
            // The pairs that share left-over tile `rest`, found while it is being summed.  Only the first of them may
            // have begun in the tile before it, which makes this tile its second piece.
            uint32_t q0 = 0, q1 = 0, second = 0;
            if (!p.whole && (KIND < EPILOGUE || a.cluster == 1)) {
                q0 = rest_owner(a, rest * a.ksteps);
                q1 = rest_owner(a, (rest + 1) * a.ksteps - 1);
                second = rest - rest_begin(a, q0) / a.ksteps;
            }
            // This thread's sums: its weight row, 32 pass rows out of every 64.
            const uint32_t c0 = 32u * (warp >> 2);
            float sum[CHUNKS][32];
#pragma unroll
            for (int j = 0; j < CHUNKS; j++)
#pragma unroll
                for (int i = 0; i < 32; i++) sum[j][i] = 0.0f;
            for (uint32_t k = p.k0; k < p.k1; k = chain_end(a, p, k), turn.next(a.bufs)) {
                const uint32_t acc = tmem + turn.buf * a.buf_columns + ((uint32_t)(warp & 3) << 21);
                mbar_wait(b_acc_full + 8 * turn.buf, turn.round & 1u, abortp, a.status, 504);
                __syncwarp();   // (after a wait that ran out the warps go on, on whatever is there: their barriers below count all of them)
                tc_fence_after();
#pragma unroll
                for (int j = 0; j < CHUNKS; j++) {
                    if (c0 + 64 * j >= a.bt) break;
#pragma unroll
                    for (int h = 0; h < 32; h += 16) {   // (sixteen at a time: 32 more registers would spill)
                        uint32_t r[16];
                        tmem_ld16(acc + c0 + 64 * j + h, r);
                        tmem_ld_wait();
#pragma unroll
                        for (int i = 0; i < 16; i++) sum[j][h + i] += __uint_as_float(r[i]);
                    }
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0)
                    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(mapa(b_acc_empty + 8 * turn.buf, first)) : "memory");
            }
            // A share's sums: four pass rows of each of 128 weight rows, then the next four.
            auto share = [&](uint32_t q) { return (float4 *)(a.part + ((size_t)(2 * q + (q == q0 ? second : 0u)) * 2 + rank) * a.bt * 128u) + wr; };
            // What follows the sums is written once and gone through chunk by chunk, the next chunk's sums moving up.
            auto finish_all = [&] {
#pragma unroll 1
                for (uint32_t c = c0, chunk = 0; c < a.bt; c += 64, chunk++) {
                    finish(sum[0], t0 + c, row, chunk);
#pragma unroll
                    for (int j = 0; j + 1 < CHUNKS; j++)
#pragma unroll
                        for (int i = 0; i < 32; i++) sum[j][i] = sum[j + 1][i];
                }
            };
            if constexpr (KIND >= EPILOGUE) {
                if (a.cluster > 1) {
                    // The pairs' sums stay in their shared memory, which no copy and no product needs any more.
#pragma unroll
                    for (int j = 0; j < CHUNKS; j++) {
                        const uint32_t c = c0 + 64 * j;
                        if (c >= a.bt) break;
#pragma unroll
                        for (int i = 0; i < 8; i++)
                            *(float4 *)(smem + ((c / 4 + i) * 128u + wr) * 16u) = make_float4(sum[j][4 * i], sum[j][4 * i + 1], sum[j][4 * i + 2], sum[j][4 * i + 3]);
                    }
                    break;
                }
            }
            if (KIND >= EPILOGUE && p.whole) {
                finish_all();
                if constexpr (KIND == LOGPROBS) finish_stats(t0, c0, row);
                continue;
            }
#pragma unroll
            for (int j = 0; j < CHUNKS; j++) {
                const uint32_t c = c0 + 64 * j;
                if (c >= a.bt) break;
                if (p.whole) {
                    if constexpr (KIND < EPILOGUE) finish(sum[j], t0 + c, row, 0);
                } else {
                    float4 *mine = share(pair) + c / 4 * 128u;
#pragma unroll
                    for (int i = 0; i < 8; i++) __stcg(mine + i * 128, make_float4(sum[j][4 * i], sum[j][4 * i + 1], sum[j][4 * i + 2], sum[j][4 * i + 3]));
                }
            }
            if (p.whole) continue;
            // The last of the tile's shares to arrive adds all of them up, in the order of k.
            __threadfence();
            asm volatile("bar.sync 1, 256;" ::: "memory");
            if (threadIdx.x == 0) {
                uint32_t *counter = a.counters + 2 * rest + rank;
                const int last = atomicAdd(counter, 1u) == q1 - q0;
                if (last) *counter = 0u;
                last_s = last;
            }
            asm volatile("bar.sync 1, 256;" ::: "memory");
            const bool last = last_s != 0;
            if (!last) continue;
            __threadfence();
            // (a chain of L2 latencies: six shares' sums are asked for at once)
            for (uint32_t c = 32u * (warp >> 2); c < a.bt && t0 + c < a.T; c += 64) {
                alignas(16) float v[32];
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    float4 sum[4] = {};
                    for (uint32_t q = q0; q <= q1; q += 6) {
                        float4 w[6][4];
#pragma unroll
                        for (int b = 0; b < 6; b++) {
                            const float4 *src = share(min(q + b, q1)) + (c / 4 + 4 * h) * 128u;
#pragma unroll
                            for (int i = 0; i < 4; i++) w[b][i] = q + b <= q1 ? __ldcg(src + i * 128) : make_float4(0.f, 0.f, 0.f, 0.f);
                        }
#pragma unroll
                        for (int b = 0; b < 6; b++)
#pragma unroll
                            for (int i = 0; i < 4; i++) {
                                sum[i].x += w[b][i].x;
                                sum[i].y += w[b][i].y;
                                sum[i].z += w[b][i].z;
                                sum[i].w += w[b][i].w;
                            }
                    }
#pragma unroll
                    for (int i = 0; i < 4; i++) *(float4 *)(v + 16 * h + 4 * i) = sum[i];
                }
                finish(v, t0 + c, row, c / 64);
            }
            if constexpr (KIND == LOGPROBS) finish_stats(t0, 32u * (warp >> 2), row);
        }
    }
    __syncwarp();
    if constexpr (KIND >= EPILOGUE) {
        if (a.cluster > 1) {
            // Sixteen pass rows at a time are added up, in the order of k, and finished by one pair of the cluster.
            cluster_sync();
            const uint32_t tile = pair / a.cluster, at = pair - tile * a.cluster, wr = (warp & 3) * 32 + lane;
            const uint32_t row = (tile / a.t_tiles) * TC_M + rank * 128u + wr, t0 = (tile % a.t_tiles) * a.bt;
            for (uint32_t c = 16 * (at + a.cluster * (warp >> 2)); warp < 8 && c < a.bt && t0 + c < a.T; c += 32 * a.cluster) {
                float4 f[MAX_CLUSTER][4];   // (all on their way at once)
#pragma unroll
                for (uint32_t q = 0; q < MAX_CLUSTER; q++) {
                    const uint32_t from = mapa(base + (c / 4 * 128u + wr) * 16u, 2 * min(q, a.cluster - 1) + rank);
#pragma unroll
                    for (int i = 0; i < 4; i++) f[q][i] = load_cluster(from + i * 128u * 16u);
                }
                float v[16];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    float4 sum = f[0][i];
#pragma unroll
                    for (uint32_t q = 1; q < MAX_CLUSTER; q++)
                        if (q < a.cluster) sum = make_float4(sum.x + f[q][i].x, sum.y + f[q][i].y, sum.z + f[q][i].z, sum.w + f[q][i].w);
                    v[4 * i] = sum.x;
                    v[4 * i + 1] = sum.y;
                    v[4 * i + 2] = sum.z;
                    v[4 * i + 3] = sum.w;
                }
                if constexpr (KIND == EPILOGUE) {
                    stage<16>(v, 0, scratch, lane);
                    finish_staged<16>(a.e, a.out, a.T, a.cols, a.cols, scratch, t0 + c, row - lane, lane);
                } else {
                    stats_s[0][warp][lane] = stats_of(a.so, a.T, a.cols, v, t0 + c, row, a.ids, scratch, lane);
                    asm volatile("bar.sync %0, 128;" ::"r"(2 + (warp >> 2)) : "memory");
                    const uint32_t t = t0 + c + lane;
                    if ((warp & 3) == 0 && lane < 16 && t < a.T) {
                        const float4 four[4] = {stats_s[0][warp][lane], stats_s[0][warp + 1][lane], stats_s[0][warp + 2][lane], stats_s[0][warp + 3][lane]};
                        a.so.stats[(size_t)t * a.so.blocks + (row >> 7)] = merge_four(four);
                    }
                    asm volatile("bar.sync %0, 128;" ::"r"(2 + (warp >> 2)) : "memory");
                }
            }
            __syncwarp();
        }
    }
    if (*abortp)
        for (int i = 0; i < 64; i++) __nanosleep(1000);   // copies and products in flight come to rest
    tc_fence_before();
    __syncthreads();
    cluster_sync();   // the partner's copies and completions still land in this CTA, and its sums are read there
    tc_fence_after();
    if (warp == TC_MMA_WARP) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(512) : "memory");
}

template <int KIND, int CHUNKS>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(TC_THREADS, 1)
matmul_pair_kernel(const __grid_constant__ CUtensorMap w_map, const __grid_constant__ CUtensorMap x_map, const __grid_constant__ PairArgs a) {
    pair_body<KIND, CHUNKS>(w_map, x_map, a);
}
// (EPILOGUE and LOGPROBS: clusters of one to MAX_CLUSTER pairs)
template <int KIND, int CHUNKS>
__global__ void __launch_bounds__(TC_THREADS, 1)
matmul_exact_kernel(const __grid_constant__ CUtensorMap w_map, const __grid_constant__ CUtensorMap x_map, const __grid_constant__ PairArgs a) {
    pair_body<KIND, CHUNKS>(w_map, x_map, a);
}

// x [n] f32 -> its high and its low bf16 part, x = hi + lo to 16 bits of mantissa; eight elements a thread.
template <bool VEC16>
__global__ void __launch_bounds__(256) split_rows_kernel(const float *__restrict__ x, size_t n, uint4 *__restrict__ hi, uint4 *__restrict__ lo) {
    dependent_entry();
    const size_t idx = (size_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (idx * 8 >= n) return;
    float v[8];
    if constexpr (VEC16) {
        *(float4 *)v = *(const float4 *)(x + idx * 8);
        *(float4 *)(v + 4) = *(const float4 *)(x + idx * 8 + 4);
    } else {
#pragma unroll
        for (int j = 0; j < 4; j++) *(float2 *)(v + 2 * j) = *(const float2 *)(x + idx * 8 + 2 * j);
    }
    uint32_t h[4], l[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
        h[j] = pack2<true>(v[2 * j], v[2 * j + 1]);
        const float2 b = unpack2<true>(h[j]);
        l[j] = pack2<true>(v[2 * j] - b.x, v[2 * j + 1] - b.y);
    }
    hi[idx] = make_uint4(h[0], h[1], h[2], h[3]);
    lo[idx] = make_uint4(l[0], l[1], l[2], l[3]);
}

// The bf16 parts of eight f32 or f16 values, largest first, cut off and not rounded: each part takes the next eight bits, so
// that PARTS of them are the value itself, and a value above the largest bf16 stays finite.
template <int PARTS>
__device__ __forceinline__ void cut_parts(const float (&v)[8], uint32_t (&out)[PARTS][4]) {
#pragma unroll
    for (int j = 0; j < 4; j++) {
        float a = v[2 * j], b = v[2 * j + 1];
#pragma unroll
        for (int p = 0; p < PARTS; p++) {
            const uint32_t ha = __float_as_uint(a) & 0xffff0000u, hb = __float_as_uint(b) & 0xffff0000u;
            out[p][j] = ha >> 16 | hb;
            a -= __uint_as_float(ha);
            b -= __uint_as_float(hb);
        }
        // What is no number, or infinite, is so in its first part alone (the bits cut off might be all that told the two
        // apart, and infinity less itself is no number).
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const uint32_t x = __float_as_uint(v[2 * j + i]), shift = 16 * i;
            if ((x & 0x7f800000u) != 0x7f800000u) continue;
            const uint32_t first = (x & 0x7fffffu ? 0x7fc0u : x >> 16) << shift;
            out[0][j] = (out[0][j] & ~(0xffffu << shift)) | first;
#pragma unroll
            for (int p = 1; p < PARTS; p++) out[p][j] &= ~(0xffffu << shift);
        }
    }
}
// Eight consecutive elements, at an address of 16 bytes' alignment where VEC says so, as f32.
template <int DTYPE, bool VEC>
__device__ __forceinline__ void load8(const void *base, size_t at, float (&v)[8]) {
    if constexpr (!VEC) {
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = load_as_f32(base, DTYPE, at + j);
    } else if constexpr (DTYPE == YX_F32) {
        *(float4 *)v = *(const float4 *)((const float *)base + at);
        *(float4 *)(v + 4) = *(const float4 *)((const float *)base + at + 4);
    } else {
        const uint4 u = *(const uint4 *)((const uint16_t *)base + at);
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const float2 f = unpack2<DTYPE == YX_BF16>(w[j]);
            v[2 * j] = f.x;
            v[2 * j + 1] = f.y;
        }
    }
}
// x [n] -> its PARTS bf16 parts, [PARTS][n]; eight elements a thread (n is a multiple of eight).
template <int DTYPE, int PARTS, bool VEC>
__global__ void __launch_bounds__(256) cut_rows_kernel(const void *__restrict__ x, size_t n, uint4 *__restrict__ out) {
    dependent_entry();
    const size_t idx = (size_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (idx * 8 >= n) return;
    float v[8];
    load8<DTYPE, VEC>(x, idx * 8, v);
    uint32_t parts[PARTS][4];
    cut_parts<PARTS>(v, parts);
#pragma unroll
    for (int p = 0; p < PARTS; p++) out[p * (n / 8) + idx] = make_uint4(parts[p][0], parts[p][1], parts[p][2], parts[p][3]);
}

// ---- passes of few rows ------------------------------------------------------------------------------------
//
// At most 32 pass rows: the weights stream through the chip once and everything else must stay out of their way.
// One launch: the activations are split into their bf16 parts on the way into shared memory by eight warps, each
// with every eighth k step, so that eight steps' loads are in flight; a step's operand is the high parts' rows and
// the low parts' rows one below the other, one MMA per 16 k takes both, and the epilogue adds the two halves of
// the accumulator.  128 weight rows by 64 k make a stage; the k steps of all tiles are laid end to end and cut
// into one equal share a CTA, so that every SM streams the same number of bytes whatever N and K are.
// A share that ends inside a tile leaves its sums in scratch, and the CTA that comes last at a tile adds them up
// in the order of k.
// The kernel starts under the one ahead of it and asks its first stages into L2 before it waits: weights are not
// written by the kernel ahead, and even if they were, L2 is where such writes land.
//
// Bound by HBM from some 200 MB on (one row on 28672 x 4096: 40 us, the part above a launch's fixed 6 to 8 us at
// 7.2 TB/s), by a chain of latencies below.  The kernel with weights straight from global memory into mma.sync
// fragments, a packing kernel before it and a finishing kernel behind took 58 us for sixteen rows of that weight;
// steps went from 419 to 340 us (one row, large), 538 to 406 us (sixteen rows), 417 to 298 us (one row, small).
constexpr int ROWS_THREADS = 14 * 32;
constexpr int ROWS_CONVERT_WARP = 6, ROWS_CONVERTERS = 8;
constexpr uint32_t ROWS_M = 128;
constexpr uint32_t ROWS_MAX = 32;           // pass rows
// k steps summed in tensor memory before the epilogue takes them over into its own f32 sums.  The tensor core drops
// what lies below its accumulator's last place: chains of 64 steps erred by 8.1e-6 of a GLU's result (16 rows x
// [28672, 4096]), the mma.sync kernel by 4.2e-6.  Chains of 16 are
// at 4.0e-6 (but 3.9e-6 against 3.7e-6 for twenty rows x [11264, 2048]), chains of eight at 3.7e-6 for 1.5 % of a step.
constexpr uint32_t ROWS_CLUSTER = 8;        // CTAs of a cluster, at most
constexpr uint32_t ROWS_CHAIN = 8, ROWS_BUFS = 4;   // (and four accumulators: the tensor cores run on while an epilogue adds shares up)

struct RowsArgs {
    const void *x;
    uint32_t T, K, cols, ksteps, units, ctas;
    uint32_t cluster;                 // CTAs that share a tile as one cluster (EPILOGUE, LOGPROBS; 1: none)
    bool whole;                       // every CTA takes whole tiles (EPILOGUE, LOGPROBS)
    uint32_t wm;                      // weight rows of a tile (a multiple of 4; ROWS_M but for whole tiles)
    uint32_t x_vec16;
    float *out;
    Epilogue e;                       // EPILOGUE (`out` is of its type)
    StatsOut so;                      // LOGPROBS
    uint32_t ids[ROWS_MAX];           // LOGPROBS: given tokens
    float *part;          // [2 * ctas shares][TP][128]
    uint32_t *counters;   // one a tile, zero between launches
    yx_dev_status *status;
};
__device__ __forceinline__ uint32_t share_begin(const RowsArgs &a, uint32_t p) { return (uint32_t)((uint64_t)p * a.units / a.ctas); }
__device__ __forceinline__ uint32_t share_owner(const RowsArgs &a, uint32_t u) { return (uint32_t)((((uint64_t)u + 1) * a.ctas - 1) / a.units); }

// TP pass rows of this lane's weight row.
template <int TP, bool GLU>
__device__ __forceinline__ void store_few(const RowsArgs &a, const float (&v)[TP], uint32_t row, int lane) {
    if constexpr (!GLU) {
        if (row >= a.cols) return;
#pragma unroll
        for (int i = 0; i < TP; i++)
            if (i < (int)a.T) a.out[(size_t)i * a.cols + row] = v[i];
    } else {
        // (see store_rows: the lower half of the warp finishes the first half of the pass rows)
        const uint32_t col = (row >> 5) * GLU_GROUP + (lane & 15), t = lane < 16 ? 0 : TP / 2;
#pragma unroll
        for (int i = 0; i < TP / 2; i++) {
            const float other = __shfl_xor_sync(0xffffffffu, lane < 16 ? v[TP / 2 + i] : v[i], 16);
            const float g = lane < 16 ? v[i] : other, u = lane < 16 ? other : v[TP / 2 + i];
            if (col < a.cols && t + i < a.T) a.out[(size_t)(t + i) * a.cols + col] = g / (1.0f + expf(-g)) * u;
        }
    }
}

// Accumulator columns of a k step's products: PARTS blocks of TP pass rows, in what an MMA of 128 weight rows takes (a
// multiple of 16), and how far apart the accumulators lie.
constexpr uint32_t rows_columns(int tp, int parts) { return (uint32_t)(tp * parts + 15) / 16 * 16; }
constexpr uint32_t rows_pitch(int tp, int parts) {
    uint32_t c = 16;
    while (c < rows_columns(tp, parts)) c *= 2;
    return c;
}
// Stages of the ring, and the warps that fill its activations in turn.  A barrier's parity tells a phase from the one before,
// not from the one two before: a warp that waits for a slot's last use to be over has to know that the use before that is, and
// knows so from its own step before, whose slot was free, as long as the warps are no more than the stages.
constexpr uint32_t rows_stage_bytes(int tp, int parts) { return W_BYTES + rows_columns(tp, parts) * 128; }
constexpr uint32_t rows_stages(int tp, int kind, int parts) {
    const uint32_t n = (kind < EPILOGUE ? TC_SMEM_BUDGET : 210 * 1024) / rows_stage_bytes(tp, parts);
    return n < TC_MAX_STAGES ? n : TC_MAX_STAGES;
}
constexpr uint32_t rows_converters(int tp, int kind, int parts) {
    return rows_stages(tp, kind, parts) < ROWS_CONVERTERS ? rows_stages(tp, kind, parts) : ROWS_CONVERTERS;
}

template <int TP, int KIND, int PARTS>
__global__ void __launch_bounds__(ROWS_THREADS, 1)
matmul_rows_kernel(const __grid_constant__ CUtensorMap w_map, const __grid_constant__ RowsArgs a) {
    extern __shared__ __align__(1024) unsigned char smem[];
    __shared__ __align__(8) uint64_t bar_store[2 * TC_MAX_STAGES + 2 * ROWS_BUFS];
    __shared__ uint32_t tmem_base_s;
    __shared__ int abort_flag;
    __shared__ int last_s;
    constexpr bool GLU_TILES = KIND == GLU;
    constexpr uint32_t NB = rows_columns(TP, PARTS), PITCH = rows_pitch(TP, PARTS), STAGE = rows_stage_bytes(TP, PARTS);
    constexpr uint32_t S = rows_stages(TP, KIND, PARTS), CONVERTERS = rows_converters(TP, KIND, PARTS);
    static_assert(CONVERTERS <= S, "a step's slot has to be free one use after the warp's step before");
    constexpr uint32_t TMEM = ROWS_BUFS * PITCH;
    constexpr int SCRATCH = KIND == EPILOGUE ? TP * 32 : KIND == LOGPROBS ? STATS_SCRATCH : 1;   // floats a warp
    __shared__ __align__(16) float scratch_s[4 * SCRATCH];
    float *scratch = scratch_s + ((threadIdx.x >> 5) & 3) * SCRATCH;
    __shared__ float4 stats_s[4][KIND == LOGPROBS ? 32 : 1];
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const uint32_t base = smem_u32(smem);
    const uint32_t b_full = smem_u32(bar_store), b_empty = b_full + 8 * TC_MAX_STAGES;
    const uint32_t b_acc_full = b_empty + 8 * TC_MAX_STAGES, b_acc_empty = b_acc_full + 8 * ROWS_BUFS;
    const uint32_t wm = KIND < EPILOGUE ? ROWS_M : a.wm;
    volatile int *abortp = &abort_flag;
    uint32_t u0, u1;
    if (KIND >= EPILOGUE && a.cluster > 1) {
        const uint32_t tile = blockIdx.x / a.cluster, at = blockIdx.x - tile * a.cluster;
        u0 = tile * a.ksteps + at * a.ksteps / a.cluster;
        u1 = tile * a.ksteps + (at + 1) * a.ksteps / a.cluster;
    } else if (KIND >= EPILOGUE && a.whole) {
        const uint64_t tiles = a.units / a.ksteps;
        u0 = (uint32_t)(blockIdx.x * tiles / a.ctas) * a.ksteps;
        u1 = (uint32_t)((blockIdx.x + 1) * tiles / a.ctas) * a.ksteps;
    } else {
        u0 = share_begin(a, blockIdx.x);
        u1 = share_begin(a, blockIdx.x + 1);
    }

    auto weight_rows = [&](uint32_t u, int &x, int &y, int &z) {
        const uint32_t tile = u / a.ksteps;
        x = (int)((u - tile * a.ksteps) * TC_KSTEP);
        y = GLU_TILES ? 0 : (int)(tile * wm);
        z = GLU_TILES ? (int)(tile * (ROWS_M / (2 * GLU_GROUP))) : 0;
    };
    if (warp == 4 && elect()) {
        prefetch_tensormap(&w_map);
        for (uint32_t u = u0; u < u1 && u - u0 < S; u++) {
            int x, y, z;
            weight_rows(u, x, y, z);
            tma_prefetch_4d(&w_map, x, y, 0, z);
        }
    }
    if (threadIdx.x == 0) {
        abort_flag = 0;
        for (uint32_t s = 0; s < S; s++) {
            mbar_init(b_full + 8 * s, 2);    // the weights' copy and the converting warp
            mbar_init(b_empty + 8 * s, 1);
        }
        for (uint32_t b = 0; b < ROWS_BUFS; b++) {
            mbar_init(b_acc_full + 8 * b, 1);
            mbar_init(b_acc_empty + 8 * b, 4);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 5) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base_s)), "n"(TMEM) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_base_s;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    auto finish = [&](const float (&v)[TP], uint32_t tile, uint32_t row) {
        if constexpr (KIND < EPILOGUE) store_few<TP, KIND == GLU>(a, v, row, lane);
        else if constexpr (KIND == EPILOGUE) {
            stage<TP>(v, 0, scratch, lane);
            finish_staged<TP>(a.e, a.out, a.T, a.cols, min(a.cols, (tile + 1) * wm), scratch, 0, row - lane, lane);
        } else {
            stats_s[warp][lane] = stats_of(a.so, a.T, min(a.cols, (tile + 1) * wm), v, 0, row, a.ids, scratch, lane);
            asm volatile("bar.sync 2, 128;" ::: "memory");
            if (warp == 0 && lane < (int)a.T) {
                const float4 four[4] = {stats_s[0][lane], stats_s[1][lane], stats_s[2][lane], stats_s[3][lane]};
                a.so.stats[(size_t)lane * a.so.blocks + tile] = merge_four(four);
            }
            asm volatile("bar.sync 2, 128;" ::: "memory");
        }
    };

    if (warp == 4) {
        // ---- weights --------------------------------------------------------------------------
        if (elect()) {
            // (see the pair kernel's: one thread, and nothing in its loop that can be kept out)
            uint32_t s = 0, phase = 0;
            int x, y, z;
            weight_rows(u0, x, y, z);
            for (uint32_t u = u0; u < u1; u++) {
                if (u - u0 >= S && !mbar_try(b_empty + 8 * s, phase ^ 1u)) {
                    mbar_wait_slow(b_empty + 8 * s, phase ^ 1u, abortp, a.status, 511);
                    if (*abortp) break;
                }
                mbar_expect_tx(b_full + 8 * s, wm * 128u);
                tma_load_4d(base + s * STAGE, &w_map, x, y, 0, z, b_full + 8 * s);
                x += TC_KSTEP;
                if (x == (int)(a.ksteps * TC_KSTEP)) {   // the next tile
                    x = 0;
                    if (GLU_TILES) z += ROWS_M / (2 * GLU_GROUP);
                    else y += wm;
                }
                if (++s == S) {
                    s = 0;
                    phase ^= 1u;
                }
            }
        }
    } else if (warp == 5) {
        // ---- MMA issuer -----------------------------------------------------------------------
        if (elect()) {
            constexpr uint32_t idesc = f16_instr_desc(true, false, ROWS_M, NB);
            uint32_t s = 0, phase = 0, n = 0, piece_end = u0;
            for (uint32_t u = u0; u < u1 && !*abortp; n++) {
                if (u == piece_end) piece_end = min(u1, (u / a.ksteps + 1) * a.ksteps);
                const uint32_t end = min(piece_end, u + ROWS_CHAIN);
                const uint32_t buf = n % ROWS_BUFS, acc = tmem + buf * PITCH;
                if (n >= ROWS_BUFS) mbar_wait(b_acc_empty + 8 * buf, (n / ROWS_BUFS - 1) & 1u, abortp, a.status, 512);
                tc_fence_after();
                for (uint32_t first = u; u < end; u++) {
                    if (!mbar_try(b_full + 8 * s, phase)) {
                        mbar_wait_slow(b_full + 8 * s, phase, abortp, a.status, 513);
                        if (*abortp) break;
                    }
                    tc_fence_after();
                    const uint32_t w_lo = desc_lo(base + s * STAGE, 0), x_lo = w_lo + W_BYTES / 16;
#pragma unroll
                    for (uint32_t kk = 0; kk < 4; kk++) umma_ss_lo(acc, w_lo + 2 * kk, x_lo + 2 * kk, idesc, u > first || kk > 0);
                    umma_commit(b_empty + 8 * s);
                    if (++s == S) {
                        s = 0;
                        phase ^= 1u;
                    }
                }
                umma_commit(b_acc_full + 8 * buf);
            }
        }
    } else if (warp >= ROWS_CONVERT_WARP) {
        // ---- activations: every eighth step is this warp's ------------------------------------------
        // (of a ring of seven stages every seventh; the eighth warp has none)
        for (uint32_t u = warp - ROWS_CONVERT_WARP < (int)CONVERTERS ? u0 + (uint32_t)(warp - ROWS_CONVERT_WARP) : u1; u < u1; u += CONVERTERS) {
            const uint32_t it = u - u0, s = it % S, use = it / S;
            const uint32_t k = (u % a.ksteps) * TC_KSTEP + (lane & 7) * 8;
            constexpr int R = TP / 4;          // 16-byte operand chunks (eight k of a pass row) a lane
            uint4 bits[R];                     // bf16 rows are operands as they are
            float v[R][8];
#pragma unroll
            for (int r = 0; r < R; r++) {
                const uint32_t t = r * 4 + (lane >> 3);
                if (t >= a.T) continue;        // (rows past T only reach accumulator columns that nobody reads)
                const size_t at = (size_t)t * a.K + k;
                if constexpr (KIND < EPILOGUE) {
                    const float *p = (const float *)a.x + at;
                    if (a.x_vec16) {
                        *(float4 *)&v[r][0] = *(const float4 *)p;
                        *(float4 *)&v[r][4] = *(const float4 *)(p + 4);
                    } else {
#pragma unroll
                        for (int j = 0; j < 4; j++) *(float2 *)&v[r][2 * j] = *(const float2 *)(p + 2 * j);
                    }
                } else if (k >= a.K) {         // (K ends inside the step, at a multiple of eight)
                    bits[r] = make_uint4(0, 0, 0, 0);
#pragma unroll
                    for (int j = 0; j < 8; j++) v[r][j] = 0.0f;
                } else if constexpr (PARTS == 1) {
                    if (a.x_vec16) {
                        bits[r] = *(const uint4 *)((const uint16_t *)a.x + at);
                    } else {
                        const uint16_t *p = (const uint16_t *)a.x + at;
                        bits[r] = make_uint4(p[0] | (uint32_t)p[1] << 16, p[2] | (uint32_t)p[3] << 16, p[4] | (uint32_t)p[5] << 16, p[6] | (uint32_t)p[7] << 16);
                    }
                } else {
                    if (a.x_vec16) load8<PARTS == 2 ? YX_F16 : YX_F32, true>(a.x, at, v[r]);
                    else load8<PARTS == 2 ? YX_F16 : YX_F32, false>(a.x, at, v[r]);
                }
            }
            if (use > 0) mbar_wait(b_empty + 8 * s, (use - 1) & 1u, abortp, a.status, 514);
            if (__any_sync(0xffffffffu, *abortp)) break;
            unsigned char *dst = smem + s * STAGE + W_BYTES;
#pragma unroll
            for (int r = 0; r < R; r++) {
                const uint32_t t = r * 4 + (lane >> 3);
                if (t >= a.T) continue;
                unsigned char *at = dst + t * 128 + (((lane & 7) ^ (t & 7)) << 4);
                if constexpr (KIND < EPILOGUE) {
                    uint32_t h[4], l[4];
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        h[j] = pack2<true>(v[r][2 * j], v[r][2 * j + 1]);
                        const float2 b = unpack2<true>(h[j]);
                        l[j] = pack2<true>(v[r][2 * j] - b.x, v[r][2 * j + 1] - b.y);
                    }
                    *(uint4 *)at = make_uint4(h[0], h[1], h[2], h[3]);
                    *(uint4 *)(at + TP * 128) = make_uint4(l[0], l[1], l[2], l[3]);
                } else if constexpr (PARTS == 1) {
                    *(uint4 *)at = bits[r];
                } else {
                    uint32_t parts[PARTS][4];
                    cut_parts<PARTS>(v[r], parts);
#pragma unroll
                    for (int p = 0; p < PARTS; p++) *(uint4 *)(at + p * TP * 128) = make_uint4(parts[p][0], parts[p][1], parts[p][2], parts[p][3]);
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(b_full + 8 * s);
        }
    } else {
        // ---- epilogue -------------------------------------------------------------------------
        uint32_t n = 0;
        for (uint32_t u = u0; u < u1;) {
            const uint32_t tile = u / a.ksteps, end = min(u1, (tile + 1) * a.ksteps);
            const bool whole = end - u == a.ksteps;
            const uint32_t wr = warp * 32 + lane, row = tile * wm + wr;
            // The CTAs that share this tile, found while the tile is being summed (the divisions take a third of a
            // microsecond).  Only the first of them may have begun in a tile before it: then this is its last piece.
            uint32_t q0 = 0, q1 = 0, later = 0;
            if (!whole && (KIND < EPILOGUE || a.cluster == 1)) {
                q0 = share_owner(a, tile * a.ksteps);
                q1 = share_owner(a, (tile + 1) * a.ksteps - 1);
                later = share_begin(a, q0) < tile * a.ksteps;
            }
            float v[TP];
#pragma unroll
            for (int i = 0; i < TP; i++) v[i] = 0.0f;
            for (; u < end; n++) {
                u = min(end, u + ROWS_CHAIN);
                const uint32_t buf = n % ROWS_BUFS, acc = tmem + buf * PITCH + ((uint32_t)warp << 21);
                mbar_wait(b_acc_full + 8 * buf, (n / ROWS_BUFS) & 1u, abortp, a.status, 515);
                __syncwarp();   // (a wait that ran out does not stop these warps: their barriers below count all of them)
                tc_fence_after();
                if constexpr (PARTS != 2) {
                    // (the parts' sums one below the other, the smallest first)
                    float part[TP];
#pragma unroll
                    for (int p = PARTS - 1; p >= 0; p--) {
#pragma unroll
                        for (int h = 0; h < TP; h += TP < 16 ? TP : 16) {
                            uint32_t r[16];
                            tmem_ld16(acc + p * TP + h, r);
                            tmem_ld_wait();
#pragma unroll
                            for (int i = 0; i < (TP < 16 ? TP : 16); i++) part[h + i] = p == PARTS - 1 ? __uint_as_float(r[i]) : part[h + i] + __uint_as_float(r[i]);
                        }
                    }
#pragma unroll
                    for (int i = 0; i < TP; i++) v[i] += part[i];
                } else if constexpr (TP == 8) {
                    uint32_t r[16];
                    tmem_ld16(acc, r);
                    tmem_ld_wait();
#pragma unroll
                    for (int i = 0; i < 8; i++) v[i] += __uint_as_float(r[i]) + __uint_as_float(r[8 + i]);
                } else {
#pragma unroll
                    for (int h = 0; h < TP / 16; h++) {
                        uint32_t r[16], q[16];
                        tmem_ld16(acc + 16 * h, r);
                        tmem_ld16(acc + TP + 16 * h, q);
                        tmem_ld_wait();
#pragma unroll
                        for (int i = 0; i < 16; i++) v[16 * h + i] += __uint_as_float(r[i]) + __uint_as_float(q[i]);
                    }
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(b_acc_empty + 8 * buf);
            }
            if (whole) {
                finish(v, tile, row);
                continue;
            }
            if constexpr (KIND >= EPILOGUE) {
                if (a.cluster > 1) {   // (as in the pair kernel: the sums stay in shared memory)
#pragma unroll
                    for (int i = 0; i < TP; i += 4) *(float4 *)(smem + (i / 4 * 128u + wr) * 16u) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
                    break;
                }
            }
            auto share = [&](uint32_t q) { return a.part + (size_t)(2 * q + (q == q0 ? later : 0u)) * TP * 128u + wr; };
            float *mine = share(blockIdx.x);
#pragma unroll
            for (int i = 0; i < TP; i++)
                if (i < (int)a.T) __stcg(mine + i * 128, v[i]);
            __threadfence();
            asm volatile("bar.sync 1, 128;" ::: "memory");
            if (threadIdx.x == 0) {
                const int last = atomicAdd(a.counters + tile, 1u) == q1 - q0;
                if (last) a.counters[tile] = 0u;
                last_s = last;
            }
            asm volatile("bar.sync 1, 128;" ::: "memory");
            const bool last = last_s != 0;
            if (!last) continue;
            __threadfence();
#pragma unroll
            for (int i = 0; i < TP; i++) v[i] = 0.0f;
            constexpr int B = 64 / TP;   // shares read at once
            for (uint32_t q = q0; q <= q1; q += B) {
                float w[B][TP];
#pragma unroll
                for (int b = 0; b < B; b++) {
                    const float *src = share(min(q + b, q1));
#pragma unroll
                    for (int i = 0; i < TP; i++) w[b][i] = i < (int)a.T && q + b <= q1 ? __ldcg(src + i * 128) : 0.0f;
                }
#pragma unroll
                for (int b = 0; b < B; b++)
#pragma unroll
                    for (int i = 0; i < TP; i++) v[i] += w[b][i];
            }
            finish(v, tile, row);
        }
    }
    __syncwarp();
    if constexpr (KIND >= EPILOGUE) {
        if (a.cluster > 1) {
            // The cluster's first CTA adds up, in the order of k, and finishes.
            cluster_sync();
            if (blockIdx.x % a.cluster == 0 && warp < 4) {
                const uint32_t wr = warp * 32 + lane;
                float v[TP];
#pragma unroll
                for (int i = 0; i < TP; i += 4) {
                    float4 f[ROWS_CLUSTER];
#pragma unroll
                    for (uint32_t q = 0; q < ROWS_CLUSTER; q++) f[q] = load_cluster(mapa(base + (i / 4 * 128u + wr) * 16u, min(q, a.cluster - 1)));
#pragma unroll
                    for (uint32_t q = 1; q < ROWS_CLUSTER; q++)
                        if (q < a.cluster) f[0] = make_float4(f[0].x + f[q].x, f[0].y + f[q].y, f[0].z + f[q].z, f[0].w + f[q].w);
                    *(float4 *)(v + i) = f[0];
                }
                finish(v, blockIdx.x / a.cluster, blockIdx.x / a.cluster * ROWS_M + wr);
            }
            __syncwarp();
            cluster_sync();   // the sums are read
        }
    }
    if (*abortp)
        for (int i = 0; i < 64; i++) __nanosleep(1000);   // copies and products in flight come to rest
    tc_fence_before();
    __syncthreads();
    if (warp == 5) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(TMEM) : "memory");
}

using EncodeTiled = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                                 const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiled encode_tiled() {
    static const EncodeTiled fn = [] {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &found) != cudaSuccess ||
            found != cudaDriverEntryPointSuccess)
            p = nullptr;
        return (EncodeTiled)p;
    }();
    return fn;
}

// A map of a bf16 tensor, innermost dimension dense, 128-byte swizzle; rows outside it read as zero.
int encode(yx_ctx *ctx, CUtensorMap *map, uint32_t rank, const void *p, const cuuint64_t *dims, const cuuint64_t *strides, const cuuint32_t *box) {
    const cuuint32_t ones[4] = {1, 1, 1, 1};
    if (!encode_tiled()) return fail(ctx, YX_ERR_CUDA, "matmul: the driver has no cuTensorMapEncodeTiled");
    const CUresult r = encode_tiled()(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, rank, const_cast<void *>(p), dims, strides, box, ones,
                                      CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                      CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? YX_OK : fail(ctx, YX_ERR_CUDA, "matmul: cuTensorMapEncodeTiled failed with " + std::to_string((int)r));
}

// The weights in boxes of `rows` rows by 64 k; for a GLU four groups of 16 gate rows and the 16 up rows of the same columns.
int encode_weights(yx_ctx *ctx, CUtensorMap *map, const void *w, uint32_t N, uint32_t K, bool glu, uint32_t rows = 128) {
    const cuuint64_t row = (cuuint64_t)K * 2;
    if (glu) {
        const cuuint64_t dims[4] = {K, GLU_GROUP, 2, N / 2 / GLU_GROUP};
        const cuuint64_t strides[3] = {row, N / 2 * row, GLU_GROUP * row};
        const cuuint32_t box[4] = {TC_KSTEP, GLU_GROUP, 2, 128 / (2 * GLU_GROUP)};
        return encode(ctx, map, 4, w, dims, strides, box);
    }
    const cuuint64_t dims[4] = {K, N, 1, 1};
    const cuuint64_t strides[3] = {row, N * row, N * row};
    const cuuint32_t box[4] = {TC_KSTEP, rows, 1, 1};
    return encode(ctx, map, 4, w, dims, strides, box);
}

int ensure_counters(yx_ctx *ctx, size_t n) {
    const size_t before = ctx->mm_counters_cap;
    if (int rc = ensure_buffer(ctx, (void **)&ctx->mm_counters, &ctx->mm_counters_cap, std::max<size_t>(n, 512) * sizeof(uint32_t))) return rc;
    if (ctx->mm_counters_cap == before) return YX_OK;
    return check_cuda(ctx, cudaMemsetAsync(ctx->mm_counters, 0, ctx->mm_counters_cap, ctx->stream), "matmul: counters");
}

// (what changes places takes 32 KiB, in LOGPROBS half of that with the statistics in the other)
constexpr uint32_t smem_budget(int kind) { return kind < EPILOGUE ? TC_SMEM_BUDGET : 194 * 1024; }

template <int KIND, int CHUNKS>
constexpr auto pair_kernel() {
    if constexpr (KIND < EPILOGUE) return matmul_pair_kernel<KIND, CHUNKS>;
    else return matmul_exact_kernel<KIND, CHUNKS>;
}

// Clusters of `size` CTAs that are on the chip together (a GPC leaves some of its SMs out).  `known` remembers: 0 not asked
// yet, -1 none.  The kernel's shared memory is opted in for.
template <typename Kernel>
int resident_of(yx_ctx *ctx, int *known, Kernel kernel, unsigned threads, size_t smem, uint32_t size, int *out) {
    if (*known == 0) {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)ctx->sm_count / size * size);
        cfg.blockDim = dim3(threads);
        cfg.dynamicSmemBytes = smem;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = size;
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        int found = 0;
        const cudaError_t e = cudaOccupancyMaxActiveClusters(&found, kernel, &cfg);
        if (e != cudaSuccess) {   // (a size this device does not place)
            cudaGetLastError();
            found = 0;
        }
        found = std::min(found, ctx->sm_count / (int)size);
        *known = found > 0 ? found : -1;
    }
    *out = std::max(*known, 0);
    return YX_OK;
}
template <int KIND, int CHUNKS>
int resident_clusters(yx_ctx *ctx, int pairs, int *out) {
    auto *kernel = pair_kernel<KIND, CHUNKS>();
    int &n = ctx->mm_clusters[KIND][CHUNKS - 2][pairs - 1];
    if (n == 0)
        if (int rc = check_cuda(ctx, cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_budget(KIND)), "matmul: shared memory attribute"))
            return rc;
    if (int rc = resident_of(ctx, &n, kernel, TC_THREADS, smem_budget(KIND), 2 * pairs, out)) return rc;
    return pairs > 1 || *out > 0 ? YX_OK : fail(ctx, YX_ERR_CUDA, "matmul: no CTA pair is placed");
}

// Pass rows are spread evenly over as few tiles as hold them: 300 rows are two tiles of 160, not 256 and 64.
uint32_t rows_of_tiles(uint32_t T, uint32_t tiles) { return ((T + tiles - 1) / tiles + 31) / 32 * 32; }
uint32_t tile_rows(uint32_t T) { return rows_of_tiles(T, (T + TC_MAX_BT - 1) / TC_MAX_BT); }

// Pairs of a cluster for each of `tiles` tiles: as many as the chip places at once.
template <int KIND, int CHUNKS>
int cluster_for(yx_ctx *ctx, uint32_t tiles, uint32_t ksteps, uint32_t *out) {
    *out = 1;
    for (uint32_t c = std::min({MAX_CLUSTER, (uint32_t)ctx->sm_count / 2 / tiles, ksteps}); c > 1; c--) {
        int resident = 0;
        if (int rc = resident_clusters<KIND, CHUNKS>(ctx, (int)c, &resident)) return rc;
        if (tiles > (uint32_t)resident) continue;
        *out = c;
        break;
    }
    return YX_OK;
}

// Tiles that pass rows taken exactly are spread over.  More than hold them where that leaves fewer pairs idle: a k step takes
// a CTA what its 16 KiB of weights and 64 bytes a pass row and part take at some 60 bytes a nanosecond, and pairs of a
// cluster share it (on the device, 300 f32 rows x [5633, 2040]: 46 tiles of 160 rows 34.6 us, 69 of 128 29.7; 600 bf16 x [4096, 4096] 40.3 and 27.7).
template <int KIND>
int exact_row_tiles(yx_ctx *ctx, const Product &p, uint32_t *out) {
    const uint32_t columns = (p.N + TC_M - 1) / TC_M, least = (p.T + TC_MAX_BT - 1) / TC_MAX_BT, ksteps = (p.K + TC_KSTEP - 1) / TC_KSTEP;
    *out = least;
    float best = 0.0f;
    for (uint32_t t = least; t <= least + 4 && (uint64_t)columns * t <= (uint64_t)ctx->sm_count / 2; t++) {
        uint32_t shared = 1;
        if (int rc = cluster_for<KIND, 2>(ctx, columns * t, ksteps, &shared)) return rc;
        const float cost = (16384.0f + 64.0f * (float)(p.parts * (int)rows_of_tiles(p.T, t))) / (float)shared;
        if (t > least && cost >= best) continue;
        *out = t;
        best = cost;
    }
    return YX_OK;
}

// How many pairs share the k steps of `tiles` left-over tiles.  Either every tile is cut into the same number of
// shares, which leaves some pairs idle, or all pairs take an equal share, which lets shares run over the end of a
// tile: one more epilogue and one more share to add up for most pairs.  A k step takes 0.26 us and 2 ns a pass row
// (62 GB/s into each SM, measured at 96 to 256 rows), the extra epilogue 3 us, adding up at all another 6; behind
// whole rounds both are hidden.  A share of fewer than four k steps costs more to add up than it saves.
uint32_t share_rest(uint32_t tiles, uint32_t ksteps, uint32_t pairs, uint32_t bt, bool hidden, float row = 0.002f) {
    const uint32_t most = std::max(1u, ksteps / 4), each = std::min(pairs / tiles, most);
    const uint32_t all = std::min(pairs, tiles * most);
    const float step = 0.26f + row * (float)bt, overrun = hidden ? 1.0f : each == 1 ? 9.0f : 3.0f;
    const float even = step * (float)((ksteps + each - 1) / each), equal = step * (float)(tiles * ksteps) / (float)all;
    return even <= equal + overrun ? tiles * each : all;
}

// What a pass of more than 32 rows is given, whatever becomes of the product.
template <int KIND, int CHUNKS>
int plan_pairs(yx_ctx *ctx, const Product &p, PairArgs &a) {
    int pairs = 0;
    if (int rc = resident_clusters<KIND, CHUNKS>(ctx, 1, &pairs)) return rc;
    a.cluster = 1;
    a.T = p.T;
    a.cols = KIND == GLU ? p.N / 2 : p.N;
    a.parts = kind_parts(KIND, p.parts);
    a.t_tiles = KIND < EPILOGUE ? (p.T + TC_MAX_BT - 1) / TC_MAX_BT : p.t_tiles;
    a.bt = rows_of_tiles(p.T, a.t_tiles);
    a.ksteps = (p.K + TC_KSTEP - 1) / TC_KSTEP;
    a.stages = std::min<uint32_t>(TC_MAX_STAGES, (smem_budget(KIND) - 1024) / (W_BYTES + a.parts * a.bt * 64u));
    const uint32_t tiles = ((p.N + TC_M - 1) / TC_M) * a.t_tiles;
    a.pairs = (uint32_t)pairs;
    a.rounds = tiles / a.pairs;
    a.rest_units = (tiles - a.rounds * a.pairs) * a.ksteps;
    if constexpr (KIND >= EPILOGUE) {
        // Tiles that leave every other pair or more idle are cut along k into one share for each pair of a cluster, whose
        // sums meet in shared memory.  Through scratch and through clusters, us: 80 rows bf16 x [4096, 4096] 17.9 and 13.3, 256 rows
        // 30 and 20, 128 x [2048, 2048] 18.4 and 8.7, 512 f32 x [1024, 2816] 39 and 23; even where clusters leave half of the pairs
        // without work, as 80 x [1024, 14336] does, 24.7 and 18.8.
        // (the sums take 512 bytes a pass row of the ring, which has room for that as long as it fills shared memory)
        if (a.rounds == 0 && a.stages * (W_BYTES + a.parts * a.bt * 64u) >= a.bt * 512u)
            if (int rc = cluster_for<KIND, CHUNKS>(ctx, tiles, a.ksteps, &a.cluster)) return rc;
    }
    const uint32_t rest = tiles - a.rounds * a.pairs;
    if (KIND >= EPILOGUE && rest > 0 && a.rounds > 0) {
        // Behind whole rounds every left-over tile gets the same number of pairs, one where they are more than half: pairs
        // that find fewer others at work are as much quicker (all pairs in equal shares and now, us: 80 rows bf16 x [50257, 4096]
        // 85.6 and 78.4, 128 x [32000, 4096] 63.8 and 55.8, 700 f16 x [11264, 2048] 85.0 and 61.2; none of eleven shapes slower).
        a.rest_pairs = rest * std::min(a.pairs / rest, std::max(1u, a.ksteps / 4));
    } else if (rest > 0 && a.cluster == 1) {
        a.rest_pairs = share_rest(rest, a.ksteps, a.pairs, a.bt, a.rounds > 0, 0.001f * (float)a.parts);
    }
    a.bufs = a.bt <= 128 ? 4 : a.bt <= 160 ? 3 : 2;
    a.buf_columns = 512 / a.bufs / 32 * 32;
    if (KIND < EPILOGUE) {
        const bool large = a.bufs < TC_MAX_BUFS && a.rounds > 0 && a.ksteps >= 2 * TC_CHAIN;
        a.chain = large ? TC_CHAIN : std::min(a.rounds > 0 ? TC_SHORT_CHAIN : TC_CUT_CHAIN, std::max(TC_LEAST_CHAIN, a.ksteps / 2));
        a.long_first = large && a.bufs == 2;
    } else {
        a.chain = KIND == EPILOGUE && p.e.out_dtype != YX_F32 ? NARROW_CHAIN[a.parts - 1] : EXACT_CHAIN[a.parts - 1];
    }
    a.status = ctx->dev_status;
    return YX_OK;
}

template <int KIND, int CHUNKS>
int launch_pairs(yx_ctx *ctx, const CUtensorMap &w_map, const CUtensorMap &x_map, const PairArgs &a) {
    const uint32_t rest = a.rest_units / a.ksteps, shares = a.cluster > 1 ? rest * a.cluster : a.rest_pairs;
    const uint32_t dealt[6] = {2, a.cluster, a.rounds, rest, shares, a.chain};
    std::copy(dealt, dealt + 6, ctx->mm_last);
    const dim3 grid(2 * (a.rounds > 0 ? a.pairs : shares)), block(TC_THREADS);
    const size_t smem = a.stages * (W_BYTES + a.parts * a.bt * 64u);
    if constexpr (KIND < EPILOGUE) return launch_dependent(ctx, "matmul kernel launch", pair_kernel<KIND, CHUNKS>(), grid, block, smem, w_map, x_map, a);
    else return launch_cluster(ctx, "matmul kernel launch", pair_kernel<KIND, CHUNKS>(), grid, block, smem, 2 * a.cluster, w_map, x_map, a);
}

// The map of `parts` matrices [T, K] one behind the other: a CTA's half of a tile's rows, of every part.
int encode_rows(yx_ctx *ctx, CUtensorMap *map, const void *x, uint32_t T, uint32_t K, uint32_t parts, uint32_t bt) {
    const cuuint64_t dims[3] = {K, T, parts};
    const cuuint64_t strides[2] = {(cuuint64_t)K * 2, (cuuint64_t)T * K * 2};
    const cuuint32_t box[3] = {TC_KSTEP, bt / 2, parts};
    return encode(ctx, map, 3, x, dims, strides, box);
}

// PLAIN and GLU.
template <int KIND, int CHUNKS>
int matmul_pair_rows(yx_ctx *ctx, const Product &p) {
    const float *x = (const float *)p.x;
    const size_t n = (size_t)p.T * p.K;
    if (int rc = ensure_buffer(ctx, (void **)&ctx->mm_packed, &ctx->mm_packed_cap, n * 4)) return rc;
    PairArgs a{};
    if (int rc = plan_pairs<KIND, CHUNKS>(ctx, p, a)) return rc;
    a.out = (float *)p.out;
    // The most any pass needs (39 MB), so that a call that is being recorded into a graph finds it whatever passes came
    // before: the shares' room does not grow with the rows (512 rows may leave no tile over, 100 rows many).
    if (int rc = ensure_buffer(ctx, (void **)&ctx->mm_part, &ctx->mm_part_cap, (size_t)a.pairs * 2 * 2 * TC_MAX_BT * 128 * sizeof(float))) return rc;
    a.part = ctx->mm_part;
    if (int rc = ensure_counters(ctx, 2 * a.pairs)) return rc;
    a.counters = ctx->mm_counters;

    CUtensorMap w_map, x_map;
    if (int rc = encode_weights(ctx, &w_map, p.w, p.N, p.K, KIND == GLU)) return rc;
    uint4 *hi = (uint4 *)ctx->mm_packed, *lo = hi + n / 8;
    if (int rc = encode_rows(ctx, &x_map, hi, p.T, p.K, 2, a.bt)) return rc;
    ctx->last_launch = yx_ctx::LAST_OTHER;
    if (int rc = launch_dependent(ctx, "matmul: activation split kernel launch", ((uintptr_t)x & 15u) == 0 ? split_rows_kernel<true> : split_rows_kernel<false>,
                                  dim3((unsigned)((n / 8 + 255) / 256)), dim3(256), 0, x, n, hi, lo))
        return rc;
    return launch_pairs<KIND, CHUNKS>(ctx, w_map, x_map, a);
}

// The scratch of the kinds that take their rows exactly: theirs alone, at the most any pass needs, and never moved.
int exact_scratch(yx_ctx *ctx, size_t tiles, float **part, uint32_t **counters) {
    if (int rc = grow(ctx, ctx->ep_part, (size_t)(ctx->sm_count / 2) * 2 * 2 * TC_MAX_BT * 128 * sizeof(float))) return rc;
    char *before = ctx->ep_counters.dev;
    if (int rc = grow(ctx, ctx->ep_counters, std::max<size_t>(tiles, 65536) * sizeof(uint32_t))) return rc;
    *part = (float *)ctx->ep_part.dev;
    *counters = (uint32_t *)ctx->ep_counters.dev;
    if (ctx->ep_counters.dev == before) return YX_OK;
    return check_cuda(ctx, cudaMemsetAsync(ctx->ep_counters.dev, 0, ctx->ep_counters.cap, ctx->stream), "matmul: counters");
}

// EPILOGUE and LOGPROBS.
template <int KIND, int CHUNKS>
int exact_pair_rows(yx_ctx *ctx, Product &p) {
    const size_t n = (size_t)p.T * p.K;
    PairArgs a{};
    if (int rc = plan_pairs<KIND, CHUNKS>(ctx, p, a)) return rc;
    a.out = (float *)p.out;
    a.e = p.e;
    p.blocks = 2 * ((p.N + TC_M - 1) / TC_M);
    a.so = StatsOut{(float4 *)p.stats, p.blocks, p.picked};
    a.ids = p.ids_dev;
    if (int rc = exact_scratch(ctx, 2 * a.pairs, &a.part, &a.counters)) return rc;
    const void *rows = p.x;
    if (p.parts > 1) {
        if (int rc = grow(ctx, ctx->ep_rows, n * 2 * p.parts)) return rc;
        rows = ctx->ep_rows.dev;
    } else if (((uintptr_t)rows & 15u) != 0) {
        if (int rc = grow(ctx, ctx->ep_rows, n * 2)) return rc;
        if (int rc = check_cuda(ctx, cudaMemcpyAsync(ctx->ep_rows.dev, rows, n * 2, cudaMemcpyDeviceToDevice, ctx->stream), "matmul: unaligned rows")) return rc;
        rows = ctx->ep_rows.dev;
    }
    CUtensorMap w_map, x_map;
    if (int rc = encode_weights(ctx, &w_map, p.w, p.N, p.K, false)) return rc;
    if (int rc = encode_rows(ctx, &x_map, rows, p.T, p.K, p.parts, a.bt)) return rc;
    ctx->last_launch = yx_ctx::LAST_OTHER;
    if (p.parts > 1) {
        const bool vec = ((uintptr_t)p.x & 15u) == 0;
        auto *kernel = p.parts == 2 ? (vec ? cut_rows_kernel<YX_F16, 2, true> : cut_rows_kernel<YX_F16, 2, false>)
                                    : (vec ? cut_rows_kernel<YX_F32, 3, true> : cut_rows_kernel<YX_F32, 3, false>);
        if (int rc = launch_dependent(ctx, "matmul: activation split kernel launch", kernel, dim3((unsigned)((n / 8 + 255) / 256)), dim3(256), 0, p.x, n,
                                      (uint4 *)ctx->ep_rows.dev))
            return rc;
    }
    // (with LOGPROBS the given tokens' kernel is ahead, or that of the slice of rows before, which start this one after their own
    // waits too)
    a.early_w = p.parts > 1 || KIND == LOGPROBS;
    return launch_pairs<KIND, CHUNKS>(ctx, w_map, x_map, a);
}

template <int TP, int KIND, int PARTS>
int matmul_few_rows(yx_ctx *ctx, Product &p) {
    constexpr uint32_t stage_bytes = rows_stage_bytes(TP, PARTS), stages = rows_stages(TP, KIND, PARTS);
    auto *kernel = matmul_rows_kernel<TP, KIND, PARTS>;
    bool &configured = ctx->mm_rows_configured[KIND][PARTS - 1][TP / 16];
    if (!configured) {
        if (int rc = check_cuda(ctx, cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, stages * stage_bytes),
                                "matmul: shared memory attribute"))
            return rc;
        configured = true;
    }
    const uint32_t T = p.T, N = p.N, K = p.K;
    RowsArgs a{};
    a.x = p.x;
    if (KIND < EPILOGUE) {
        // Other CTAs still read the rows when a tile's result is written: a result over its own rows takes them from a copy.
        const uintptr_t x0 = (uintptr_t)p.x, o0 = (uintptr_t)p.out;
        if (o0 < x0 + (size_t)T * K * 4 && x0 < o0 + (size_t)T * (KIND == GLU ? N / 2 : N) * 4) {
            if (int rc = ensure_buffer(ctx, (void **)&ctx->mm_packed, &ctx->mm_packed_cap, (size_t)ROWS_MAX * K * 4)) return rc;
            if (int rc = check_cuda(ctx, cudaMemcpyAsync(ctx->mm_packed, p.x, (size_t)T * K * 4, cudaMemcpyDeviceToDevice, ctx->stream), "matmul: rows under the result"))
                return rc;
            a.x = ctx->mm_packed;
        }
    }
    a.T = T;
    a.K = K;
    a.cols = KIND == GLU ? N / 2 : N;
    a.ksteps = (K + TC_KSTEP - 1) / TC_KSTEP;
    uint32_t tiles = (N + ROWS_M - 1) / ROWS_M;
    a.wm = ROWS_M;
    a.units = tiles * a.ksteps;
    a.ctas = std::min((uint32_t)ctx->sm_count, std::max(1u, a.units / 2));
    a.cluster = 1;
    if constexpr (KIND >= EPILOGUE) {
        // (as in the pair kernel)
        for (uint32_t c = std::min({ROWS_CLUSTER, (uint32_t)ctx->sm_count / tiles, a.ksteps}); c > 1; c--) {
            int resident = 0;
            if (int rc = resident_of(ctx, &ctx->mm_rows_clusters[KIND][PARTS - 1][TP / 16][c - 1], kernel, ROWS_THREADS, stages * stage_bytes, c, &resident)) return rc;
            if (tiles > (uint32_t)resident) continue;
            a.cluster = c;
            a.ctas = tiles * c;
            break;
        }
        // Whole tiles where there is one round of them or the last keeps half of the SMs busy, and then tiles as low as fill the
        // rounds: cheaper than adding up shares (us: 88 tiles of 32 k steps, 8 f16 rows, 13.7 in equal shares and 10.8 as 148 lower ones, 79
        // of 16 steps 9.0 and 6.8, 224 of 64 44.5 and 42.3; but 157 of 32 16.9 and 17.6, 172 of 64 32.4 and 33.1).
        const uint32_t sms = (uint32_t)ctx->sm_count, last = tiles % sms;
        if (a.cluster == 1 && (tiles <= sms || last == 0 || last * 2 >= sms)) {
            const uint32_t most = (tiles + sms - 1) / sms * sms, each = (N + most - 1) / most;
            a.whole = true;
            a.wm = std::clamp((each + 3) / 4 * 4, 32u, ROWS_M);
            tiles = (N + a.wm - 1) / a.wm;
            a.units = tiles * a.ksteps;
            a.ctas = std::min(sms, tiles);
        }
    }
    a.x_vec16 = ((uintptr_t)a.x & 15u) == 0;
    a.out = (float *)p.out;
    a.e = p.e;
    p.blocks = tiles;
    a.so = StatsOut{(float4 *)p.stats, p.blocks, p.picked};
    if (KIND == LOGPROBS) std::copy(p.ids_host, p.ids_host + T, a.ids);
    a.status = ctx->dev_status;
    if (KIND < EPILOGUE) {
        // (for any number of rows and any weight, as in matmul_pair_rows: one row may be followed by sixteen in a recording)
        if (int rc = ensure_buffer(ctx, (void **)&ctx->mm_part, &ctx->mm_part_cap, (size_t)2 * ctx->sm_count * ROWS_MAX * 128 * sizeof(float))) return rc;
        if (int rc = ensure_counters(ctx, tiles)) return rc;
        a.part = ctx->mm_part;
        a.counters = ctx->mm_counters;
    } else if (int rc = exact_scratch(ctx, tiles, &a.part, &a.counters)) {
        return rc;
    }
    CUtensorMap w_map;
    if (int rc = encode_weights(ctx, &w_map, p.w, N, K, KIND == GLU, a.wm)) return rc;
    const uint32_t dealt[6] = {1, a.cluster, a.whole, tiles, a.ctas, ROWS_CHAIN};
    std::copy(dealt, dealt + 6, ctx->mm_last);
    ctx->last_launch = yx_ctx::LAST_OTHER;
    return launch_cluster(ctx, "matmul kernel launch", kernel, dim3(a.ctas), dim3(ROWS_THREADS), stages * stage_bytes, a.cluster > 1 ? a.cluster : 0, w_map, a);
}

template <int KIND>
int matmul_tc(yx_ctx *ctx, Product &p) {
    if (p.T <= 8) return matmul_few_rows<8, KIND, 2>(ctx, p);
    if (p.T <= 16) return matmul_few_rows<16, KIND, 2>(ctx, p);
    if (p.T <= 32) return matmul_few_rows<32, KIND, 2>(ctx, p);
    const uint32_t rows = tile_rows(p.T);
    if (rows <= 128) return matmul_pair_rows<KIND, 2>(ctx, p);
    if (rows <= 192) return matmul_pair_rows<KIND, 3>(ctx, p);
    return matmul_pair_rows<KIND, 4>(ctx, p);
}

template <int KIND, int PARTS>
int exact_few_rows(yx_ctx *ctx, Product &p) {
    // (eight columns of one part are fewer than an MMA takes)
    if constexpr (PARTS > 1)
        if (p.T <= 8) return matmul_few_rows<8, KIND, PARTS>(ctx, p);
    if (p.T <= 16) return matmul_few_rows<16, KIND, PARTS>(ctx, p);
    return matmul_few_rows<32, KIND, PARTS>(ctx, p);
}
template <int KIND>
int exact_tc(yx_ctx *ctx, Product &p) {
    if (p.T <= ROWS_MAX)
        return p.parts == 1 ? exact_few_rows<KIND, 1>(ctx, p) : p.parts == 2 ? exact_few_rows<KIND, 2>(ctx, p) : exact_few_rows<KIND, 3>(ctx, p);
    if (int rc = exact_row_tiles<KIND>(ctx, p, &p.t_tiles)) return rc;
    const uint32_t rows = rows_of_tiles(p.T, p.t_tiles);
    if (rows <= 128) return exact_pair_rows<KIND, 2>(ctx, p);
    if (rows <= 192) return exact_pair_rows<KIND, 3>(ctx, p);
    return exact_pair_rows<KIND, 4>(ctx, p);
}

}  // namespace

// Takes K a multiple of 128, w 16-byte aligned, x 8-byte aligned; with `glu`, a multiple of 16 result columns.
int launch_matmul_tc(yx_ctx *ctx, const float *x, const void *w, uint32_t T, uint32_t N, uint32_t K, bool glu, float *out) {
    Product p{};
    p.x = x;
    p.w = w;
    p.T = T;
    p.N = N;
    p.K = K;
    p.parts = 2;
    p.out = out;
    return glu ? matmul_tc<GLU>(ctx, p) : matmul_tc<PLAIN>(ctx, p);
}

bool exact_tc_takes(const Product &p) { return p.K % 8 == 0 && ((uintptr_t)p.w & 15u) == 0; }
bool exact_tc_copies_rows(const Product &p) { return p.T > ROWS_MAX && (p.parts > 1 || ((uintptr_t)p.x & 15u) != 0); }
bool exact_tc_reads_rows_late(const Product &p) { return p.T <= ROWS_MAX || p.parts == 1; }
// (lower tiles are at most as many more as complete a round of SMs)
uint32_t most_logprob_blocks(yx_ctx *ctx, const Product &p) { return 2 * ((p.N + TC_M - 1) / TC_M) + (uint32_t)ctx->sm_count; }
int launch_matmul_epilogue_tc(yx_ctx *ctx, Product &p) { return exact_tc<EPILOGUE>(ctx, p); }
int launch_matmul_logprobs_tc(yx_ctx *ctx, Product &p) { return exact_tc<LOGPROBS>(ctx, p); }

}  // namespace yx
