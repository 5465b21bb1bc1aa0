// Key blocks for each query block, by a cheap score.
//
//   score[b, h, i, j] = mean over the rows of query block i of q[b, ·, h]
//                     · mean over the unmasked keys of block j of k[b, ·, h / group]
// and per (b, h, i) the `topk` blocks of the highest score among those with an
// unmasked key, a tie going to the lower block; they are written in ascending
// order with −1 behind them.
//
// A choice is discontinuous: two scores that differ in the last bits of an f32
// sum would be ordered by the order of that sum. So means and scores are f64
// throughout, which the storage types' values enter exactly.
//
// Three kernels:
//  * block_means: one pass over q and k, the bytes that the operator cannot do
//    without. A thread adds eight channels of every R-th row of a block, and
//    shared memory joins the R sums in a fixed order.
//  * block_scores: a tiled f64 product of the means, per (item, head), written
//    as integers that order as the scores do.
//  * block_topk: a warp per row of scores, its keys in registers: the topk-th
//    largest is found by bisection, counting the keys at or above a candidate,
//    and the survivors are written by prefix counts.
// Measured on a B200: 65536 queries x 16 heads, 65536 keys x 8 x 128 bf16, 64 of 1024 blocks: 187 us, the means
// 73 (5.5 TB/s), the scores 82 (77 % of the f64 tensor rate), the choice 34; 16 x 4096 x 8 x 40 f16: 31 us.
#include <algorithm>

#include "mbx_device.cuh"
#include "mbx_internal.h"

namespace mbx {
namespace {

constexpr int kMeanThreads = 256;

struct MeanSide {
    const void* x;
    int64_t x_stride, rows;    // elements between rows; rows of an item
    int block, blocks;         // rows of a block, blocks of an item
    int width, cols, groups;   // channels of a row; 16-byte pieces of it a CTA takes; CTAs of a block
    const uint8_t* mask;       // [n][rows] or null
    double* mean;              // [n][blocks][width]
    uint8_t* live;             // [n][blocks]: 1 where a row was unmasked (null: not wanted)
};

struct MeanArgs {
    MeanSide side[2];  // q, k
};

// Grid: (blocks of q, then of k; groups of columns; items). A thread adds a 16-byte piece of every
// lanes-th row. It has a ring of kRing rows of its own in shared memory that cp.async fills, so that
// up to 32 KB a CTA are on their way with few registers and nobody waits for another thread: with
// register loads the conversions to f64 (an eighth of the f32 rate) and the loads took turns, at
// 4.1 TB/s. Rows that the mask hides, or past the last one, are filled with zeros.
constexpr int kRing = 8;

template <class T>
__global__ void __launch_bounds__(kMeanThreads, 5) block_means_kernel(const __grid_constant__ MeanArgs args) {
    cudaGridDependencySynchronize();
    constexpr int E = 16 / sizeof(T);  // channels of a piece
    __shared__ __align__(16) uint8_t ring[kRing * kMeanThreads * 16];
    __shared__ uint8_t keep[MBX_ATTENTION_BLOCK_Q];
    const bool is_k = (int)blockIdx.x >= args.side[0].blocks;
    const MeanSide& a = args.side[is_k];
    if ((int)blockIdx.y >= a.groups) return;
    const int blk = (int)blockIdx.x - (is_k ? args.side[0].blocks : 0);
    const int64_t item = blockIdx.z, r0 = (int64_t)blk * a.block, at = item * a.blocks + blk;
    const int rows = (int)min((int64_t)a.block, a.rows - r0);
    const int lanes = kMeanThreads / a.cols, rl = threadIdx.x / a.cols, col = threadIdx.x - rl * a.cols;
    const int ch = (blockIdx.y * a.cols + col) * E;  // first channel
    int count = rows;
    if (a.mask) {
        const uint8_t m = (int)threadIdx.x < rows ? a.mask[item * a.rows + r0 + threadIdx.x] : 0;
        if (threadIdx.x < MBX_ATTENTION_BLOCK_Q) keep[threadIdx.x] = m;
        count = __syncthreads_count(m != 0);
    }
    const T* next = static_cast<const T*>(a.x) + (item * a.rows + r0 + rl) * a.x_stride + ch;  // to be requested
    const int64_t step = lanes * a.x_stride;
    const uint32_t ring_at = (uint32_t)__cvta_generic_to_shared(ring) + threadIdx.x * 16;
    const int mine = rl < lanes && ch < a.width ? (rows - rl + lanes - 1) / lanes : 0;  // rows of this thread
    const bool masked = a.mask != nullptr;
    auto request = [&](int i, int slot) {  // the i-th of them
        if (i < mine) {
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(ring_at + slot * (kMeanThreads * 16)),
                         "l"(next), "r"(masked && !keep[rl + i * lanes] ? 0 : 16)
                         : "memory");
            next += step;
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    double sum[E] = {};
#pragma unroll
    for (int i = 0; i < kRing; ++i) request(i, i);
    for (int i0 = 0; i0 < mine; i0 += kRing) {
#pragma unroll
        for (int slot = 0; slot < kRing; ++slot) {
            if (i0 + slot >= mine) break;
            asm volatile("cp.async.wait_group %0;" ::"n"(kRing - 1) : "memory");
            uint4 raw;
            asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                         : "=r"(raw.x), "=r"(raw.y), "=r"(raw.z), "=r"(raw.w)
                         : "r"(ring_at + slot * (kMeanThreads * 16))
                         : "memory");
            float v[E];
            if constexpr (E == 8) {
                widen8<T>(raw, v);
            } else {
                v[0] = __uint_as_float(raw.x), v[1] = __uint_as_float(raw.y);
                v[2] = __uint_as_float(raw.z), v[3] = __uint_as_float(raw.w);
            }
            request(i0 + slot + kRing, slot);
#pragma unroll
            for (int c = 0; c < E; ++c) sum[c] += (double)v[c];
        }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();
    double* part = reinterpret_cast<double*>(ring);  // at most 16 KB of its 32
#pragma unroll
    for (int i = 0; i < E; ++i) part[i * kMeanThreads + threadIdx.x] = sum[i];
    __syncthreads();
    for (int e = threadIdx.x; e < a.cols * E; e += kMeanThreads) {
        const int c = e / E, i = e % E, to = (blockIdx.y * a.cols + c) * E + i;
        double s = 0.0;
        for (int w = 0; w < lanes; ++w) s += part[i * kMeanThreads + w * a.cols + c];
        if (to < a.width) a.mean[at * a.width + to] = s / (double)max(count, 1);
    }
    if (a.live && blockIdx.y == 0 && threadIdx.x == 0) a.live[at] = count > 0;
}

// An integer that orders as the score does: 0 for a block without an unmasked key (never chosen), then −inf … +inf,
// NaN above all; −0 is +0.
__device__ __forceinline__ uint64_t order_key(double s, bool live) {
    if (!live) return 0;
    if (isnan(s)) return ~0ull;
    const int64_t b = __double_as_longlong(s + 0.0);
    return b < 0 ? ~(uint64_t)b : (uint64_t)b | (1ull << 63);
}

// keys[b][h][i][j] for a 2·WI × 2·WJ tile, a WI × WJ part a warp, kSK channels a step. f64 products by mma.sync
// (m16n8k4; f64 has no tcgen05 kind): eight values a lane from shared memory for 4096 products of a 32 × 32
// part, where a 8 × 4 tile of plain FMAs reads 12 for 1024 and is bound by shared memory at 52 % of the f64 rate.
// The small tile spreads a small problem over more CTAs.
constexpr int kSK = 16, kScoreThreads = 128;

struct ScoreArgs {
    const double *qm, *km;  // [n][q_blocks][heads][dim], [n][k_blocks][kv_heads][dim]
    const uint8_t* live;    // [n][k_blocks]
    uint64_t* key;          // [n][heads][q_blocks][k_blocks]
    int heads, kv_heads, dim, q_blocks, k_blocks;
};

__device__ __forceinline__ void mma_f64(double (&c)[4], const double (&a)[2], double b) {
    asm("mma.sync.aligned.m16n8k4.row.col.f64.f64.f64.f64 {%0, %1, %2, %3}, {%4, %5}, {%6}, {%0, %1, %2, %3};"
        : "+d"(c[0]), "+d"(c[1]), "+d"(c[2]), "+d"(c[3])
        : "d"(a[0]), "d"(a[1]), "d"(b));
}

template <int WI, int WJ>
__global__ void __launch_bounds__(kScoreThreads, 4) block_scores_kernel(const ScoreArgs a) {
    constexpr int TI = 2 * WI, TJ = 2 * WJ, MI = WI / 16, NJ = WJ / 8;
    cudaGridDependencySynchronize();
    // 20 values a row of 16: four channels of four rows fall into different banks.
    constexpr int ROW = kSK + 4;
    __shared__ __align__(16) double qs[2][TI][ROW], ks[2][TJ][ROW];
    const int64_t item = blockIdx.z / a.heads;
    const int h = blockIdx.z % a.heads, kh = h / (a.heads / a.kv_heads);
    const int i0 = blockIdx.y * TI, j0 = blockIdx.x * TJ;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int wi = (warp >> 1) * WI, wj = (warp & 1) * WJ, lr4 = lane >> 2, lc4 = lane & 3;
    // A thread brings channels 2·lc, 2·lc + 1 of rows lr, lr + 16, … of a step; outside there are zeros.
    const int lc = threadIdx.x % 8 * 2, lr = threadIdx.x / 8;
    const double* q = a.qm + (item * a.q_blocks * a.heads + h) * a.dim + lc;
    const double* k = a.km + (item * a.k_blocks * a.kv_heads + kh) * a.dim + lc;
    const int64_t q_row = (int64_t)a.heads * a.dim, k_row = (int64_t)a.kv_heads * a.dim;
    auto copy = [](double* to, const double* from, bool in) {
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"((uint32_t)__cvta_generic_to_shared(to)),
                     "l"(from), "r"(in ? 16 : 0)
                     : "memory");
    };
    auto fetch = [&](int b, int c0) {
        const bool in = c0 + lc < a.dim;
#pragma unroll
        for (int r = 0; r < TI / 16; ++r) {
            const bool ok = in && i0 + lr + 16 * r < a.q_blocks;
            copy(&qs[b][lr + 16 * r][lc], ok ? q + (i0 + lr + 16 * r) * q_row + c0 : a.qm, ok);
        }
#pragma unroll
        for (int r = 0; r < TJ / 16; ++r) {
            const bool ok = in && j0 + lr + 16 * r < a.k_blocks;
            copy(&ks[b][lr + 16 * r][lc], ok ? k + (j0 + lr + 16 * r) * k_row + c0 : a.km, ok);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    double acc[MI][NJ][4] = {};
    fetch(0, 0);
    for (int c0 = 0, b = 0; c0 < a.dim; c0 += kSK, b ^= 1) {
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        __syncthreads();  // this step is there, and everybody is done with the one before it
        if (c0 + kSK < a.dim) fetch(b ^ 1, c0 + kSK);
#pragma unroll
        for (int c = 0; c < kSK; c += 4) {
            double qv[MI][2], kv[NJ];
#pragma unroll
            for (int r = 0; r < MI; ++r)
#pragma unroll
                for (int e = 0; e < 2; ++e) qv[r][e] = qs[b][wi + r * 16 + e * 8 + lr4][c + lc4];
#pragma unroll
            for (int s = 0; s < NJ; ++s) kv[s] = ks[b][wj + s * 8 + lr4][c + lc4];
#pragma unroll
            for (int r = 0; r < MI; ++r)
#pragma unroll
                for (int s = 0; s < NJ; ++s) mma_f64(acc[r][s], qv[r], kv[s]);
        }
    }
#pragma unroll
    for (int s = 0; s < NJ; ++s) {
        const int j = j0 + wj + s * 8 + lc4 * 2;
        bool live[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) live[e] = j + e < a.k_blocks && a.live[item * a.k_blocks + j + e] != 0;
#pragma unroll
        for (int r = 0; r < MI; ++r)
#pragma unroll
            for (int f = 0; f < 2; ++f) {
                const int i = i0 + wi + r * 16 + f * 8 + lr4;
                if (i >= a.q_blocks) continue;
                uint64_t* to = a.key + ((int64_t)blockIdx.z * a.q_blocks + i) * a.k_blocks + j;
#pragma unroll
                for (int e = 0; e < 2; ++e)
                    if (j + e < a.k_blocks) to[e] = order_key(acc[r][s][2 * f + e], live[e]);
            }
    }
}

__device__ __forceinline__ double key_score(uint64_t key) {
    return __longlong_as_double((int64_t)(key >> 63 ? key & ~(1ull << 63) : ~key));
}

constexpr int kTopWarps = 4;

// The K-th largest of a row's keys by bisection on their bits. N > 0: the row's k_blocks <= 32 · N keys stay in
// registers; N = 0: any number, read again for every count.
template <int N>
__global__ void __launch_bounds__(kTopWarps * 32) block_topk_kernel(const uint64_t* __restrict__ keys, int64_t rows,
                                                                    int k_blocks, int64_t topk,
                                                                    int32_t* __restrict__ index) {
    cudaGridDependencySynchronize();
    const int64_t row = blockIdx.x * (int64_t)kTopWarps + (threadIdx.x >> 5);
    if (row >= rows) return;
    const int lane = threadIdx.x & 31;
    const uint64_t* s = keys + row * k_blocks;
    uint64_t mine[N > 0 ? N : 1];
#pragma unroll
    for (int u = 0; u < N; ++u) mine[u] = u * 32 + lane < k_blocks ? s[u * 32 + lane] : 0;
    auto for_each = [&](auto&& f) {
        if constexpr (N > 0) {
#pragma unroll
            for (int u = 0; u < N; ++u) f(mine[u]);
        } else {
            for (int j = lane; j < k_blocks; j += 32) f(s[j]);
        }
    };
    auto count_at_least = [&](uint64_t t) {
        int c = 0;
        for_each([&](uint64_t v) { c += v >= t; });
        return __reduce_add_sync(0xffffffffu, c);
    };
    // The high words' range (of the blocks that count) and how many there are.
    uint32_t top = 0, low = ~0u;
    int live = 0;
    for_each([&](uint64_t v) {
        const uint32_t w = (uint32_t)(v >> 32);
        live += v != 0;
        top = max(top, w);
        if (v != 0) low = min(low, w);
    });
    live = __reduce_add_sync(0xffffffffu, live);
    top = __reduce_max_sync(0xffffffffu, top);
    low = __reduce_min_sync(0xffffffffu, low);
    const int k = (int)min(topk, (int64_t)live);
    // The largest threshold that k keys or more reach: on the high words, between the row's own extremes, and only
    // where several keys share the last high word on the low ones.
    uint64_t lo = 1;
    int at_least = live;
    if (k > 0 && live > k) {
        // Halving the scores' range finds the place among scores of one magnitude in few steps, where the integers'
        // range is mostly exponents that no score has; halving the integers' bounds the steps for any others.
        uint64_t a32 = low, b32 = (uint64_t)top + 1;
        for (int step = 0; at_least != k && b32 - a32 > 1; ++step) {
            uint64_t mid = a32 + (b32 - a32) / 2;
            if (step < 16) {
                const uint64_t m = order_key(0.5 * key_score(a32 << 32) + 0.5 * key_score(b32 << 32), true) >> 32;
                if (m > a32 && m < b32) mid = m;
            }
            int c = 0;
            for_each([&](uint64_t v) { c += (uint32_t)(v >> 32) >= (uint32_t)mid; });
            c = __reduce_add_sync(0xffffffffu, c);
            if (c >= k)
                a32 = mid, at_least = c;
            else
                b32 = mid;
        }
        lo = max(a32 << 32, (uint64_t)1);
        uint64_t span = 1ull << 32;
        while (at_least != k && span > 1) {
            span /= 2;
            const int c = count_at_least(lo + span);
            if (c >= k) lo += span, at_least = c;
        }
    }
    // Above lo: all of them; equal to lo: the lowest blocks, as many as are still wanted.
    const bool exact = at_least == k;
    int ties = 0;
    if (!exact) ties = k - (lo == ~0ull ? 0 : count_at_least(lo + 1));
    int32_t* out = index + row * topk;
    int done = 0, tied = 0;
    auto write = [&](int j0, uint64_t key) {
        bool take = k > 0 && (exact ? key >= lo : key > lo);
        const bool tie = !exact && key == lo;
        const unsigned before = (1u << lane) - 1;
        const unsigned tm = __ballot_sync(0xffffffffu, tie);
        if (tie) take = tied + __popc(tm & before) < ties;
        tied += __popc(tm);
        const unsigned m = __ballot_sync(0xffffffffu, take);
        if (take) out[done + __popc(m & before)] = j0 + lane;
        done += __popc(m);
    };
    if constexpr (N > 0) {
#pragma unroll
        for (int u = 0; u < N; ++u) write(u * 32, mine[u]);
    } else {
        for (int j0 = 0; j0 < k_blocks; j0 += 32) write(j0, j0 + lane < k_blocks ? s[j0 + lane] : 0);
    }
    for (int64_t e = k + lane; e < topk; e += 32) out[e] = -1;
}

template <class T>
void launch_means(mbx_ctx* ctx, const MeanArgs& a, int64_t n) {
    const dim3 grid((unsigned)(a.side[0].blocks + a.side[1].blocks),
                    (unsigned)std::max(a.side[0].groups, a.side[1].groups), (unsigned)n);
    launch_after(ctx, "block_means", block_means_kernel<T>, grid, kMeanThreads, 0, a);
}

MeanSide mean_side(const void* x, int dtype, int64_t stride, int64_t rows, int block, int blocks, int64_t width,
                   const uint8_t* mask, double* mean, uint8_t* live, int64_t n, int sms) {
    MeanSide m{x, stride, rows, block, blocks, (int)width, 0, 0, mask, mean, live};
    // 64 pieces (a KB) of a row for a CTA, evenly; 32 where that leaves fewer than four CTAs an SM. A CTA's fixed
    // costs want long columns (65536 x 16 x 128 bf16: 217 us in all with 32, 202 with 64, 200 with 128), a small
    // problem many CTAs (2 x 1961 and 4133 x 80 f32: 25 us with 32, 27 with 64, 34 with 128).
    const int pieces = (int)width / (dtype == MBX_DTYPE_F32 ? 4 : 8);
    const int most = n * blocks * ((pieces + 63) / 64) < 4 * sms ? 32 : 64;
    m.groups = (pieces + most - 1) / most;
    m.cols = (pieces + m.groups - 1) / m.groups;
    return m;
}

struct SelectLayout {
    size_t qm, km, key, live, total;
};

SelectLayout select_layout(const BlockShape& s) {
    const size_t qb = (s.nq + MBX_ATTENTION_BLOCK_Q - 1) / MBX_ATTENTION_BLOCK_Q;
    const size_t kb = (s.nk + s.block_k - 1) / s.block_k;
    SelectLayout l;
    l.qm = 0;
    l.km = l.qm + align256(8 * (size_t)s.n * qb * s.heads * s.dim);
    l.key = l.km + align256(8 * (size_t)s.n * kb * s.kv_heads * s.dim);
    l.live = l.key + align256(8 * (size_t)s.n * s.heads * qb * kb);
    l.total = l.live + align256((size_t)s.n * kb);
    return l;
}

template <int N>
void launch_topk(mbx_ctx* ctx, const uint64_t* keys, int64_t rows, int kb, int64_t topk, int32_t* index) {
    launch_after(ctx, "block_topk", block_topk_kernel<N>, dim3((unsigned)((rows + kTopWarps - 1) / kTopWarps)), kTopWarps * 32,
                 0, keys, rows, kb, topk, index);
}

}  // namespace

size_t block_select_bytes(const BlockShape& s) { return select_layout(s).total; }

void launch_block_select(mbx_ctx* ctx, const BlockShape& s, const void* q, int64_t q_stride, const void* k,
                         int64_t k_stride, const uint8_t* key_mask, int64_t topk, int32_t* index, void* workspace) {
    const SelectLayout l = select_layout(s);
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    const int qb = (int)((s.nq + MBX_ATTENTION_BLOCK_Q - 1) / MBX_ATTENTION_BLOCK_Q);
    const int kb = (int)((s.nk + s.block_k - 1) / s.block_k);
    uint64_t* keys = reinterpret_cast<uint64_t*>(ws + l.key);
    if (kb > 0) {
        MeanArgs m{};
        m.side[0] = mean_side(q, s.dtype, q_stride, s.nq, MBX_ATTENTION_BLOCK_Q, qb, s.heads * s.dim, nullptr,
                              reinterpret_cast<double*>(ws + l.qm), nullptr, s.n, ctx->sm_count);
        m.side[1] = mean_side(k, s.dtype, k_stride, s.nk, (int)s.block_k, kb, s.kv_heads * s.dim, key_mask,
                              reinterpret_cast<double*>(ws + l.km), ws + l.live, s.n, ctx->sm_count);
        if (s.dtype == MBX_DTYPE_F32)
            launch_means<float>(ctx, m, s.n);
        else if (s.dtype == MBX_DTYPE_F16)
            launch_means<__half>(ctx, m, s.n);
        else
            launch_means<__nv_bfloat16>(ctx, m, s.n);
        ScoreArgs sc{m.side[0].mean, m.side[1].mean, ws + l.live, keys, (int)s.heads, (int)s.kv_heads, (int)s.dim, qb,
                     kb};
        const unsigned z = (unsigned)(s.n * s.heads);
        if ((int64_t)z * ((qb + 63) / 64) * ((kb + 63) / 64) >= 4 * (int64_t)ctx->sm_count)
            launch_after(ctx, "block_scores", block_scores_kernel<32, 32>, dim3((kb + 63) / 64, (qb + 63) / 64, z), kScoreThreads,
                         0, sc);
        else
            launch_after(ctx, "block_scores", block_scores_kernel<16, 16>, dim3((kb + 31) / 32, (qb + 31) / 32, z), kScoreThreads,
                         0, sc);
    }
    const int64_t rows = s.n * s.heads * qb;
    if (kb <= 64) return launch_topk<2>(ctx, keys, rows, kb, topk, index);
    if (kb <= 256) return launch_topk<8>(ctx, keys, rows, kb, topk, index);
    if (kb <= 1024) return launch_topk<32>(ctx, keys, rows, kb, topk, index);
    launch_topk<0>(ctx, keys, rows, kb, topk, index);
}

}  // namespace mbx
