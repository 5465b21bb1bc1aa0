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
//  * block_means: one pass over q and k (the bytes that bound the whole
//    operator at ordinary sizes). A warp reads 32 lanes × 8 channels of a row,
//    eight warps share a block's rows, and shared memory joins their sums in
//    a fixed order.
//  * block_scores: a tiled f64 product of the means, per (item, head).
//  * block_topk: the keys of one row of scores, as order-preserving integers;
//    the topk-th largest is found bit by bit, counting the keys at or above a
//    candidate, and the survivors are written by prefix counts.
#include "mbx_device.cuh"
#include "mbx_internal.h"

namespace mbx {
namespace {

constexpr int kMeanWarps = 8;

struct MeanArgs {
    const void* x;
    int64_t x_stride, rows;  // elements between rows; rows of an item
    int block, blocks, chunks;  // rows of a block, blocks of an item, 8-channel chunks of a row
    const uint8_t* mask;     // [n][rows] or null
    double* mean;            // [n][blocks][chunks * 8]
    uint8_t* live;           // [n][blocks]: 1 where a row was unmasked (null: not wanted)
};

template <class T>
__global__ void __launch_bounds__(kMeanWarps * 32) block_means_kernel(const MeanArgs a) {
    __shared__ double part[kMeanWarps][32][9];
    __shared__ int counts[kMeanWarps];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t item = blockIdx.z, blk = blockIdx.x;
    const int chunk = blockIdx.y * 32 + lane;
    const int64_t r0 = blk * a.block;
    const int rows = (int)min((int64_t)a.block, a.rows - r0);
    const T* x = static_cast<const T*>(a.x) + (item * a.rows + r0) * a.x_stride + (int64_t)chunk * 8;
    const uint8_t* mask = a.mask ? a.mask + item * a.rows + r0 : nullptr;
    double sum[8] = {};
    int count = 0;
#pragma unroll 4
    for (int r = warp; r < rows; r += kMeanWarps) {
        const bool keep = !mask || mask[r];
        count += keep;
        if (keep && chunk < a.chunks) {
            float v[8];
            widen8<T>(load_raw8(x + r * a.x_stride), v);
#pragma unroll
            for (int i = 0; i < 8; ++i) sum[i] += (double)v[i];
        }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) part[warp][lane][i] = sum[i];
    if (lane == 0) counts[warp] = count;
    __syncthreads();
    count = 0;
    for (int w = 0; w < kMeanWarps; ++w) count += counts[w];
    // 256 sums of 8 parts: thread → (lane's chunk, channel).
    const int cl = threadIdx.x >> 3, i = threadIdx.x & 7;
    double s = 0.0;
    for (int w = 0; w < kMeanWarps; ++w) s += part[w][cl][i];
    if (blockIdx.y * 32 + cl < a.chunks)
        a.mean[((item * a.blocks + blk) * a.chunks + blockIdx.y * 32 + cl) * 8 + i] = s / (double)max(count, 1);
    if (a.live && blockIdx.y == 0 && threadIdx.x == 0) a.live[item * a.blocks + blk] = count > 0;
}

// scores[b][h][i][j] for a 64 × 64 tile; 16 × 16 threads of 4 × 4 outputs, 16 channels of K a step.
constexpr int kST = 64, kSK = 16;

struct ScoreArgs {
    const double *qm, *km;  // [n][q_blocks][heads][dim], [n][k_blocks][kv_heads][dim]
    double* score;          // [n][heads][q_blocks][k_blocks]
    int heads, kv_heads, dim, q_blocks, k_blocks;
};

__global__ void __launch_bounds__(256) block_scores_kernel(const ScoreArgs a) {
    __shared__ double qs[kSK][kST + 1], ks[kSK][kST + 1];
    const int64_t item = blockIdx.z / a.heads;
    const int h = blockIdx.z % a.heads, kh = h / (a.heads / a.kv_heads);
    const int i0 = blockIdx.y * kST, j0 = blockIdx.x * kST;
    const int tr = threadIdx.x / 16, tc = threadIdx.x % 16;
    double acc[4][4] = {};
    for (int c0 = 0; c0 < a.dim; c0 += kSK) {
        for (int e = threadIdx.x; e < kST * kSK; e += 256) {
            const int r = e / kSK, c = e % kSK;
            const bool in = c0 + c < a.dim;
            qs[c][r] = in && i0 + r < a.q_blocks
                           ? a.qm[((item * a.q_blocks + i0 + r) * a.heads + h) * a.dim + c0 + c] : 0.0;
            ks[c][r] = in && j0 + r < a.k_blocks
                           ? a.km[((item * a.k_blocks + j0 + r) * a.kv_heads + kh) * a.dim + c0 + c] : 0.0;
        }
        __syncthreads();
#pragma unroll
        for (int c = 0; c < kSK; ++c) {
            double qv[4], kv[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) qv[r] = qs[c][tr + 16 * r], kv[r] = ks[c][tc + 16 * r];
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int s = 0; s < 4; ++s) acc[r][s] = fma(qv[r], kv[s], acc[r][s]);
        }
        __syncthreads();
    }
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const int i = i0 + tr + 16 * r, j = j0 + tc + 16 * s;
            if (i < a.q_blocks && j < a.k_blocks)
                a.score[(((int64_t)blockIdx.z) * a.q_blocks + i) * a.k_blocks + j] = acc[r][s];
        }
}

// An integer that orders as the score does: 0 for a block without an unmasked key (never chosen), then −inf … +inf,
// NaN above all; −0 is +0.
__device__ __forceinline__ uint64_t order_key(double s, bool live) {
    if (!live) return 0;
    if (isnan(s)) return ~0ull;
    const int64_t b = __double_as_longlong(s + 0.0);
    return b < 0 ? ~(uint64_t)b : (uint64_t)b | (1ull << 63);
}

constexpr int kTopThreads = 128;

__global__ void __launch_bounds__(kTopThreads) block_topk_kernel(const double* __restrict__ score,
                                                                 const uint8_t* __restrict__ live, int64_t rows_item,
                                                                 int k_blocks, int64_t topk,
                                                                 int32_t* __restrict__ index) {
    __shared__ int red[kTopThreads / 32];
    const int64_t row = blockIdx.x;
    const double* s = score + row * k_blocks;
    const uint8_t* lv = live + row / rows_item * k_blocks;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    auto count_at_least = [&](uint64_t t) {  // keys >= t, the same in every thread
        int c = 0;
        for (int j = threadIdx.x; j < k_blocks; j += kTopThreads) c += order_key(s[j], lv[j]) >= t;
        c = __reduce_add_sync(0xffffffffu, c);
        __syncthreads();
        if (lane == 0) red[warp] = c;
        __syncthreads();
        c = 0;
        for (int w = 0; w < kTopThreads / 32; ++w) c += red[w];
        return c;
    };
    const int all = count_at_least(1);
    const int k = (int)min(topk, (int64_t)all);
    // The largest threshold that k keys reach; 0 keys (k = 0) leave it at the top.
    uint64_t t = k == 0 ? ~0ull : 0;
    for (int bit = 63; bit >= 0 && k > 0; --bit) {
        const uint64_t c = t | (1ull << bit);
        const int n = count_at_least(c);
        if (n >= k) t = c;
        if (n == k) break;
    }
    const int at_least = k == 0 ? 0 : count_at_least(t);
    const int above = at_least == k ? k : (t == ~0ull ? 0 : count_at_least(t + 1));
    const int ties = k - (at_least == k ? at_least : above);  // keys equal to t to take, lowest block first
    int32_t* out = index + row * topk;
    if (warp == 0 && k > 0) {
        int done = 0, tied = 0;
        for (int j0 = 0; j0 < k_blocks; j0 += 32) {
            const int j = j0 + lane;
            const uint64_t key = j < k_blocks ? order_key(s[j], lv[j]) : 0;
            bool take = at_least == k ? key >= t : key > t;
            const bool tie = at_least != k && key == t && j < k_blocks;
            const unsigned tm = __ballot_sync(0xffffffffu, tie);
            if (tie) take = tied + __popc(tm & ((1u << lane) - 1)) < ties;
            tied += __popc(tm);
            const unsigned m = __ballot_sync(0xffffffffu, take);
            if (take) out[done + __popc(m & ((1u << lane) - 1))] = j;
            done += __popc(m);
        }
    }
    for (int64_t e = k + threadIdx.x; e < topk; e += kTopThreads) out[e] = -1;
}

template <class T>
void launch_means(mbx_ctx* ctx, const MeanArgs& a, int64_t n) {
    const dim3 grid((unsigned)a.blocks, (unsigned)((a.chunks + 31) / 32), (unsigned)n);
    block_means_kernel<T><<<grid, kMeanWarps * 32, 0, ctx->stream>>>(a);
    after_launch(ctx, "block_means");
}

void launch_means_any(mbx_ctx* ctx, int dtype, const MeanArgs& a, int64_t n) {
    if (dtype == MBX_DTYPE_F32) return launch_means<float>(ctx, a, n);
    if (dtype == MBX_DTYPE_F16) return launch_means<__half>(ctx, a, n);
    launch_means<__nv_bfloat16>(ctx, a, n);
}

struct SelectLayout {
    size_t qm, km, score, live, total;
};

SelectLayout select_layout(const BlockShape& s) {
    const size_t qb = (s.nq + MBX_ATTENTION_BLOCK_Q - 1) / MBX_ATTENTION_BLOCK_Q;
    const size_t kb = (s.nk + s.block_k - 1) / s.block_k;
    SelectLayout l;
    l.qm = 0;
    l.km = l.qm + align256(8 * (size_t)s.n * qb * s.heads * s.dim);
    l.score = l.km + align256(8 * (size_t)s.n * kb * s.kv_heads * s.dim);
    l.live = l.score + align256(8 * (size_t)s.n * s.heads * qb * kb);
    l.total = l.live + align256((size_t)s.n * kb);
    return l;
}

}  // namespace

size_t block_select_bytes(const BlockShape& s) { return select_layout(s).total; }

void launch_block_select(mbx_ctx* ctx, const BlockShape& s, const void* q, int64_t q_stride, const void* k,
                         int64_t k_stride, const uint8_t* key_mask, int64_t topk, int32_t* index, void* workspace) {
    const SelectLayout l = select_layout(s);
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    const int qb = (int)((s.nq + MBX_ATTENTION_BLOCK_Q - 1) / MBX_ATTENTION_BLOCK_Q);
    const int kb = (int)((s.nk + s.block_k - 1) / s.block_k);
    if (kb > 0) {
        MeanArgs mq{q, q_stride, s.nq, MBX_ATTENTION_BLOCK_Q, qb, (int)(s.heads * s.dim / 8), nullptr,
                    reinterpret_cast<double*>(ws + l.qm), nullptr};
        launch_means_any(ctx, s.dtype, mq, s.n);
        MeanArgs mk{k, k_stride, s.nk, (int)s.block_k, kb, (int)(s.kv_heads * s.dim / 8), key_mask,
                    reinterpret_cast<double*>(ws + l.km), ws + l.live};
        launch_means_any(ctx, s.dtype, mk, s.n);
        ScoreArgs sc{mq.mean, mk.mean, reinterpret_cast<double*>(ws + l.score), (int)s.heads, (int)s.kv_heads,
                     (int)s.dim, qb, kb};
        const dim3 grid((unsigned)((kb + kST - 1) / kST), (unsigned)((qb + kST - 1) / kST),
                        (unsigned)(s.n * s.heads));
        block_scores_kernel<<<grid, 256, 0, ctx->stream>>>(sc);
        after_launch(ctx, "block_scores");
    }
    block_topk_kernel<<<(unsigned)(s.n * s.heads * qb), kTopThreads, 0, ctx->stream>>>(
        reinterpret_cast<const double*>(ws + l.score), ws + l.live, s.heads * qb, kb, topk, index);
    after_launch(ctx, "block_topk");
}

}  // namespace mbx
