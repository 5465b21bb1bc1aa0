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
#include "mbx_device.cuh"
#include "mbx_internal.h"

namespace mbx {
namespace {

constexpr int kMeanThreads = 256;

struct MeanSide {
    const void* x;
    int64_t x_stride, rows;    // elements between rows; rows of an item
    int block, blocks;         // rows of a block, blocks of an item
    int chunks, cols, groups;  // 8-channel chunks of a row; those of one CTA; CTAs of a block
    const uint8_t* mask;       // [n][rows] or null
    double* mean;              // [n][blocks][chunks · 8]
    uint8_t* live;             // [n][blocks]: 1 where a row was unmasked (null: not wanted)
};

struct MeanArgs {
    MeanSide side[2];  // q, k
    int64_t first_k;   // CTAs before this one are q's
};

template <class T>
__global__ void __launch_bounds__(kMeanThreads) block_means_kernel(const __grid_constant__ MeanArgs args) {
    __shared__ double part[kMeanThreads * 8];
    __shared__ int count;
    const bool is_k = blockIdx.x >= args.first_k;
    const MeanSide& a = args.side[is_k];
    const int64_t cta = blockIdx.x - (is_k ? args.first_k : 0);
    const int group = (int)(cta % a.groups);
    const int64_t at = cta / a.groups;  // item · blocks + block
    const int64_t item = at / a.blocks, r0 = (at - item * a.blocks) * a.block;
    const int rows = (int)min((int64_t)a.block, a.rows - r0);
    const int lanes = kMeanThreads / a.cols, rl = threadIdx.x / a.cols, col = threadIdx.x - rl * a.cols;
    const int chunk = group * a.cols + col;
    const bool on = rl < lanes && chunk < a.chunks;
    const T* x = static_cast<const T*>(a.x) + (item * a.rows + r0) * a.x_stride + (int64_t)chunk * 8;
    const uint8_t* mask = a.mask ? a.mask + item * a.rows + r0 : nullptr;
    if (threadIdx.x == 0) count = 0;
    __syncthreads();
    double sum[8] = {};
    if (on) {
        constexpr int U = sizeof(T) == 2 ? 8 : 4;  // rows in flight
        typename Raw8<T>::type raw[U];
        for (int r = rl; r < rows; r += U * lanes) {
            bool keep[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int ru = r + u * lanes;
                keep[u] = ru < rows && (!mask || mask[ru]);
                if (keep[u]) raw[u] = load_raw8(x + ru * a.x_stride);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (!keep[u]) continue;
                float v[8];
                widen8<T>(raw[u], v);
#pragma unroll
                for (int i = 0; i < 8; ++i) sum[i] += (double)v[i];
            }
        }
    }
    if (mask) {
        for (int r = threadIdx.x; r < rows; r += kMeanThreads)
            if (mask[r]) atomicAdd(&count, 1);
    } else if (threadIdx.x == 0) {
        count = rows;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) part[i * kMeanThreads + threadIdx.x] = sum[i];
    __syncthreads();
    const int n = count;
    for (int e = threadIdx.x; e < a.cols * 8; e += kMeanThreads) {
        const int c = e >> 3, i = e & 7;
        double s = 0.0;
        for (int w = 0; w < lanes; ++w) s += part[i * kMeanThreads + w * a.cols + c];
        if (group * a.cols + c < a.chunks)
            a.mean[(at * a.chunks + group * a.cols + c) * 8 + i] = s / (double)max(n, 1);
    }
    if (a.live && group == 0 && threadIdx.x == 0) a.live[at] = n > 0;
}

// An integer that orders as the score does: 0 for a block without an unmasked key (never chosen), then −inf … +inf,
// NaN above all; −0 is +0.
__device__ __forceinline__ uint64_t order_key(double s, bool live) {
    if (!live) return 0;
    if (isnan(s)) return ~0ull;
    const int64_t b = __double_as_longlong(s + 0.0);
    return b < 0 ? ~(uint64_t)b : (uint64_t)b | (1ull << 63);
}

// keys[b][h][i][j] for a TI × TJ tile; 64 threads of (TI / 8) × (TJ / 8) outputs, kSK channels a step. The
// wide tile gives 64 products for 16 values read from shared memory, which is what f64 arithmetic needs to
// run at its rate; the narrow one spreads a small problem over more CTAs.
constexpr int kSK = 16;

struct ScoreArgs {
    const double *qm, *km;  // [n][q_blocks][heads][dim], [n][k_blocks][kv_heads][dim]
    const uint8_t* live;    // [n][k_blocks]
    uint64_t* key;          // [n][heads][q_blocks][k_blocks]
    int heads, kv_heads, dim, q_blocks, k_blocks;
};

template <int TI, int TJ>
__global__ void __launch_bounds__(64) block_scores_kernel(const ScoreArgs a) {
    constexpr int RI = TI / 8, RJ = TJ / 8;
    __shared__ double qs[2][kSK][TI + 1], ks[2][kSK][TJ + 1];
    const int64_t item = blockIdx.z / a.heads;
    const int h = blockIdx.z % a.heads, kh = h / (a.heads / a.kv_heads);
    const int i0 = blockIdx.y * TI, j0 = blockIdx.x * TJ;
    const int tr = threadIdx.x / 8, tc = threadIdx.x % 8;
    // A thread brings channel lc of rows lr, lr + 4, … of a step.
    const int lc = threadIdx.x % kSK, lr = threadIdx.x / kSK;
    const double* q = a.qm + (item * a.q_blocks * a.heads + h) * a.dim + lc;
    const double* k = a.km + (item * a.k_blocks * a.kv_heads + kh) * a.dim + lc;
    const int64_t q_row = (int64_t)a.heads * a.dim, k_row = (int64_t)a.kv_heads * a.dim;
    double qr[TI / 4], kr[TJ / 4];
    auto fetch = [&](int c0) {
        const bool in = c0 + lc < a.dim;
#pragma unroll
        for (int r = 0; r < TI / 4; ++r) {
            const int i = i0 + lr + 4 * r;
            qr[r] = in && i < a.q_blocks ? q[i * q_row + c0] : 0.0;
        }
#pragma unroll
        for (int r = 0; r < TJ / 4; ++r) {
            const int j = j0 + lr + 4 * r;
            kr[r] = in && j < a.k_blocks ? k[j * k_row + c0] : 0.0;
        }
    };
    double acc[RI][RJ] = {};
    fetch(0);
    for (int c0 = 0, b = 0; c0 < a.dim; c0 += kSK, b ^= 1) {
#pragma unroll
        for (int r = 0; r < TI / 4; ++r) qs[b][lc][lr + 4 * r] = qr[r];
#pragma unroll
        for (int r = 0; r < TJ / 4; ++r) ks[b][lc][lr + 4 * r] = kr[r];
        __syncthreads();
        if (c0 + kSK < a.dim) fetch(c0 + kSK);
#pragma unroll
        for (int c = 0; c < kSK; ++c) {
            double qv[RI], kv[RJ];
#pragma unroll
            for (int r = 0; r < RI; ++r) qv[r] = qs[b][c][tr + 8 * r];
#pragma unroll
            for (int s = 0; s < RJ; ++s) kv[s] = ks[b][c][tc + 8 * s];
#pragma unroll
            for (int r = 0; r < RI; ++r)
#pragma unroll
                for (int s = 0; s < RJ; ++s) acc[r][s] = fma(qv[r], kv[s], acc[r][s]);
        }
    }
#pragma unroll
    for (int s = 0; s < RJ; ++s) {
        const int j = j0 + tc + 8 * s;
        if (j >= a.k_blocks) continue;
        const bool live = a.live[item * a.k_blocks + j] != 0;
#pragma unroll
        for (int r = 0; r < RI; ++r) {
            const int i = i0 + tr + 8 * r;
            if (i < a.q_blocks) a.key[((int64_t)blockIdx.z * a.q_blocks + i) * a.k_blocks + j] = order_key(acc[r][s], live);
        }
    }
}

constexpr int kTopWarps = 4;

// The K-th largest of a row's keys by bisection on their bits. N > 0: the row's k_blocks <= 32 · N keys stay in
// registers; N = 0: any number, read again for every count.
template <int N>
__global__ void __launch_bounds__(kTopWarps * 32) block_topk_kernel(const uint64_t* __restrict__ keys, int64_t rows,
                                                                    int k_blocks, int64_t topk,
                                                                    int32_t* __restrict__ index) {
    const int64_t row = blockIdx.x * (int64_t)kTopWarps + (threadIdx.x >> 5);
    if (row >= rows) return;
    const int lane = threadIdx.x & 31;
    const uint64_t* s = keys + row * k_blocks;
    uint64_t mine[N > 0 ? N : 1];
#pragma unroll
    for (int u = 0; u < N; ++u) mine[u] = u * 32 + lane < k_blocks ? s[u * 32 + lane] : 0;
    auto count_at_least = [&](uint64_t t) {
        int c = 0;
        if constexpr (N > 0) {
#pragma unroll
            for (int u = 0; u < N; ++u) c += mine[u] >= t;
        } else {
            for (int j = lane; j < k_blocks; j += 32) c += s[j] >= t;
        }
        return __reduce_add_sync(0xffffffffu, c);
    };
    const int k = (int)min(topk, (int64_t)count_at_least(1));
    // lo: the largest threshold known to leave k keys or more; at hi there are fewer.
    uint64_t lo = 1, hi = ~0ull;
    int at_least = k == 0 ? 0 : count_at_least(lo);
    if (k > 0 && count_at_least(hi) >= k) lo = hi, at_least = count_at_least(lo);
    if (at_least > k && lo != hi) {
        // Narrow the range to the keys' own before halving it: scores share their leading bits.
        uint64_t top = 0, low = ~0ull;
        auto see = [&](uint64_t v) {
            if (v == 0) return;
            top = max(top, v), low = min(low, v);
        };
        if constexpr (N > 0) {
#pragma unroll
            for (int u = 0; u < N; ++u) see(mine[u]);
        } else {
            for (int j = lane; j < k_blocks; j += 32) see(s[j]);
        }
        for (int o = 16; o > 0; o >>= 1) {
            top = max(top, (uint64_t)__shfl_xor_sync(0xffffffffu, top, o));
            low = min(low, (uint64_t)__shfl_xor_sync(0xffffffffu, low, o));
        }
        lo = low, hi = top == ~0ull ? top : top + 1;
        while (at_least != k && hi - lo > 1) {
            const uint64_t mid = lo + (hi - lo) / 2;
            const int c = count_at_least(mid);
            if (c >= k)
                lo = mid, at_least = c;
            else
                hi = mid;
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
void launch_means(mbx_ctx* ctx, const MeanArgs& a, int64_t ctas) {
    block_means_kernel<T><<<(unsigned)ctas, kMeanThreads, 0, ctx->stream>>>(a);
    after_launch(ctx, "block_means");
}

MeanSide mean_side(const void* x, int64_t stride, int64_t rows, int block, int blocks, int64_t width,
                   const uint8_t* mask, double* mean, uint8_t* live) {
    MeanSide m{x, stride, rows, block, blocks, (int)(width / 8), 0, 0, mask, mean, live};
    // At most 64 chunks a CTA (a KB of a 16-bit row), evenly: no group of few leftovers.
    m.groups = (m.chunks + 63) / 64;
    m.cols = (m.chunks + m.groups - 1) / m.groups;
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
    block_topk_kernel<N><<<(unsigned)((rows + kTopWarps - 1) / kTopWarps), kTopWarps * 32, 0, ctx->stream>>>(
        keys, rows, kb, topk, index);
    after_launch(ctx, "block_topk");
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
        m.side[0] = mean_side(q, q_stride, s.nq, MBX_ATTENTION_BLOCK_Q, qb, s.heads * s.dim, nullptr,
                              reinterpret_cast<double*>(ws + l.qm), nullptr);
        m.side[1] = mean_side(k, k_stride, s.nk, (int)s.block_k, kb, s.kv_heads * s.dim, key_mask,
                              reinterpret_cast<double*>(ws + l.km), ws + l.live);
        m.first_k = s.n * qb * m.side[0].groups;
        const int64_t ctas = m.first_k + s.n * kb * m.side[1].groups;
        MBX_REQUIRE(ctas < (int64_t(1) << 31), "block_select: too many blocks");
        if (s.dtype == MBX_DTYPE_F32)
            launch_means<float>(ctx, m, ctas);
        else if (s.dtype == MBX_DTYPE_F16)
            launch_means<__half>(ctx, m, ctas);
        else
            launch_means<__nv_bfloat16>(ctx, m, ctas);
        ScoreArgs sc{m.side[0].mean, m.side[1].mean, ws + l.live, keys, (int)s.heads, (int)s.kv_heads, (int)s.dim, qb,
                     kb};
        const unsigned z = (unsigned)(s.n * s.heads);
        if ((int64_t)z * ((qb + 63) / 64) * ((kb + 63) / 64) >= 4 * (int64_t)ctx->sm_count)
            block_scores_kernel<64, 64><<<dim3((kb + 63) / 64, (qb + 63) / 64, z), 64, 0, ctx->stream>>>(sc);
        else
            block_scores_kernel<32, 32><<<dim3((kb + 31) / 32, (qb + 31) / 32, z), 64, 0, ctx->stream>>>(sc);
        after_launch(ctx, "block_scores");
    }
    const int64_t rows = s.n * s.heads * qb;
    if (kb <= 64) return launch_topk<2>(ctx, keys, rows, kb, topk, index);
    if (kb <= 256) return launch_topk<8>(ctx, keys, rows, kb, topk, index);
    if (kb <= 1024) return launch_topk<32>(ctx, keys, rows, kb, topk, index);
    launch_topk<0>(ctx, keys, rows, kb, topk, index);
}

}  // namespace mbx
