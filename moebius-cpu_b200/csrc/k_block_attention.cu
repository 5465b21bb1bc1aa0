// Softmax attention of query blocks over listed key blocks.
//
//   out[b, r, h] = Σ_j p_j v[b, j, h/g] / Σ_j p_j,  p_j = exp(scale · q[b, r, h]·k[b, j, h/g] − m)
// over the keys j of the blocks that index[b, h, r / 128] lists and that the
// key mask keeps; a row without any such key is zero.
//
// The rows kernel: one pass over the listed keys with a running maximum and sum (f32). A group of
// lanes holds one key's channels, eight a lane, so a warp works on several keys at a time; every
// group keeps its own maximum, sum and output for R query rows and the groups and warps are joined
// at the end. Where there are few rows the listed blocks are split over several CTAs, whose partial
// (output, maximum, sum) a second kernel joins.
#include <algorithm>

#include "block_attention.h"
#include "mbx_device.cuh"
#include "mbx_internal.h"

namespace mbx {
namespace {

constexpr int kRowWarps = 4;

// Lanes of a key's group: the power of two that holds dim / 8.
template <class T, int R>
__global__ void __launch_bounds__(kRowWarps * 32) attention_rows_kernel(const AttnArgs a, int group) {
    // One slot per (warp, group, row) and then the join: maxima, sums, outputs.
    extern __shared__ float sh[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int li = lane & (group - 1), gi = lane / group, groups = 32 / group;
    const int slots = kRowWarps * groups, slot = warp * groups + gi;
    const bool holds = li * 8 < a.dim;
    const int tiles = (int)((a.nq + R - 1) / R);
    const int64_t cta = blockIdx.x / a.splits;
    const int split = (int)(blockIdx.x - cta * a.splits);
    const int64_t r0 = cta % tiles * R;
    const int h = (int)(cta / tiles % a.heads);
    const int64_t item = cta / tiles / a.heads;
    const int kh = h / (a.heads / a.kv_heads);
    // A tile of R rows never straddles two query blocks: R divides 128.
    const int32_t* list = a.index + ((item * a.heads + h) * a.q_blocks + r0 / MBX_ATTENTION_BLOCK_Q) * a.topk;
    const T* q = static_cast<const T*>(a.q) + (item * a.nq + r0) * a.q_stride + (int64_t)h * a.dim + li * 8;
    const T* k = static_cast<const T*>(a.k) + item * a.nk * a.k_stride + (int64_t)kh * a.dim + li * 8;
    const T* v = static_cast<const T*>(a.v) + item * a.nk * a.v_stride + (int64_t)kh * a.dim + li * 8;
    const uint8_t* mask = a.mask ? a.mask + item * a.nk : nullptr;

    float qv[R][8], acc[R][8] = {}, m[R], l[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        m[r] = -INFINITY, l[r] = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) qv[r][i] = 0.0f;
        if (holds && r0 + r < a.nq) widen8<T>(load_raw8(q + r * a.q_stride), qv[r]);
#pragma unroll
        for (int i = 0; i < 8; ++i) qv[r][i] *= a.scale;
    }

    const int64_t first = a.topk * split / a.splits, last = a.topk * (split + 1) / a.splits;
    for (int64_t e = first; e < last; ++e) {
        const int blk = list[e];
        if (blk < 0 || blk >= a.k_blocks) continue;
        const int64_t j0 = (int64_t)blk * a.block_k;
        const int keys = (int)min((int64_t)a.block_k, a.nk - j0);
        for (int s = slot; s - gi - warp * groups < keys; s += slots) {  // the same trips in every lane of the block
            const int64_t j = j0 + s;
            const bool on = s < keys && (!mask || mask[j]);
            float kv[8] = {}, vv[8] = {};
            if (on && holds) {
                widen8<T>(load_raw8(k + j * a.k_stride), kv);
                widen8<T>(load_raw8(v + j * a.v_stride), vv);
            }
#pragma unroll
            for (int r = 0; r < R; ++r) {
                float d = 0.0f;
#pragma unroll
                for (int i = 0; i < 8; ++i) d = fmaf(qv[r][i], kv[i], d);
                for (int o = group >> 1; o > 0; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
                if (on && d != -INFINITY) {
                    const float mn = fmaxf(m[r], d);
                    const float c = exp2f(m[r] - mn), p = exp2f(d - mn);
                    m[r] = mn;
                    l[r] = l[r] * c + p;
#pragma unroll
                    for (int i = 0; i < 8; ++i) acc[r][i] = fmaf(acc[r][i], c, p * vv[i]);
                }
            }
        }
    }

    float* sm = sh;                  // [slots][R]
    float* sl = sm + slots * R;      // [slots][R]
    float* so = sl + slots * R;      // [slots][R][dim]
    if (li == 0) {
#pragma unroll
        for (int r = 0; r < R; ++r) sm[slot * R + r] = m[r], sl[slot * R + r] = l[r];
    }
    if (holds) {
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int i = 0; i < 8; ++i) so[(slot * R + r) * a.dim + li * 8 + i] = acc[r][i];
    }
    __syncthreads();
    for (int e = threadIdx.x; e < R * a.dim; e += kRowWarps * 32) {
        const int r = e / a.dim, ch = e - r * a.dim;
        if (r0 + r >= a.nq) continue;
        float top = -INFINITY;
        for (int s = 0; s < slots; ++s) top = fmaxf(top, sm[s * R + r]);
        float sum = 0.0f, o = 0.0f;
        for (int s = 0; s < slots; ++s) {
            const float ms = sm[s * R + r];
            const float w = ms == -INFINITY ? 0.0f : exp2f(ms - top);
            sum = fmaf(w, sl[s * R + r], sum);
            o = fmaf(w, so[(s * R + r) * a.dim + ch], o);
        }
        const int64_t row = (item * a.nq + r0 + r) * a.heads + h;
        if (a.splits == 1) {
            static_cast<T*>(a.out)[row * a.dim + ch] = (T)(sum == 0.0f ? 0.0f : o / sum);
        } else {
            float* p = a.part + (row * a.splits + split) * (a.dim + 4);
            p[ch] = o;
            if (ch == 0) p[a.dim] = top, p[a.dim + 1] = sum;
        }
    }
}

// Joins the splits' partial results: a CTA per (row, head). The splits' weights are worked out once in shared memory;
// then each warp adds every fourth split, a lane four channels, eight splits in flight.
constexpr int kMaxSplits = 64;

template <class T>
__global__ void __launch_bounds__(128) attention_join_kernel(const AttnArgs a) {
    __shared__ float weight[kMaxSplits];
    __shared__ float4 acc[4][32];
    __shared__ float total;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, stride = a.dim + 4;
    const float* p = a.part + (int64_t)blockIdx.x * a.splits * stride;
    if (warp == 0) {
        float m[2], l[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int s = lane + 32 * i;
            m[i] = s < a.splits ? p[s * stride + a.dim] : -INFINITY;
            l[i] = s < a.splits ? p[s * stride + a.dim + 1] : 0.0f;
        }
        float top = fmaxf(m[0], m[1]);
        for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const float w = m[i] == -INFINITY ? 0.0f : exp2f(m[i] - top);
            weight[lane + 32 * i] = w;
            sum = fmaf(w, l[i], sum);
        }
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane == 0) total = sum;
    }
    __syncthreads();
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (lane * 4 < a.dim) {
#pragma unroll 8
        for (int s = warp; s < a.splits; s += 4) {
            const float4 v = *reinterpret_cast<const float4*>(p + s * stride + lane * 4);
            const float w = weight[s];
            o = f4_fma(make_float4(w, w, w, w), v, o);
        }
    }
    acc[warp][lane] = o;
    __syncthreads();
    if ((int)threadIdx.x < a.dim) {
        const float* x = reinterpret_cast<const float*>(acc);
        const float y = (x[threadIdx.x] + x[128 + threadIdx.x]) + (x[256 + threadIdx.x] + x[384 + threadIdx.x]);
        static_cast<T*>(a.out)[(int64_t)blockIdx.x * a.dim + threadIdx.x] = (T)(total == 0.0f ? 0.0f : y / total);
    }
}

constexpr int kRowsR = 4;
constexpr int64_t kSms = 148;

// Which kernel takes a problem, and over how many CTAs a list is split: enough to fill the card
// twice over, never more than there are blocks (rows) or tiles of 64 keys (tensor cores).
struct Plan {
    bool rows;
    int splits;
    size_t part_bytes, split_bytes;
};

Plan plan_of(const BlockShape& s, int64_t topk) {
    Plan p{};
    p.rows = s.dtype == MBX_DTYPE_F32 && s.nq < 16;
    const int64_t tile = p.rows ? kRowsR : MBX_ATTENTION_BLOCK_Q;
    const int64_t ctas = std::max<int64_t>(1, s.n * s.heads * ((s.nq + tile - 1) / tile));
    const int64_t pieces = p.rows ? topk : (topk * s.block_k + 63) / 64;
    p.splits = (int)std::max<int64_t>(1, std::min({(2 * kSms + ctas - 1) / ctas, pieces, int64_t(kMaxSplits)}));
    if (p.splits > 1)
        p.part_bytes = align256(sizeof(float) * (size_t)(s.n * s.nq * s.heads) * p.splits * (s.dim + 4));
    if (!p.rows && s.dtype == MBX_DTYPE_F32) p.split_bytes = attention_split_bytes(s);
    return p;
}

template <class T>
void launch_rows(mbx_ctx* ctx, const AttnArgs& a, int64_t n) {
    int group = 1;
    while (group * 8 < a.dim) group *= 2;
    const int slots = kRowWarps * (32 / group);
    const size_t smem = sizeof(float) * (size_t)slots * kRowsR * (a.dim + 2);
    const int64_t ctas = n * a.heads * ((a.nq + kRowsR - 1) / kRowsR) * a.splits;
    MBX_REQUIRE(ctas < (int64_t(1) << 31), "block_attention: too many query rows");
    ensure_smem_limit((const void*)attention_rows_kernel<T, kRowsR>, (int)smem, "attention_rows");
    attention_rows_kernel<T, kRowsR><<<(unsigned)ctas, kRowWarps * 32, smem, ctx->stream>>>(a, group);
    after_launch(ctx, "attention_rows");
}

template <class T>
void launch_join(mbx_ctx* ctx, const AttnArgs& a, int64_t n) {
    const int64_t rows = n * a.nq * a.heads;
    MBX_REQUIRE(rows < (int64_t(1) << 31), "block_attention: too many query rows");
    attention_join_kernel<T><<<(unsigned)rows, 128, 0, ctx->stream>>>(a);
    after_launch(ctx, "attention_join");
}

}  // namespace

size_t block_attention_bytes(const BlockShape& s, int64_t topk) {
    const Plan p = plan_of(s, topk);
    return p.part_bytes + p.split_bytes;
}

void launch_block_attention(mbx_ctx* ctx, const BlockShape& s, const void* q, int64_t q_stride, const void* k,
                            int64_t k_stride, const void* v, int64_t v_stride, const uint8_t* key_mask,
                            const int32_t* index, int64_t topk, float scale, void* out, void* workspace) {
    const Plan p = plan_of(s, topk);
    AttnArgs a{};
    a.q = q, a.k = k, a.v = v;
    a.q_stride = q_stride, a.k_stride = k_stride, a.v_stride = v_stride;
    a.nq = s.nq, a.nk = s.nk, a.topk = topk;
    a.heads = (int)s.heads, a.kv_heads = (int)s.kv_heads, a.dim = (int)s.dim, a.block_k = (int)s.block_k;
    a.k_blocks = (int)((s.nk + s.block_k - 1) / s.block_k);
    a.q_blocks = (int)((s.nq + MBX_ATTENTION_BLOCK_Q - 1) / MBX_ATTENTION_BLOCK_Q);
    a.mask = key_mask, a.index = index;
    a.scale = scale * 1.4426950408889634f;  // log2(e)
    a.out = out;
    a.part = static_cast<float*>(workspace);
    a.splits = p.splits;
    if (p.rows)
        launch_rows<float>(ctx, a, s.n);
    else
        launch_attention_tc(ctx, a, s.dtype, s.n, static_cast<uint8_t*>(workspace) + p.part_bytes);
    if (p.splits == 1) return;
    if (s.dtype == MBX_DTYPE_F32) return launch_join<float>(ctx, a, s.n);
    if (s.dtype == MBX_DTYPE_F16) return launch_join<__half>(ctx, a, s.n);
    launch_join<__nv_bfloat16>(ctx, a, s.n);
}

}  // namespace mbx
