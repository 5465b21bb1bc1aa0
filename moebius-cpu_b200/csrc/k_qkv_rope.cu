// Per-head norm and rotary positions of a packed projection, in one pass.
//
// A token's row of x is [q heads | k heads | v heads] of `dim` channels each,
// as a 1×1 convolution writes it. For every q and k head
//   y = x · gamma / sqrt(mean(x²) + eps)                 (norm, optional)
// and then, for each axis a of (time, height, width) with its section of
// D_a channels and the token's position p_a, pair i of the section turns by
// p_a · theta^(−2i / D_a):
//   (y0, y1) → (y0·cos − y1·sin, y1·cos + y0·sin).
// Channels behind the last section keep their value; v heads are only
// converted.
//
// Bound by memory: each value is read once and written once, with about eight flops in between; what keeps a
// kernel from that bound is its instructions. A group of dim / 8 lanes holds one head (eight channels a lane,
// 16-byte accesses), so a warp works on 32 / (dim / 8) heads at a time and the norm is a few shuffles;
// v needs no heads and is converted as one run. Cosines and sines belong to a token, not to a head: the
// block computes each once into shared memory and a lane keeps its channels' in registers while it walks the
// token's heads. Pairs of halves meet through shared memory, nine floats a lane against bank conflicts.
// Measured on a B200: 65536 tokens x 32 heads x 128 bf16 in 213 us (5.0 TB/s read and written, instructions
// issued in 60 % of the cycles), 65536 x 24 x 40 f32 -> f16 in halves in 100 us (3.8 TB/s, 62 %). Four blocks an SM
// leave 64 registers a thread, of which halves spill 2 to 6.
// Angles: theta^(−2i / D_a) / 2π and its product with the position are f64, as
// an f32 product is off by 6e-8 of the angle, 0.06 rad at a position of 1e6;
// the part behind the whole turns then fits f32, and sincospif takes it.
#include <cmath>

#include "mbx_device.cuh"
#include "mbx_internal.h"

namespace mbx {
namespace {

constexpr int kWarps = 8;
constexpr int kMaxPairs = kRopeMaxDim / 2;

struct RopeArgs {
    const void* x;
    void *q, *k, *v;
    const float *q_gamma, *k_gamma, *pos;
    uint32_t tokens, total;           // tokens of an item, of all items
    int64_t x_stride;                 // elements between tokens of x
    int64_t pos_item;                 // floats between two items' positions (0: shared)
    int heads, kv_heads, dim;
    int lanes, per_warp;              // lanes of a head, heads of a warp's step
    int warps_per_token, per_block;   // warps that share a token; tokens of a block
    int pairs0, pairs1, pairs;        // pairs of the sections before the second, third axis; of all
    int norm;
    float eps;
    double turns[kMaxPairs];          // theta^(−2i / D_a) / 2π of every pair
};

// Sum over the L lanes of a head (this one is its li-th, the first is `lane0`), the same in each: for a power of two
// by halves, else sums of 1, 2, 4 … neighbours, cyclically, by the binary digits of L.
__device__ __forceinline__ float head_sum(float v, int L, int li, int lane0) {
    if ((L & (L - 1)) == 0) {
#pragma unroll
        for (int o = 1; o < 32; o *= 2)
            if (o < L) v += __shfl_xor_sync(0xffffffffu, v, o);
        return v;
    }
    float t = v;
    int n = 1;
    for (int bit = 30 - __clz(L); bit >= 0; --bit) {
        int from = li + n;
        from -= from >= L ? L : 0;
        t += __shfl_sync(0xffffffffu, t, lane0 + from);
        n *= 2;
        if (L >> bit & 1) {
            from = li + 1;
            from -= from >= L ? L : 0;
            t = v + __shfl_sync(0xffffffffu, t, lane0 + from);
            ++n;
        }
    }
    return __shfl_sync(0xffffffffu, t, lane0);  // the lanes added in different orders
}

__device__ __forceinline__ void read8(float (&v)[8], const float* p) {
    const float4 x = reinterpret_cast<const float4*>(p)[0], y = reinterpret_cast<const float4*>(p)[1];
    v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w, v[4] = y.x, v[5] = y.y, v[6] = y.z, v[7] = y.w;
}

template <class TIn, class TOut, bool HALVES>
__global__ void __launch_bounds__(kWarps * 32, 4) qkv_norm_rope_kernel(const __grid_constant__ RopeArgs a) {
    cudaGridDependencySynchronize();
    extern __shared__ __align__(16) float smem[];
    float* cos_t = smem;                        // [per_block][dim]
    float* sin_t = cos_t + a.per_block * a.dim;  // [per_block][dim], the sign of each channel's partner in it
    float* gam = sin_t + a.per_block * a.dim;    // [2][dim]
    float* xch = gam + 2 * a.dim;                // [kWarps][32 · 9], HALVES: normalised rows, 9 floats a lane
    int* partner = reinterpret_cast<int*>(xch + (HALVES ? kWarps * 32 * 9 : 0));  // [dim], HALVES
    const uint32_t t0 = blockIdx.x * (uint32_t)a.per_block;
    const int count = (int)min((uint32_t)a.per_block, a.total - t0);  // tokens here

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane / a.lanes, li = lane - g * a.lanes;  // head of the warp's step, lane of the head
    const bool holds = g < a.per_warp;
    const int rows = a.heads + a.kv_heads, step = a.warps_per_token * a.per_warp;  // heads between two steps
    const int tl = warp / a.warps_per_token, part = warp - tl * a.warps_per_token, apart = kWarps / a.warps_per_token;
    const TIn* x0 = static_cast<const TIn*>(a.x) + t0 * a.x_stride;
    using Raw = typename Raw8<TIn>::type;
    Raw raw{};
    const int h_first = part * a.per_warp + g;
    const TIn* x = x0 + tl * a.x_stride + h_first * a.dim + li * 8;
    // A lane loads what x is at only for a head and a token that exist: a step may hold more heads than a token has.
    auto fetch = [&](int h, int t) {
        if (holds && h < rows && t < count) raw = load_raw8(x);
    };
    // The first step's values are on their way while the block computes its table, the next step's while it works on one.
    fetch(h_first, tl);

    // A thread keeps one pair and goes through the tokens (more threads than pairs share them).
    if (a.pairs > 0) {
        const int lanes = kWarps * 32 / a.pairs, t_first = threadIdx.x / a.pairs, p = threadIdx.x - t_first * a.pairs;
        const int axis = p < a.pairs0 ? 0 : (p < a.pairs1 ? 1 : 2);
        const int first = axis == 0 ? 0 : (axis == 1 ? a.pairs0 : a.pairs1);
        const int half = (axis == 0 ? a.pairs0 : (axis == 1 ? a.pairs1 : a.pairs)) - first;
        const int e0 = HALVES ? first + p : 2 * p;  // section starts at channel 2·first
        const int e1 = HALVES ? e0 + half : e0 + 1;
        const double turns = a.turns[p];
        if (HALVES && t_first == 0) partner[e0] = e1, partner[e1] = e0;
        uint32_t item = t0 / a.tokens, in_item = t0 - item * a.tokens + t_first;
        for (int t = t_first; t < count && t_first < lanes; t += lanes, in_item += lanes) {
            while (in_item >= a.tokens) in_item -= a.tokens, ++item;
            const double turn = (double)__ldg(a.pos + item * a.pos_item + (int64_t)in_item * 3 + axis) * turns;
            float s, c;
            sincospif(2.0f * (float)(turn - rint(turn)), &s, &c);
            cos_t[t * a.dim + e0] = c, sin_t[t * a.dim + e0] = -s;
            cos_t[t * a.dim + e1] = c, sin_t[t * a.dim + e1] = s;
        }
    }
    const int rest = a.dim - 2 * a.pairs;  // channels that keep their value
    for (int e = threadIdx.x; e < count * rest; e += kWarps * 32) {
        const int t = e / rest, ch = e - t * rest + 2 * a.pairs;
        cos_t[t * a.dim + ch] = 1.0f, sin_t[t * a.dim + ch] = 0.0f;
        if (HALVES && t == 0) partner[ch] = ch;
    }
    for (int e = threadIdx.x; e < a.dim; e += kWarps * 32) {
        gam[e] = a.q_gamma ? a.q_gamma[e] : 1.0f;
        gam[a.dim + e] = a.k_gamma ? a.k_gamma[e] : 1.0f;
    }
    __syncthreads();

    const int ch = holds ? li * 8 : 0;  // first channel of this lane
    int pa[8];
    if (HALVES) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int pos = (holds ? g : 0) * a.dim + partner[ch + i];
            pa[i] = warp * 32 * 9 + pos + (pos >> 3);
        }
    }
    const float inv_dim = 1.0f / (float)a.dim;
    for (int t = tl; t < count; t += apart) {
        const uint32_t token = t0 + t;
        // Rows of q and of k, each in its own tensor: row h of the token is at `row + h · dim`.
        TOut* q_row = static_cast<TOut*>(a.q) + (int64_t)token * a.heads * a.dim + li * 8;
        TOut* k_row = static_cast<TOut*>(a.k) + ((int64_t)token * a.kv_heads - a.heads) * a.dim + li * 8;
        float co[8], si[8];
        read8(co, cos_t + t * a.dim + ch);
        read8(si, sin_t + t * a.dim + ch);
        for (int h0 = part * a.per_warp; h0 < rows; h0 += step) {
            const int h = h0 + g;
            float y[8];
            widen8<TIn>(raw, y);
            if (h0 + step < rows) {
                x += step * a.dim;
                fetch(h + step, t);
            } else {
                x += apart * a.x_stride - (h0 - part * a.per_warp) * a.dim;
                fetch(h_first, t + apart);
            }
            const bool is_q = h < a.heads;
            if (a.norm) {
                float ss = 0.0f;
#pragma unroll
                for (int i = 0; i < 8; ++i) ss = fmaf(y[i], y[i], ss);
                const float r = rsqrtf(fmaf(head_sum(ss, a.lanes, li, lane - li), inv_dim, a.eps));
                float gm[8];
                read8(gm, gam + (is_q ? 0 : a.dim) + ch);
#pragma unroll
                for (int i = 0; i < 8; ++i) y[i] *= r * gm[i];
            }
            float z[8];
            if (HALVES) {
                __syncwarp();
#pragma unroll
                for (int i = 0; i < 8; ++i) xch[(warp * 32 + lane) * 9 + i] = y[i];
                __syncwarp();
#pragma unroll
                for (int i = 0; i < 8; ++i) z[i] = fmaf(y[i], co[i], xch[pa[i]] * si[i]);
            } else {
#pragma unroll
                for (int i = 0; i < 8; i += 2) {
                    z[i] = fmaf(y[i], co[i], y[i + 1] * si[i]);
                    z[i + 1] = fmaf(y[i + 1], co[i + 1], y[i] * si[i + 1]);
                }
            }
            if (holds && h < rows) store8((is_q ? q_row : k_row) + h * a.dim, z);
        }
        if (a.v) {
            const TIn* from = x0 + t * a.x_stride + rows * a.dim;
            TOut* to = static_cast<TOut*>(a.v) + (int64_t)token * a.kv_heads * a.dim;
            const int pieces = a.kv_heads * a.dim / 8;
#pragma unroll 2
            for (int e = part * 32 + lane; e < pieces; e += a.warps_per_token * 32) {
                float y[8];
                widen8<TIn>(load_raw8(from + e * 8), y);
                store8(to + e * 8, y);
            }
        }
    }
}

template <class TIn, class TOut>
void launch_typed(mbx_ctx* ctx, const RopeArgs& a, bool halves) {
    const int64_t blocks = ((int64_t)a.total + a.per_block - 1) / a.per_block;
    const size_t smem = 4 * ((size_t)(2 * a.per_block + 2) * a.dim + (halves ? kWarps * 32 * 9 + a.dim : 0));
    const auto kernel = halves ? qkv_norm_rope_kernel<TIn, TOut, true> : qkv_norm_rope_kernel<TIn, TOut, false>;
    ensure_smem_limit((const void*)kernel, (int)smem, "qkv_norm_rope");
    launch_after(ctx, "qkv_norm_rope", kernel,
                 dim3((unsigned)blocks), kWarps * 32, smem, a);
}

}  // namespace

void launch_qkv_norm_rope(mbx_ctx* ctx, const QkvRope& r) {
    RopeArgs a{};
    a.x = r.x, a.q = r.q, a.k = r.k, a.v = r.v;
    a.q_gamma = r.q_gamma, a.k_gamma = r.k_gamma, a.pos = r.positions;
    a.tokens = (uint32_t)r.tokens, a.total = (uint32_t)(r.n * r.tokens), a.x_stride = r.x_stride;
    a.pos_item = r.position_items == 1 ? 0 : r.tokens * 3;
    a.heads = (int)r.heads, a.kv_heads = (int)r.kv_heads, a.dim = (int)r.dim;
    a.lanes = a.dim / 8;
    a.per_warp = 32 / a.lanes;
    const int units = (a.heads + a.kv_heads + a.per_warp - 1) / a.per_warp;  // warp steps of a token
    // A warp keeps a token's cosines while it walks the heads, and takes two tokens where that leaves every SM eight
    // blocks (65536 x 32 x 128 bf16: 213 us with one, 210 with two, 221 with four); a token's heads are spread over more
    // warps where whole tokens would leave most of the card idle.
    a.warps_per_token = 1;
    while (a.warps_per_token < kWarps && a.warps_per_token < units &&
           (int64_t)a.total * a.warps_per_token < (int64_t)ctx->sm_count * kWarps)
        a.warps_per_token *= 2;
    a.per_block = kWarps / a.warps_per_token;
    if ((int64_t)a.total >= 2 * 8 * kWarps * (int64_t)ctx->sm_count) a.per_block *= 2;
    a.norm = r.norm, a.eps = r.eps;
    if (r.positions) {
        constexpr double kTwoPi = 6.283185307179586476925286766559;
        int p = 0;
        for (int axis = 0; axis < 3; ++axis) {
            const int half = (int)r.axis_dims[axis] / 2;
            const double step = half ? std::pow(r.theta, -1.0 / half) : 1.0;
            double f = 1.0 / kTwoPi;  // pair i: theta^(−2i / D_a) / 2π
            for (int i = 0; i < half; ++i, f *= step) a.turns[p++] = f;
            if (axis == 0) a.pairs0 = p;
            if (axis == 1) a.pairs1 = p;
        }
        a.pairs = p;
    }
    const bool halves = r.pairing == MBX_ROPE_HALVES && a.pairs > 0;
    if (r.x_dtype == MBX_DTYPE_F32) {
        if (r.out_dtype == MBX_DTYPE_F32) return launch_typed<float, float>(ctx, a, halves);
        if (r.out_dtype == MBX_DTYPE_F16) return launch_typed<float, __half>(ctx, a, halves);
        return launch_typed<float, __nv_bfloat16>(ctx, a, halves);
    }
    if (r.x_dtype == MBX_DTYPE_F16) return launch_typed<__half, __half>(ctx, a, halves);
    launch_typed<__nv_bfloat16, __nv_bfloat16>(ctx, a, halves);
}

}  // namespace mbx
