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
// Bound by memory: each value is read once and written once, with about eight
// flops in between. A group of dim / 8 lanes holds one head (eight channels a
// lane, 16-byte accesses), so a warp works on 32 / (dim / 8) heads at a time
// and the norm is a few shuffles. Cosines and sines belong to a token, not to
// a head: the block computes each once into shared memory and a lane keeps its
// channels' in registers while it walks the token's heads.
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
    int64_t tokens, total, x_stride;  // tokens of an item, of all items; elements between tokens of x
    int64_t pos_item;                 // floats between two items' positions (0: shared)
    int heads, kv_heads, rows, dim;   // rows = heads + kv_heads, + kv_heads where v is written
    int lanes, per_warp, units;       // lanes of a head, heads of a warp, warp steps of a token
    int warps_per_token;
    int pairs0, pairs1, pairs;        // pairs of the sections before the second, third axis; of all
    int norm;
    float eps;
    double turns[kMaxPairs];          // theta^(−2i / D_a) / 2π of every pair
};

template <class TIn, class TOut, bool HALVES>
__global__ void __launch_bounds__(kWarps * 32) qkv_norm_rope_kernel(const __grid_constant__ RopeArgs a) {
    extern __shared__ float smem[];
    const int tpb = kWarps / a.warps_per_token;  // tokens of this block
    float* cos_t = smem;                         // [tpb][dim]
    float* sin_t = cos_t + tpb * a.dim;          // [tpb][dim], the sign of each channel's partner in it
    float* gam = sin_t + tpb * a.dim;            // [2][dim]
    float* xch = gam + 2 * a.dim;                // [kWarps][32 · 9], HALVES: normalised rows, 9 floats a lane
    int* partner = reinterpret_cast<int*>(xch + (HALVES ? kWarps * 32 * 9 : 0));  // [dim], HALVES
    const int64_t t0 = (int64_t)blockIdx.x * tpb;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane / a.lanes, li = lane - g * a.lanes;  // head of the warp's step, lane of the head
    const int tl = warp / a.warps_per_token;
    const int64_t token = t0 + tl;
    const bool in = g < a.per_warp && token < a.total;
    const TIn* xrow = static_cast<const TIn*>(a.x) + token * a.x_stride + li * 8;
    using Raw = typename Raw8<TIn>::type;
    int u = warp - tl * a.warps_per_token;
    Raw raw{};
    // The first step's values are on their way while the block computes its table.
    if (in && u * a.per_warp + g < a.rows) raw = load_raw8(xrow + (int64_t)(u * a.per_warp + g) * a.dim);

    for (int e = threadIdx.x; e < tpb * a.pairs; e += kWarps * 32) {
        const int t = e / a.pairs, p = e - t * a.pairs;
        if (t0 + t >= a.total) continue;
        const int axis = p < a.pairs0 ? 0 : (p < a.pairs1 ? 1 : 2);
        const int first = axis == 0 ? 0 : (axis == 1 ? a.pairs0 : a.pairs1);
        const int half = (axis == 0 ? a.pairs0 : (axis == 1 ? a.pairs1 : a.pairs)) - first;
        const int64_t item = (t0 + t) / a.tokens, in_item = (t0 + t) - item * a.tokens;
        const double turn = (double)__ldg(a.pos + item * a.pos_item + in_item * 3 + axis) * a.turns[p];
        float s, c;
        sincospif((float)(2.0 * (turn - rint(turn))), &s, &c);
        const int e0 = HALVES ? first + p : 2 * p;  // section starts at channel 2·first
        const int e1 = HALVES ? e0 + half : e0 + 1;
        cos_t[t * a.dim + e0] = c, sin_t[t * a.dim + e0] = -s;
        cos_t[t * a.dim + e1] = c, sin_t[t * a.dim + e1] = s;
        if (HALVES && t == 0) partner[e0] = e1, partner[e1] = e0;
    }
    for (int e = threadIdx.x; e < tpb * (a.dim - 2 * a.pairs); e += kWarps * 32) {
        const int t = e / (a.dim - 2 * a.pairs), ch = e - t * (a.dim - 2 * a.pairs) + 2 * a.pairs;
        cos_t[t * a.dim + ch] = 1.0f, sin_t[t * a.dim + ch] = 0.0f;
        if (HALVES && t == 0) partner[ch] = ch;
    }
    for (int e = threadIdx.x; e < a.dim; e += kWarps * 32) {
        gam[e] = a.q_gamma ? a.q_gamma[e] : 1.0f;
        gam[a.dim + e] = a.k_gamma ? a.k_gamma[e] : 1.0f;
    }
    __syncthreads();

    const bool holds = g < a.per_warp;
    float co[8], si[8];
    int pa[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        co[i] = holds ? cos_t[tl * a.dim + li * 8 + i] : 1.0f;
        si[i] = holds ? sin_t[tl * a.dim + li * 8 + i] : 0.0f;
        if (HALVES) {
            const int pos = g * a.dim + (holds ? partner[li * 8 + i] : 0);
            pa[i] = pos + (pos >> 3);
        }
    }
    float* mine = xch + warp * 32 * 9;

    for (; u < a.units; u += a.warps_per_token) {
        const int h = u * a.per_warp + g;
        const bool on = in && h < a.rows;
        float y[8];
        widen8<TIn>(raw, y);
        const int hn = h + a.warps_per_token * a.per_warp;
        if (in && hn < a.rows) raw = load_raw8(xrow + (int64_t)hn * a.dim);
        const bool is_q = h < a.heads, is_v = h >= a.heads + a.kv_heads;
        if (a.norm) {
            float ss = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) ss = fmaf(y[i], y[i], ss);
            // Sum over the head's lanes, whose number need not be a power of two.
            for (int o = 16; o > 0; o >>= 1) {
                if (o >= a.lanes) continue;
                const float other = __shfl_down_sync(0xffffffffu, ss, o);
                if (li + o < a.lanes && li < o) ss += other;
            }
            ss = __shfl_sync(0xffffffffu, ss, min(31, g * a.lanes));
            const float r = is_v ? 1.0f : 1.0f / sqrtf(ss / (float)a.dim + a.eps);
            const float* gm = gam + (is_q ? 0 : a.dim) + (holds ? li * 8 : 0);
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] *= is_v ? 1.0f : r * gm[i];
        }
        float z[8];
        if (HALVES) {
            __syncwarp();
#pragma unroll
            for (int i = 0; i < 8; ++i) mine[lane * 9 + i] = y[i];
            __syncwarp();
#pragma unroll
            for (int i = 0; i < 8; ++i) z[i] = fmaf(y[i], co[i], mine[pa[i]] * si[i]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                z[i] = fmaf(y[i], co[i], y[i + 1] * si[i]);
                z[i + 1] = fmaf(y[i + 1], co[i + 1], y[i] * si[i + 1]);
            }
        }
        if (!on) continue;
        if (is_v) {
            store8(static_cast<TOut*>(a.v) + (token * a.kv_heads + (h - a.heads - a.kv_heads)) * a.dim + li * 8, y);
        } else if (is_q) {
            store8(static_cast<TOut*>(a.q) + (token * a.heads + h) * a.dim + li * 8, z);
        } else {
            store8(static_cast<TOut*>(a.k) + (token * a.kv_heads + (h - a.heads)) * a.dim + li * 8, z);
        }
    }
}

template <class TIn, class TOut>
void launch_typed(mbx_ctx* ctx, const RopeArgs& a, bool halves) {
    const int tpb = kWarps / a.warps_per_token;
    const int64_t blocks = (a.total + tpb - 1) / tpb;
    MBX_REQUIRE(blocks < (int64_t(1) << 31), "qkv_norm_rope: too many tokens");
    const size_t smem = 4 * ((size_t)(2 * tpb + 2) * a.dim + (halves ? kWarps * 32 * 9 + a.dim : 0));
    if (halves)
        qkv_norm_rope_kernel<TIn, TOut, true><<<(unsigned)blocks, kWarps * 32, smem, ctx->stream>>>(a);
    else
        qkv_norm_rope_kernel<TIn, TOut, false><<<(unsigned)blocks, kWarps * 32, smem, ctx->stream>>>(a);
    after_launch(ctx, "qkv_norm_rope");
}

}  // namespace

void launch_qkv_norm_rope(mbx_ctx* ctx, const QkvRope& r) {
    RopeArgs a{};
    a.x = r.x, a.q = r.q, a.k = r.k, a.v = r.v;
    a.q_gamma = r.q_gamma, a.k_gamma = r.k_gamma, a.pos = r.positions;
    a.tokens = r.tokens, a.total = r.n * r.tokens, a.x_stride = r.x_stride;
    a.pos_item = r.position_items == 1 ? 0 : r.tokens * 3;
    a.heads = (int)r.heads, a.kv_heads = (int)r.kv_heads, a.dim = (int)r.dim;
    a.rows = a.heads + a.kv_heads * (r.v ? 2 : 1);
    a.lanes = a.dim / 8;
    a.per_warp = 32 / a.lanes;
    a.units = (a.rows + a.per_warp - 1) / a.per_warp;
    // A warp keeps one token's cosines while it walks the heads; a token's heads are spread over
    // more warps where whole tokens would leave most of the card idle.
    a.warps_per_token = 1;
    while (a.warps_per_token < kWarps && a.warps_per_token < a.units &&
           a.total * a.warps_per_token < (int64_t)ctx->sm_count * kWarps)
        a.warps_per_token *= 2;
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
