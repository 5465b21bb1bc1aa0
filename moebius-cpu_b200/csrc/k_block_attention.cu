// Softmax attention of query blocks over listed key blocks.
//
//   out[b, r, h] = Σ_j p_j v[b, j, h/g] / Σ_j p_j,  p_j = exp(scale · q[b, r, h]·k[b, j, h/g] − m)
// over the keys j of the blocks that index[b, h, r / 128] lists and that the
// key mask keeps; a row without any such key is zero.
//
// Many query rows go to the tensor cores (k_block_attention_tc.cu); this file has the kernel for few rows, the one
// that joins split lists, and the choice between them.
//
// The rows kernel reads every listed key and value once for R query rows and is bound by that. A group
// of dim / 8 lanes holds one key's channels, eight a lane, so a warp works on several keys at a time, and
// U keys of a group are on their way together. Every group keeps its own running maximum, sum and
// output (f32); groups and warps are joined at the end through shared memory. A list is split over
// CTAs, and a second kernel joins their partial (output, maximum, sum). Measured on a B200: one row of 16 heads x 128
// bf16 over 4096 of 65536 keys each in 13 us, 2.5 TB/s: two latencies of the list and its keys, and the join.
#include <algorithm>

#include "block_attention.h"
#include "mbx_device.cuh"
#include "mbx_internal.h"

namespace mbx {
namespace {

template <class T>
__device__ __forceinline__ void store_out(const AttnArgs& a, int64_t at, float v) {
    if (a.out_f32)
        static_cast<float*>(a.out)[at] = v;
    else
        static_cast<T*>(a.out)[at] = (T)v;
}

constexpr int kRowWarps = 4;
constexpr int kListPart = 1024;  // list entries in shared memory at a time

// Loads that stay where they are written: left to itself the compiler moves a value's load behind the dot products.
__device__ __forceinline__ void load_now(uint4& r, const void* p) {
    asm volatile("ld.global.nc.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p));
}
__device__ __forceinline__ void load_now(Raw8f& r, const float* p) {
    asm volatile("ld.global.nc.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(r.a.x), "=f"(r.a.y), "=f"(r.a.z), "=f"(r.a.w) : "l"(p));
    asm volatile("ld.global.nc.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(r.b.x), "=f"(r.b.y), "=f"(r.b.z), "=f"(r.b.w)
                 : "l"(p + 4));
}

// Lanes of a key's group: the power of two that holds dim / 8.
template <class T, int R, int U>
__global__ void __launch_bounds__(kRowWarps * 32) attention_rows_kernel(const AttnArgs a, int lg_group) {
    cudaGridDependencySynchronize();
    // One slot per (warp, group, row) for the join at the end: maxima, sums, outputs.
    extern __shared__ float sh[];
    __shared__ int list[kListPart];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int group = 1 << lg_group, li = lane & (group - 1), gi = lane >> lg_group, groups = 32 >> lg_group;
    const int slots = kRowWarps * groups, slot = warp * groups + gi;
    const bool holds = li * 8 < a.dim;
    const uint32_t tiles = (uint32_t)((a.nq + R - 1) / R);
    const uint32_t cta = blockIdx.x / (uint32_t)a.splits, head_at = cta / tiles;
    const int split = (int)(blockIdx.x - cta * a.splits);
    const int64_t r0 = (int64_t)(cta - head_at * tiles) * R;
    const int64_t item = head_at / (uint32_t)a.heads;
    const int h = (int)(head_at - (uint32_t)item * a.heads), kh = h / (a.heads / a.kv_heads);
    // A tile of R rows never straddles two query blocks: R divides 128.
    const int32_t* index = a.index + ((item * a.heads + h) * a.q_blocks + r0 / MBX_ATTENTION_BLOCK_Q) * a.topk;
    const T* q = static_cast<const T*>(a.q) + (item * a.nq + r0) * a.q_stride + (int64_t)h * a.dim + li * 8;
    const T* k0 = static_cast<const T*>(a.k) + item * a.nk * a.k_stride + (int64_t)kh * a.dim;
    const T* v0 = static_cast<const T*>(a.v) + item * a.nk * a.v_stride + (int64_t)kh * a.dim;
    const T *k = k0 + li * 8, *v = v0 + li * 8;
    const uint8_t* mask = a.mask ? a.mask + item * a.nk : nullptr;
    const int lg_block = 31 - __clz(a.block_k);

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

    const int first = (int)(a.topk * split / a.splits), last = (int)(a.topk * (split + 1) / a.splits);
    using Raw = typename Raw8<T>::type;
    for (int part = first; part < last; part += kListPart) {
        const int entries = min(kListPart, last - part);
        __syncthreads();
        for (int e = threadIdx.x; e < entries; e += kRowWarps * 32) list[e] = index[part + e];
        __syncthreads();
        const int64_t end = (int64_t)entries << lg_block;  // in the list's keys
        for (int64_t p0 = (int64_t)warp * U * groups; p0 < end; p0 += (int64_t)kRowWarps * U * groups) {
            Raw kr[U], vr[U];
            bool on[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int64_t p = p0 + u * groups + gi;
                const int blk = p < end ? list[p >> lg_block] : -1;
                const int64_t j = ((int64_t)blk << lg_block) + (p & (a.block_k - 1));
                on[u] = (uint32_t)blk < (uint32_t)a.k_blocks && j < a.nk && (!mask || mask[j]);
                // Every lane loads, from the item's first key where it has none, so that all loads are under way at once.
                const bool real = on[u] && holds;
                load_now(kr[u], real ? k + j * a.k_stride : k0);
                load_now(vr[u], real ? v + j * a.v_stride : v0);
            }
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (!(on[u] && holds)) kr[u] = Raw{}, vr[u] = Raw{};
            float d[U][R];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                float kv[8];
                widen8<T>(kr[u], kv);
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    d[u][r] = 0.0f;
#pragma unroll
                    for (int i = 0; i < 8; ++i) d[u][r] = fmaf(qv[r][i], kv[i], d[u][r]);
                }
            }
            for (int o = group >> 1; o > 0; o >>= 1) {
#pragma unroll
                for (int u = 0; u < U; ++u)
#pragma unroll
                    for (int r = 0; r < R; ++r) d[u][r] += __shfl_xor_sync(0xffffffffu, d[u][r], o);
            }
#pragma unroll
            for (int r = 0; r < R; ++r) {
                float mn = m[r];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    if (!on[u]) d[u][r] = -INFINITY;
                    mn = fmaxf(mn, d[u][r]);
                }
                const float ref = mn == -INFINITY ? 0.0f : mn;  // nothing yet: every weight is 2^-inf
                const float c = exp2f(m[r] - ref);
                m[r] = mn, l[r] *= c;
#pragma unroll
                for (int i = 0; i < 8; ++i) acc[r][i] *= c;
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    d[u][r] = exp2f(d[u][r] - ref);
                    l[r] += d[u][r];
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                float vv[8];
                widen8<T>(vr[u], vv);
#pragma unroll
                for (int r = 0; r < R; ++r)
#pragma unroll
                    for (int i = 0; i < 8; ++i) acc[r][i] = fmaf(d[u][r], vv[i], acc[r][i]);
            }
        }
    }

    float* sm = sh;              // [slots][R]
    float* sl = sm + slots * R;  // [slots][R]
    float* so = sl + slots * R;  // [slots][R][dim]
    if (li == 0) {
#pragma unroll
        for (int r = 0; r < R; ++r) sm[slot * R + r] = m[r], sl[slot * R + r] = l[r];
    }
    if (holds) {
#pragma unroll
        for (int r = 0; r < R; ++r) store8(so + (slot * R + r) * a.dim + li * 8, acc[r]);
    }
    __syncthreads();
    for (int e = threadIdx.x; e < R * a.dim; e += kRowWarps * 32) {
        const int r = e / a.dim, ch = e - r * a.dim;
        if (r0 + r >= a.nq) continue;
        float top = -INFINITY;
        for (int s = 0; s < slots; ++s) top = fmaxf(top, sm[s * R + r]);
        const float ref = top == -INFINITY ? 0.0f : top;
        float sum = 0.0f, o = 0.0f;
#pragma unroll 4
        for (int s = 0; s < slots; ++s) {
            const float w = exp2f(sm[s * R + r] - ref);
            sum = fmaf(w, sl[s * R + r], sum);
            o = fmaf(w, so[(s * R + r) * a.dim + ch], o);
        }
        const int64_t row = (item * a.nq + r0 + r) * a.heads + h;
        if (a.splits == 1) {
            store_out<T>(a, row * a.dim + ch, sum == 0.0f ? 0.0f : o / sum);
        } else {
            float* p = a.part + (row * a.splits + split) * (a.dim + 4);
            p[ch] = o;
            if (ch == 0) p[a.dim] = top, p[a.dim + 1] = sum;
        }
    }
}

// Joins the splits' partial results: a CTA per (row, head). The splits' weights are worked out once in shared memory;
// then each warp adds every fourth split, a lane four channels, eight splits in flight.
constexpr int kMaxSplits = 256;

template <class T>
__global__ void __launch_bounds__(128) attention_join_kernel(const AttnArgs a) {
    __shared__ float weight[kMaxSplits];
    __shared__ float4 acc[4][32];
    __shared__ float total;
    cudaGridDependencySynchronize();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, stride = a.dim + 4;
    const float* p = a.part + (int64_t)blockIdx.x * a.splits * stride;
    if (warp == 0) {
        constexpr int MINE = kMaxSplits / 32;
        float m[MINE], l[MINE], top = -INFINITY;
#pragma unroll
        for (int i = 0; i < MINE; ++i) {
            const int s = lane + 32 * i;
            m[i] = s < a.splits ? p[s * stride + a.dim] : -INFINITY;
            l[i] = s < a.splits ? p[s * stride + a.dim + 1] : 0.0f;
        }
#pragma unroll
        for (int i = 0; i < MINE; ++i) top = fmaxf(top, m[i]);
        for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < MINE; ++i) {
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
        store_out<T>(a, (int64_t)blockIdx.x * a.dim + threadIdx.x, total == 0.0f ? 0.0f : y / total);
    }
}

constexpr int64_t kSms = 148;  // of a B200: the workspace functions have no context to ask

// Which kernel takes a problem, and over how many CTAs a list is split.
struct Plan {
    int rows;  // query rows of a CTA of the rows kernel; 0: the tensor cores
    int splits;
    size_t part_bytes, split_bytes;
};

Plan plan_of(const BlockShape& s, int64_t topk) {
    Plan p{};
    // 16 bits: the rows kernel for one or two rows of few heads (16 heads x 128 over 4096 of 65536 keys bf16: 14.5 us
    // against 16.5, four rows 26 against 16; 128 heads: 72 us against 61). f32: while it reads no more than twice the keys
    // that the tensor cores' operands would have to be split for (the same shape, 32 rows: 127 us against 221, 64: 207
    // against 222; 16 x 1024 of 4096 keys x 8 x 40, 16 rows: 70 against 103, 32: 117 against 105, 64: 199 against 110).
    const bool few = s.dtype == MBX_DTYPE_F32
                         ? (s.nq + 3) / 4 * s.heads * std::min(topk * s.block_k, s.nk) <= 2 * s.nk * s.kv_heads
                         : s.nq <= 2 && s.n * s.heads < 64;
    if (few) p.rows = s.nq == 1 ? 1 : s.nq == 2 ? 2 : 4;
    // Enough CTAs to fill the card four times over (rows) or twice (tensor cores), with equal shares of the list's blocks
    // or tiles of 64 keys, but no more than kFillSplits.
    constexpr int64_t kFillSplits = 64;
    const int64_t tile = p.rows ? p.rows : MBX_ATTENTION_BLOCK_Q;
    const int64_t ctas = std::max<int64_t>(1, s.n * s.heads * ((s.nq + tile - 1) / tile));
    const int64_t pieces = std::max<int64_t>(1, p.rows ? topk : (topk * s.block_k + 63) / 64);
    int64_t want = std::min(((p.rows ? 4 : 2) * kSms + ctas - 1) / ctas, kFillSplits);
    // The tensor core truncates as it adds, so a 16-bit result's unbroken sum falls behind by 2^-23.2 each 16 keys (f16,
    // equal weights over 2^21 keys: 1.4 %, in shares of 2^15 0.03 % with the rounding). Half of the result's own half step is the most it
    // may lose: 2^15 keys for f16, 2^18 for bf16. f32 sums are broken anyway.
    if (!p.rows && s.dtype != MBX_DTYPE_F32)
        want = std::max(want, (pieces * 64 - 1 >> (s.dtype == MBX_DTYPE_F16 ? 15 : 18)) + 1);
    const int64_t share = (pieces + want - 1) / want;
    p.splits = (int)((pieces + share - 1) / share);
    if (p.splits > 1)
        p.part_bytes = align256(sizeof(float) * (size_t)(s.n * s.nq * s.heads) * p.splits * (s.dim + 4));
    if (!p.rows && s.dtype == MBX_DTYPE_F32) p.split_bytes = attention_split_bytes(s);
    return p;
}

template <class T, int R>
void launch_rows(mbx_ctx* ctx, const AttnArgs& a, int64_t n) {
    int lg_group = 0;
    while ((8 << lg_group) < a.dim) ++lg_group;
    const int slots = kRowWarps * (32 >> lg_group);
    const size_t smem = sizeof(float) * (size_t)slots * R * (a.dim + 2);
    const int64_t ctas = n * a.heads * ((a.nq + R - 1) / R) * a.splits;
    MBX_REQUIRE(ctas < (int64_t(1) << 31), "block_attention: too many query rows");
    constexpr int U = (sizeof(T) == 2 ? 4 : 2) * (R == 1 ? 2 : 1);  // 128 bytes of keys and values a lane, 256 for one row
    ensure_smem_limit((const void*)attention_rows_kernel<T, R, U>, (int)smem, "attention_rows");
    launch_after(ctx, "attention_rows", attention_rows_kernel<T, R, U>, dim3((unsigned)ctas), kRowWarps * 32, smem, a, lg_group);
}

template <class T>
void launch_rows_any(mbx_ctx* ctx, const AttnArgs& a, int64_t n, int rows) {
    if (rows == 1) return launch_rows<T, 1>(ctx, a, n);
    if (rows == 2) return launch_rows<T, 2>(ctx, a, n);
    launch_rows<T, 4>(ctx, a, n);
}

template <class T>
void launch_join(mbx_ctx* ctx, const AttnArgs& a, int64_t n) {
    const int64_t rows = n * a.nq * a.heads;
    MBX_REQUIRE(rows < (int64_t(1) << 31), "block_attention: too many query rows");
    launch_after(ctx, "attention_join", attention_join_kernel<T>, dim3((unsigned)rows), 128, 0, a);
}

}  // namespace

size_t block_attention_bytes(const BlockShape& s, int64_t topk) {
    const Plan p = plan_of(s, topk);
    return p.part_bytes + p.split_bytes;
}

void launch_block_attention(mbx_ctx* ctx, const BlockShape& s, const void* q, int64_t q_stride, const void* k,
                            int64_t k_stride, const void* v, int64_t v_stride, const uint8_t* key_mask,
                            const int32_t* index, int64_t topk, float scale, void* out, bool out_f32,
                            void* workspace) {
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
    a.out = out, a.out_f32 = out_f32;
    a.part = static_cast<float*>(workspace);
    a.splits = p.splits;
    if (p.rows) {
        if (s.dtype == MBX_DTYPE_F32)
            launch_rows_any<float>(ctx, a, s.n, p.rows);
        else if (s.dtype == MBX_DTYPE_F16)
            launch_rows_any<__half>(ctx, a, s.n, p.rows);
        else
            launch_rows_any<__nv_bfloat16>(ctx, a, s.n, p.rows);
    } else {
        launch_attention_tc(ctx, a, s.dtype, s.n, static_cast<uint8_t*>(workspace) + p.part_bytes);
    }
    if (p.splits == 1) return;
    if (s.dtype == MBX_DTYPE_F32) return launch_join<float>(ctx, a, s.n);
    if (s.dtype == MBX_DTYPE_F16) return launch_join<__half>(ctx, a, s.n);
    launch_join<__nv_bfloat16>(ctx, a, s.n);
}

}  // namespace mbx
