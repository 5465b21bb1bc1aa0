// What the kernels of mbx_block_attention share (k_block_attention.cu, k_block_attention_tc.cu).
#pragma once

#include "mbx_internal.h"

namespace mbx {

struct AttnArgs {
    const void *q, *k, *v;
    int64_t q_stride, k_stride, v_stride, nq, nk, topk;
    int heads, kv_heads, dim, block_k, k_blocks, q_blocks;
    const uint8_t* mask;   // [n][nk] or null
    const int32_t* index;  // [n][heads][q_blocks][topk]
    float scale;           // scale · log2(e): exponentials are 2^x
    void* out;             // [n][nq][heads][dim]
    bool out_f32;          // float32, whatever the operands' type
    float* part;           // splits > 1: [n][nq][heads][splits][dim + 4]: Σ p v, log2 of what p is relative to, Σ p, 2 unused
    int splits;            // CTAs that share a list
};

// The tensor-core kernel. f32 operands: `split` holds their f16 parts (attention_split_bytes).
void launch_attention_tc(mbx_ctx* ctx, const AttnArgs& a, int dtype, int64_t n, void* split);
size_t attention_split_bytes(const BlockShape& s);

}  // namespace mbx
