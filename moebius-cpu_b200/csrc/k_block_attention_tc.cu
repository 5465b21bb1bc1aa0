// Block attention on the sm_100a tensor cores (tcgen05.mma, accumulators and weights in TMEM,
// TMA-fed operands).
//
// A CTA takes one query block (128 rows) of one (item, head), or a share of its list, and walks
// the listed key blocks in tiles of 64 or 128 keys (a part of a block, or several blocks with a TMA
// box each, so any block size feeds the same tile). Seven warps:
//   warps 0-3  softmax: a thread owns a query row (a TMEM lane). It reads S from TMEM, keeps the
//              running maximum and sum in f32 registers and writes the weights 2^(c·s − c·m)
//              back to TMEM, as the second product's left operand.
//   warps 4, 6 producers: TMA for Q once and for K of every tile, with the tile's bits of valid keys; TMA
//              for V. (One warp for both would hold back the next K until P·V frees a V stage.)
//   warp 5     MMA issuer (one lane) and TMEM allocation.
// Two CTAs share an SM (one for f32 with more than 64 channels), 256 TMEM columns each, and two ways
// to let a tile's Q·Kᵀ run while the softmax warps work on the tile before it:
//   16-bit, up to 64 channels: tiles of 128 keys, S, a P of its own and O (128 + 64 + 64 columns). Q·Kᵀ
//     of the next tile begins when S has been read for the last time, half way through the weights.
//   otherwise: tiles of 64 keys, two S tiles in turn, P over its S, and O (f32: twice). Q·Kᵀ of the tile
//     after the next begins when P·V has read P. The price is N = 64, at which reading Q from shared
//     memory takes 1.5 times the product's own cycles; with one S tile of 128 keys instead, P·V and Q·Kᵀ
//     stand between two softmax steps (1.3 times the time at 128 channels).
// A tile's fixed costs in the softmax warps (waits, exchange, addresses: some 400 of 1570 cycles for 64 keys)
// are what the longer tile halves. Two threads a row, for twice the warps, cost more than they hid.
// Shared memory: Q, K and V in 128-byte-swizzled panels of 64 channels; V serves as the N-major
// operand as it lies, so nothing is transposed.
//
// 16-bit operands: P is rounded to their type: half a step of a weight, beside half a step of the
// result at the end: 2.16e-4 of the exact result at 1024 px and 1.73e-3 for video, where the result's rounding
// alone is 2.07e-4 and 1.66e-3. Weights in two parts come to that, for half as many tensor products again and more
// instructions a weight (1024 px 573 us against 462, video 761 against 623): not worth it in types whose users
// round more elsewhere; float32 operands have them. The weights are relative to a reference that is raised only when a row's
// maximum outgrows it by 2^8, so O, which accumulates in TMEM over the whole list, is rarely
// rescaled. The reference comes off S before the factor: as one fused step, its own product is rounded to a
// step of f32, which past logits of 2^24 is more than one and past 2^27 more than f16's weights can hold
// (0.7 to 3.5 % of the time; a branch for large references cost as much).
//
// f32 operands: two f16 parts of every value after a power-of-two scale, each 16 keys of a head of k and
// of v with one of their own (beforehand, attention_split_kernel), each query row with its own (as its CTA
// begins). A value is held to 2^-22 of itself or 2^-39 of the largest that it shares the scale with, whichever
// is more, and no other block's values matter. Three products (lo·hi, hi·lo, hi·hi; lo·lo is 2^-22 of the
// whole), and the weights in two parts after a scale of 2^7. The scales of k go into the factor of the
// exponents, those of v into what the weights are relative to: with x = log2 of a weight and 2^e the scale of
// its v, O gathers 2^(x − e − m) times the scaled v, m being the running maximum of x − e, while the sum of
// weights is relative to that of x. Both are whole numbers, so every rescaling is exact.
// The tensor core truncates as it adds into its f32 accumulator, so a long sum there drifts by about 2^-25 a
// step: the softmax threads add each tile's P·V to a second set of TMEM columns, rounding to nearest, and the
// next tile begins a fresh sum. (16 x 4096 x 8 x 40 over 1024 keys, relative to the exact result: 3.2e-7, with
// sums over two tiles 5.5e-7 and 1 % less time; a plain f32 softmax has 5.9e-7. With 80 channels 3.2e-7 against
// 5.5e-7 and 7 % less time; plain 5.1e-7.)
//
// Masked keys: S becomes −inf; their V rows become zero in shared memory (16-bit) or while
// splitting (f32), since zero times what a mask hides may be NaN.
// Measured on a B200, in a burst of ten calls and in a run of two seconds, in which the card clocks down:
// 32768 queries x 16 heads x 128 bf16 over 2048 keys each in 546 and 615 us (1007 and 894 TFLOP/s; tensor cores
// 50 % busy, exponentials 51 %), 2 x 16384 x 16 x 64 f16 over 2048 keys in 450 and 457 us (611 and 601 TFLOP/s;
// exponentials 59 %), 16 x 4096 x 8 x 40 f32 over 1024 keys in 521 and 563 us with the split (165 and 153 TFLOP/s,
// three times that in products).
// Every wait is bounded; on timeout the CTA records the error, waits (bounded) for its copies and
// MMAs in flight, frees TMEM and returns. It looks for them when every warp has stopped: a producer may be through
// with its part before another warp gives up.
#include <algorithm>
#include <type_traits>

#include "block_attention.h"
#include "mbx_device.cuh"
#include "mbx_tc.cuh"

namespace mbx {
namespace {

constexpr int kRows = MBX_ATTENTION_BLOCK_Q;
constexpr uint32_t kQPanel = kRows * 128;   // bytes of 64 channels of the query block
constexpr int kThreads = 224;
// Tiles whose bits of valid keys are kept: a slot is written again 8 tiles on, when Q·Kᵀ of a tile at most 4 before
// that is complete, which was begun when the tile two before it, or a later one, had been read.
constexpr int kMaskSlots = 8;
constexpr float kLazy = 8.0f;   // log2 of the largest weight
constexpr int kWeightExp = 7;   // f32 operands: weights are scaled by 2^7 before their split, up to 2^15
constexpr int kScaleExp = 14;   // f32 operands: the largest magnitude is scaled to [2^14, 2^15)
constexpr int kChunk = 16;      // f32 operands: keys that share a scale; every block is a multiple
constexpr float kNone = -1e30f;  // f32 operands: the running maximum before the first key

struct TcArgs {
    AttnArgs a;
    const int32_t* exps;  // f32 operands: exponents of the scales, k and then v, [n][kv_heads][chunks] each
    int chunks;
    int64_t n;
    int* err;
};

// The two layouts (above).
template <int PANELS, bool SPLIT>
constexpr bool own_p() {
    return PANELS == 1 && !SPLIT;
}
template <int PANELS, bool SPLIT>
constexpr int keys_of() {
    return own_p<PANELS, SPLIT>() ? 128 : 64;
}
template <int PANELS, bool SPLIT>
constexpr uint32_t col_o() {
    return own_p<PANELS, SPLIT>() ? 128 + 64 : 2 * 64;
}
template <int PANELS, bool SPLIT>
constexpr uint32_t tmem_cols() {
    return col_o<PANELS, SPLIT>() + PANELS * 64 * (SPLIT ? 2 : 1) <= 256 ? 256 : 512;
}
constexpr int kStages = 2;  // tiles of K, and of V, in shared memory

template <int PANELS, bool SPLIT>
constexpr int smem_of() {
    return PANELS * (SPLIT ? 2 : 1) * (int)(kQPanel + 2 * kStages * keys_of<PANELS, SPLIT>() * 128) + 1024;
}

// Columns of the warp's 32 lanes, complete on return: the wait is part of the statement, so that nothing that uses the
// registers can be moved before it.
__device__ __forceinline__ void tmem_ld16_wait(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {"
        "%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15 "
        "}, [%16];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_ld64_wait(uint32_t taddr, uint32_t (&r)[64]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x64.b32 {"
        "%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, "
        "%21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32, %33, %34, %35, %36, %37, %38, %39, "
        "%40, %41, %42, %43, %44, %45, %46, %47, %48, %49, %50, %51, %52, %53, %54, %55, %56, %57, %58, "
        "%59, %60, %61, %62, %63 "
        "}, [%64];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]),
          "=r"(r[32]), "=r"(r[33]), "=r"(r[34]), "=r"(r[35]), "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]),
          "=r"(r[40]), "=r"(r[41]), "=r"(r[42]), "=r"(r[43]), "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]),
          "=r"(r[48]), "=r"(r[49]), "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), "=r"(r[55]),
          "=r"(r[56]), "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]), "=r"(r[62]), "=r"(r[63])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_st16_u32(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {"
        "%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16 "
        "};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
        "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ float max3(float a, uint32_t b, uint32_t c) {
    float y;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(__uint_as_float(b)), "f"(__uint_as_float(c)));
    return y;
}

__device__ __forceinline__ uint32_t pack2(float lo, float hi, __half) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi, __nv_bfloat16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// The exponent of the power of two that scales values whose largest magnitude has these bits; zeros ask for as little
// room as the smallest values.
__device__ __forceinline__ int scale_exponent(uint32_t bits) {
    return min(kScaleExp + 127 - max((int)(bits >> 23), 1), 126);
}
// 2^d for a whole number d, 0 for one of -127 or less.
__device__ __forceinline__ float pow2(float d) {
    d = fminf(fmaxf(d, -127.0f), 127.0f);
    return __uint_as_float((__float_as_uint(d + 12582912.0f) + 127u) << 23);  // 3 · 2^22: d in the low bits
}
// The larger of two magnitudes' bits, of finite values.
__device__ __forceinline__ uint32_t larger(uint32_t bits, float v) {
    const uint32_t b = __float_as_uint(v) & 0x7fffffffu;
    return b < 0x7f800000u ? max(bits, b) : bits;
}
// A value as two f16 parts, packed pairwise: hi = v rounded, lo = the rest rounded.
__device__ __forceinline__ void split2(float a, float b, uint32_t& hi, uint32_t& lo) {
    const __half2 h = __floats2half2_rn(a, b);
    const float2 f = __half22float2(h);
    float x, y;
    unpair(fma2(pair(f.x, f.y), pair(-1.0f, -1.0f), pair(a, b)), x, y);
    const __half2 r = __floats2half2_rn(x, y);
    hi = *reinterpret_cast<const uint32_t*>(&h), lo = *reinterpret_cast<const uint32_t*>(&r);
}

// Shared-memory descriptor of an N-major operand (rows are K): 64-channel panels of 128-byte rows,
// 128-byte swizzle; 8-row groups 1024 bytes apart (SBO), panels `panel` bytes apart (LBO).
__device__ __forceinline__ uint64_t sw128_desc_mn(uint32_t saddr, uint32_t panel) {
    uint64_t d = 0;
    d |= (uint64_t)((saddr & 0x3ffffu) >> 4);
    d |= (uint64_t)(panel >> 4) << 16;
    d |= (uint64_t)(1024 >> 4) << 32;
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)2 << 61;
    return d;
}

// Instruction descriptor, kind::f16: D f32, A and B both f16 or both bf16, M = 128, N = n.
__device__ __forceinline__ uint32_t idesc_16(bool bf16, int n, bool negate_a, bool b_mn) {
    return (1u << 4) | ((uint32_t)bf16 << 7) | ((uint32_t)bf16 << 10) | ((uint32_t)negate_a << 13) |
           ((uint32_t)b_mn << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(kRows >> 4) << 24);
}

__device__ __forceinline__ void mma_16_ss(uint32_t d, uint64_t ad, uint64_t bd, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(ad), "l"(bd), "r"(idesc), "r"(accumulate)
        : "memory");
}

__device__ __forceinline__ void mma_16_ts(uint32_t d, uint32_t a, uint64_t bd, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a), "l"(bd), "r"(idesc), "r"(accumulate)
        : "memory");
}

// One lane of a converged warp.
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}

template <class OUT>
constexpr bool is_f32() {
    return std::is_same<OUT, float>::value;
}

// After a timeout, when every warp has stopped: MMAs in flight finish before TMEM is freed, and copies land before the
// CTA's memory is given up. Out of line, as the kernel needs its registers.
struct Settle {
    int fin, q_full, k_full, v_full;
    bool split;
    int stages;
};
__device__ __noinline__ void settle(uint32_t bars, Settle s, const int* issued, int* err) {
    const long long deadline = clock64() + kWaitLimit;
    const int warp = threadIdx.x >> 5;
    auto drain = [&](int b, int phase, int site) {
        drain_wait(bars + 8u * (uint32_t)b, (uint32_t)phase & 1u, deadline, err, site, kKAttention);
    };
    if (warp == 5) {
        if (elect_one()) {  // the lane that issued them
            mma_commit(bars + 8u * (uint32_t)s.fin);
            drain(s.fin, 0, 34);
        }
        __syncwarp();
    } else if (warp >= 4 && (threadIdx.x & 31) == 0) {
        const int v = warp == 6, done = issued[v];
        if (!s.split && !v && done > 0) drain(s.q_full, 0, 40);  // Q comes with tile 0, which waits for nothing
        for (int i = max(0, done - s.stages); i < done; ++i) drain((v ? s.v_full : s.k_full) + i % s.stages, i / s.stages, 40);
    }
    __syncthreads();
}

// OUT: the type of the tensors; the operands' type is OUT, or f16 parts where OUT is float.
template <class OUT, int PANELS>
__global__ void __launch_bounds__(kThreads, is_f32<OUT>() && PANELS == 2 ? 1 : 2)
    attention_tc_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                        const __grid_constant__ CUtensorMap map_v, const __grid_constant__ TcArgs args) {
    cudaGridDependencySynchronize();
    constexpr bool SPLIT = is_f32<OUT>();
    constexpr bool BF16 = std::is_same<OUT, __nv_bfloat16>::value;
    constexpr int PLANES = SPLIT ? 2 : 1;
    constexpr int STAGES = kStages, KEYS = keys_of<PANELS, SPLIT>(), WORDS = KEYS / 32;
    constexpr uint32_t kPanel = KEYS * 128;            // bytes of 64 channels of a tile of K or V
    constexpr uint32_t OP = PANELS * PLANES * kPanel;  // bytes of a tile of K or V
    constexpr uint32_t TMEM = tmem_cols<PANELS, SPLIT>(), kColO = col_o<PANELS, SPLIT>();
    constexpr bool OWN_P = own_p<PANELS, SPLIT>();
    constexpr int NS = OWN_P ? 1 : 2;  // S tiles
    constexpr uint32_t PCOL = OWN_P ? KEYS : 0;
    constexpr int DCOLS = PANELS * 64;
    using Part = typename std::conditional<BF16, __nv_bfloat16, __half>::type;
    const AttnArgs& a = args.a;

    // Barriers of S and P, one for each S tile, and of O, one for even and one for odd tiles: a waiter is then never two
    // phases behind, which a parity could not tell from none.
    enum {
        kKFull = 0,
        kKEmpty = kKFull + STAGES,
        kVFull = kKEmpty + STAGES,
        kVEmpty = kVFull + STAGES,
        kVClean = kVEmpty + STAGES,
        kQFull = kVClean + STAGES,
        kSFull,                 // [NS] a tile's S is complete
        kSEmpty = kSFull + NS,  // and read, where P has columns of its own
        kPFull,                 // [NS] a tile's weights are written
        kOFull = kPFull + NS,   // [2] a tile's P·V is complete
        kOEmpty = kOFull + 2,  // f32: a tile's sum is taken
        kFin,
        kBars
    };
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t bars[kBars];
    __shared__ volatile uint32_t valid[kMaskSlots][4];
    __shared__ __align__(16) float k_unscale[SPLIT ? kMaskSlots : 1][4], v_exp[SPLIT ? kMaskSlots : 1][4];  // of 16 keys each
    __shared__ uint32_t q_top[SPLIT ? kRows : 1];  // f32: bits of the query rows' largest magnitudes
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_flag, issued[2];  // issued: tiles of K, of V whose copies were begun
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* gbase = smem_raw + (base - smem_u32(smem_raw));
    const uint32_t sv = base, sk = sv + STAGES * OP, sq = sk + STAGES * OP;
    const uint32_t bar0 = smem_u32(bars);
    auto bar = [&](int i) { return bar0 + 8u * (uint32_t)i; };

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t cta = blockIdx.x / (uint32_t)a.splits;  // (item, head, query block)
    const int split = (int)(blockIdx.x - cta * a.splits);
    const uint32_t head_at = cta / (uint32_t)a.q_blocks;
    const int qb = (int)(cta - head_at * a.q_blocks);
    const int item = (int)(head_at / (uint32_t)a.heads);
    const int h = (int)(head_at - (uint32_t)item * a.heads);
    const int kh = h / (a.heads / a.kv_heads);
    const int32_t* list = a.index + (int64_t)cta * a.topk;
    const uint8_t* mask = a.mask ? a.mask + (int64_t)item * a.nk : nullptr;
    const bool cleans = !SPLIT && mask != nullptr;

    // Entries up to the last one that names a block: every warp looks for itself, while the rest is set up.
    int listed = 0;
#pragma unroll 2
    for (int e = lane; e < (int)a.topk; e += 32)
        if ((uint32_t)list[e] < (uint32_t)a.k_blocks) listed = e + 1;
    if (threadIdx.x == 0) {
        for (int i = 0; i < STAGES; ++i) {
            mbar_init(bar(kKFull + i), 1), mbar_init(bar(kKEmpty + i), 1);
            mbar_init(bar(kVFull + i), 1), mbar_init(bar(kVEmpty + i), 1), mbar_init(bar(kVClean + i), 1);
        }
        for (int i = 0; i < NS; ++i) mbar_init(bar(kSFull + i), 2), mbar_init(bar(kPFull + i), 4);
        for (int i = 0; i < 2; ++i) mbar_init(bar(kOFull + i), 1);
        mbar_init(bar(kSEmpty), 4);
        mbar_init(bar(kQFull), SPLIT ? 4 : 1), mbar_init(bar(kOEmpty), 4), mbar_init(bar(kFin), 1);
        abort_flag = 0;
        fence_mbarrier_init();
    }
    if (SPLIT && threadIdx.x < kRows) q_top[threadIdx.x] = 0;
    if (warp == 5) {
        tmem_alloc(smem_u32(&tmem_slot), TMEM);
        tmem_relinquish();
    }
    listed = __reduce_max_sync(0xffffffffu, listed);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    const int rows_box = min(a.block_k, KEYS), boxes = KEYS / rows_box;  // TMA boxes of a tile
    const int all_tiles = (int)(((int64_t)listed * a.block_k + KEYS - 1) / KEYS);
    const int t0 = a.splits == 1 ? 0 : (int)((uint32_t)all_tiles * split / (uint32_t)a.splits);  // at most 2^17 · 64
    const int tiles = a.splits == 1 ? all_tiles : (int)((uint32_t)all_tiles * (split + 1) / (uint32_t)a.splits) - t0;
    volatile int* abort_p = &abort_flag;
    auto wait = [&](int b, int phase, int site) {
        return mbar_wait(bar(b), (uint32_t)phase & 1u, args.err, site, abort_p, true, kWaitLimit, kKAttention);
    };

    // The same answer in every lane: what follows is done by whole warps.
    auto warp_wait = [&](int b, int phase, int site) { return __all_sync(0xffffffffu, wait(b, phase, site)) != 0; };

    if (warp < 4) {
        // ---------------------------------------------------------------- softmax
        const uint32_t lanes = tmem + ((uint32_t)(warp * 32) << 16);
        const int64_t row = (int64_t)qb * kRows + threadIdx.x;
        // One arrival for the warp, after everything that its lanes have done.
        auto arrive = [&](int b) {
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(b));
        };
        // A negative scale negates Q in the instruction descriptor. The least normal value in place of 0 (a scale of
        // 0, or far below what matters) keeps −inf · c = −inf.
        float c = fabsf(a.scale);
        if constexpr (SPLIT) {
            // Q in two parts, a row at a power of two of its own. A warp reads whole rows: a lane takes pieces of eight
            // channels, and the rows' magnitudes meet in shared memory.
            const int pieces = a.dim >> 3, wide = (a.dim + 15) / 16 * 2;  // of a row of q; of the operand, to 16 channels
            const float* x = static_cast<const float*>(a.q) + ((int64_t)item * a.nq + (int64_t)qb * kRows) * a.q_stride +
                             (int64_t)h * a.dim;
            constexpr int MOST = PANELS * 8;
            Raw8f raw[MOST];
#pragma unroll
            for (int k = 0; k < MOST; ++k) {
                const int i = (int)threadIdx.x + k * kRows, r = i / wide, p = i - r * wide;
                raw[k] = Raw8f{};
                if (r < kRows && p < pieces && (int64_t)qb * kRows + r < a.nq)
                    raw[k] = load_raw8(x + r * a.q_stride + p * 8);
            }
#pragma unroll
            for (int k = 0; k < MOST; ++k) {
                const int r = ((int)threadIdx.x + k * kRows) / wide;
                float v[8];
                widen8<float>(raw[k], v);
                uint32_t top = 0;
#pragma unroll
                for (int e = 0; e < 8; ++e) top = larger(top, v[e]);
                if (r < kRows && top) atomicMax(&q_top[r], top);
            }
            asm volatile("bar.sync 1, 128;" ::: "memory");  // the four softmax warps, none of which can have given up yet
#pragma unroll
            for (int k = 0; k < MOST; ++k) {
                const int i = (int)threadIdx.x + k * kRows, r = i / wide, p = i - r * wide;
                if (r >= kRows) continue;
                const float f = ldexpf(1.0f, scale_exponent(q_top[r]));
                float v[8];
                widen8<float>(raw[k], v);
                uint32_t hi[4], lo[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) split2(v[2 * e] * f, v[2 * e + 1] * f, hi[e], lo[e]);
                uint8_t* to = gbase + (sq - base) + (p >> 3) * kQPanel + r * 128 + ((p & 7) ^ (r & 7)) * 16;  // swizzled
                *reinterpret_cast<uint4*>(to) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                *reinterpret_cast<uint4*>(to + PANELS * kQPanel) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
            }
            fence_proxy_async_smem();
            arrive(kQFull);
            c = ldexpf(c, -scale_exponent(q_top[threadIdx.x]));
        }
        if (!SPLIT) c = fmaxf(c, 1.17549435e-38f);  // f32: with the scale of k in it
        // What the weights are relative to, in units of S, and their sum. f32: log2 of what the sum is relative to, and of
        // what O is, relative to that.
        float ref = SPLIT ? kNone : -INFINITY, l = 0.0f, off_o = 0.0f;
        // O's columns, 16 at a time, as far as there are channels.
        auto columns = [&](auto&& f) {
#pragma unroll
            for (int i = 0; i < DCOLS; i += 16)
                if (i < a.dim) f(i);
        };
        bool ok = true;
        for (int j = 0; j < tiles; ++j) {
            const int slot = j % kMaskSlots;
            const int b = j % NS;
            const uint32_t sp = lanes + b * KEYS, pp = lanes + PCOL + b * KEYS;  // its S and P
            ok = warp_wait(kSFull + b, j / NS, 21);
            if (!ok) break;
            tc_fence_after();
            uint32_t w[WORDS], some = 0xffffffffu;
#pragma unroll
            for (int i = 0; i < WORDS; ++i) w[i] = valid[slot][i], some &= w[i];
            uint32_t s[64];
            auto read = [&](int q) {  // 64 columns of S
                tmem_ld64_wait(sp + q * 64, s);
                if (some != 0xffffffffu) {
#pragma unroll
                    for (int i = 0; i < 64; ++i)
                        if (!(w[q * 2 + (i >> 5)] >> (i & 31) & 1u)) s[i] = 0xff800000u;
                }
            };
            // Maxima of 16 keys each for f32 operands, whose scales differ.
            float t[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int q = 0; q < KEYS / 64; ++q) {
                read(q);
#pragma unroll
                for (int i = 0; i < 64; i += 2) {
                    const int u = SPLIT ? i / kChunk : i >> 1 & 3;
                    t[u] = max3(t[u], s[i], s[i + 1]);
                }
            }
            constexpr int CHUNKS = SPLIT ? 4 : 1;
            float cs[CHUNKS], raw[CHUNKS];  // factor of S in the exponent; f32: the largest S, and in t times the factor
            float top, top_o = 0.0f;
            bool raise;
            if constexpr (SPLIT) {
                const float4 fk = *reinterpret_cast<const float4*>(k_unscale[slot]), e = *reinterpret_cast<const float4*>(v_exp[slot]);
                const float fks[4] = {fk.x, fk.y, fk.z, fk.w}, es[4] = {e.x, e.y, e.z, e.w};
                top = top_o = -INFINITY;
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    cs[u] = fmaxf(c * fks[u], 1.17549435e-38f);
                    raw[u] = t[u];
                    t[u] *= cs[u];
                    top = fmaxf(top, t[u]), top_o = fmaxf(top_o, t[u] - ref - es[u]);
                }
                raise = top - ref > kLazy || top_o - off_o > kLazy;
            } else {
                cs[0] = c;
                top = fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3]));
                raise = ref == -INFINITY ? top > ref : (top - ref) * c > kLazy;
            }
            // Raise the reference when a weight would pass 2^8.
            if (__any_sync(0xffffffffu, raise)) {
                float f = 1.0f;
                if constexpr (SPLIT) {
                    if (raise) {
                        const float4 e = *reinterpret_cast<const float4*>(v_exp[slot]);
                        const float es[4] = {e.x, e.y, e.z, e.w};
                        const float up = top - ref > kLazy ? ceilf(top) : ref, was = fmaxf(off_o - (up - ref), -1000.0f);
                        l *= pow2(ref - up);
                        ref = up, off_o = was;
#pragma unroll
                        for (int u = 0; u < 4; ++u)
                            if (t[u] - ref - es[u] - was > kLazy) off_o = fmaxf(off_o, ceilf(t[u] - ref - es[u]));
                        f = pow2(was - off_o);
                    }
                } else {
                    if (raise) {
                        f = ref == -INFINITY ? 0.0f : ex2((ref - top) * c);
                        ref = top;
                    }
                    l *= f;
                }
                if (j > 0) {
                    ok = warp_wait(kOFull + ((j - 1) & 1), (j - 1) >> 1, 22);
                    if (!ok) break;
                    tc_fence_after();
#pragma unroll
                    for (int r = 0; r < (SPLIT ? 2 : 1); ++r) {
                        if (r == 1 && j == 1) continue;  // nothing has been taken yet
                        columns([&](int i) {
                            uint32_t o[16];
                            tmem_ld16_wait(lanes + kColO + r * DCOLS + i, o);
#pragma unroll
                            for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                            tmem_st16_u32(lanes + kColO + r * DCOLS + i, o);
                        });
                    }
                }
            }
            if (OWN_P && j > 0) {  // P of the last tile has been read
                ok = warp_wait(kOFull + ((j - 1) & 1), (j - 1) >> 1, 23);
                if (!ok) break;
                tc_fence_after();
            }
            // A weight is 2^((S - from) cs - less). f32: from is the chunk's largest S; off is log2 of what the weights are
            // relative to, beside ref.
            float from[CHUNKS], less[CHUNKS], off[CHUNKS];
            if constexpr (SPLIT) {
                // Where v is so small that its weights would be lost to the sum, they are kept, but below what counts for O.
                const float4 e = *reinterpret_cast<const float4*>(v_exp[slot]);
                const float es[4] = {e.x, e.y, e.z, e.w};
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const float d = fmaxf(t[u] - ref, -65536.0f);
                    from[u] = raw[u] == -INFINITY ? 0.0f : raw[u];
                    off[u] = fminf(off_o + es[u], ceilf(d) + 60.0f) - (float)kWeightExp, less[u] = off[u] - d;
                }
            } else {
                from[0] = ref == -INFINITY ? 0.0f : ref;
            }
            uint64_t sum = 0;
            auto gather = [&](float factor) {
                float l0, l1;
                unpair(sum, l0, l1);
                l = SPLIT ? fmaf(factor, l0 + l1, l) : l + (l0 + l1);
                sum = 0;
            };
#pragma unroll
            for (int q = KEYS / 64 - 1; q >= 0; --q) {  // the last 64 keys first: they are in registers
                if (q < KEYS / 64 - 1) {
                    read(q);
                    tc_fence_before();
                    arrive(kSEmpty);
                }
#pragma unroll
                for (int g = 0; g < 2; ++g) {  // 32 keys: 16 columns of P, and for f32 16 more of its low part
                    uint32_t hi[16], lo[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const int at = g * 32 + 2 * i, u = SPLIT ? at / kChunk : 0;
                        const uint64_t x = add2(pair(__uint_as_float(s[at]), __uint_as_float(s[at + 1])), pair(-from[u], -from[u]));
                        float p0, p1;
                        unpair(SPLIT ? fma2(x, pair(cs[u], cs[u]), pair(-less[u], -less[u])) : mul2(x, pair(c, c)), p0, p1);
                        p0 = ex2(p0), p1 = ex2(p1);
                        sum = add2(sum, pair(p0, p1));
                        if (SPLIT && (at + 2) % kChunk == 0) gather(pow2(off[u] + (float)kWeightExp));
                        if constexpr (SPLIT)
                            split2(p0, p1, hi[i], lo[i]);
                        else
                            hi[i] = pack2(p0, p1, Part());
                    }
                    tmem_st16_u32(pp + q * 32 + g * 16, hi);
                    if (SPLIT) tmem_st16_u32(pp + 32 + g * 16, lo);
                }
            }
            if (!SPLIT) gather(1.0f);
            tmem_wait_st();
            tc_fence_before();
            arrive(kPFull + b);
            if (SPLIT && j > 0) {
                ok = warp_wait(kOFull + ((j - 1) & 1), (j - 1) >> 1, 25);
                if (!ok) break;
                tc_fence_after();
                columns([&](int i) {
                    uint32_t o[16];
                    tmem_ld16_wait(lanes + kColO + i, o);
                    if (j > 1) {
                        uint32_t r[16];
                        tmem_ld16_wait(lanes + kColO + DCOLS + i, r);
#pragma unroll
                        for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) + __uint_as_float(r[e]));
                    }
                    tmem_st16_u32(lanes + kColO + DCOLS + i, o);
                });
                tmem_wait_st();
                tc_fence_before();
                arrive(kOEmpty);
            }
        }
        if (ok && tiles > 0) ok = warp_wait(kOFull + ((tiles - 1) & 1), (tiles - 1) >> 1, 26);
        if (ok) {
            tc_fence_after();
            const bool store = row < a.nq;
            const int64_t at = ((int64_t)item * a.nq + row) * a.heads + h;
            // One factor for the row: 1 / l, or for a share of the list 1. f32: the weights' own scale taken out, and what O
            // is relative to turned into what the sum is, in two steps as the power of two may leave f32's range.
            float f = a.splits > 1 ? (SPLIT ? 1.0f / (1 << kWeightExp) : 1.0f) : (l == 0.0f ? 0.0f : 1.0f / l), f2 = 1.0f;
            if constexpr (SPLIT) {
                const float half = floorf(0.5f * off_o);
                f *= pow2(half), f2 = pow2(off_o - half);
            }
            float* part = a.part + (at * a.splits + split) * (a.dim + 4);
            if (a.splits > 1 && store) {
                part[a.dim] = l == 0.0f ? -INFINITY : (SPLIT ? ref : ref * c);
                part[a.dim + 1] = SPLIT ? l / (1 << kWeightExp) : l;
            }
            columns([&](int i) {
                uint32_t o[16], r[16];
                if (tiles > 0) tmem_ld16_wait(lanes + kColO + i, o);
                if (SPLIT && tiles > 1) tmem_ld16_wait(lanes + kColO + DCOLS + i, r);
#pragma unroll
                for (int g = 0; g < 16; g += 8) {
                    float y[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        float v = __uint_as_float(o[g + e]);
                        if (SPLIT && tiles > 1) v += __uint_as_float(r[g + e]);
                        y[e] = l == 0.0f ? 0.0f : (SPLIT ? v * f * f2 : v * f);
                    }
                    if (!store || i + g >= a.dim) continue;
                    if (a.splits > 1)
                        store8(part + i + g, y);
                    else if (!SPLIT && a.out_f32)
                        store8(static_cast<float*>(a.out) + at * a.dim + i + g, y);
                    else
                        store8(static_cast<OUT*>(a.out) + at * a.dim + i + g, y);
                }
            });
        }
    } else if (warp != 5) {
        // ---------------------------------------------------------------- producer
        auto load = [&](const CUtensorMap* map, uint32_t dst, uint32_t bytes, int full_bar, int head, int token,
                        int n_boxes, int rows) {  // one lane for each box of `rows` rows
            if (lane == 0) mbar_arrive_expect_tx(bar(full_bar), bytes);
            __syncwarp();
            if (lane < n_boxes) {
#pragma unroll
                for (int p = 0; p < PLANES * PANELS; ++p)
                    tma_load_4d(dst + p * (bytes / (PLANES * PANELS)) + lane * rows * 128, map, (p % PANELS) * 64, head,
                                token, item + (p / PANELS) * (int)args.n, bar(full_bar));
            }
            __syncwarp();
        };
        const bool is_v = warp == 6;
        int done = 0;
        if (!SPLIT && !is_v && tiles > 0) load(&map_q, sq, PANELS * kQPanel, kQFull, h, qb * kRows, 1, kRows);
        // The list and the mask are read ahead of the tiles that they are for: a lane holds the first token of one
        // box (32 / boxes tiles at a time, the next ones on their way), and its keys' mask bytes of the next tile.
        const int lg_block = 31 - __clz(a.block_k), lg_rows = 31 - __clz(rows_box), lg_boxes = 31 - __clz(boxes);
        const int batch = 32 >> lg_boxes;
        auto first_token = [&](int tile) {  // of this lane's box in the batch that begins with `tile`
            const int at = (t0 + tile) * KEYS + (lane << lg_rows), e = at >> lg_block;  // in the list's keys
            const int blk = e < listed ? list[e] : -1;
            return (uint32_t)blk < (uint32_t)a.k_blocks ? (blk << lg_block) + (at & (a.block_k - 1))
                                                        : (int)a.nk;  // past the last key: zeros
        };
        auto cut = [&](int t) {  // the batch's boxes with a key past the last one
            return __ballot_sync(0xffffffffu, (int64_t)t + rows_box > a.nk);
        };
        int tokens = first_token(0), tokens_next = tiles > batch ? first_token(batch) : 0;
        uint32_t short_boxes = cut(tokens);
        const uint32_t box_bits = (1u << boxes) - 1;
        uint8_t keep[WORDS];
        int64_t t_key[WORDS];
        bool checks = false;  // the tile's keys are looked at one by one
        int k_exp = 0, v_scale = 0;  // f32: the scales of the next tile's 16 keys that lanes 0-3 look after
        auto look_up = [&](int j) {
            const int box0 = (j & (batch - 1)) << lg_boxes;
            if (SPLIT && !is_v) {
                const int key = (lane & 3) * kChunk;
                const int64_t t = (int64_t)__shfl_sync(0xffffffffu, tokens, box0 + (key >> lg_rows)) + (key & (rows_box - 1));
                const int32_t* exps = args.exps + ((int64_t)item * a.kv_heads + kh) * args.chunks + t / kChunk;
                const bool in = t < a.nk;
                k_exp = in ? exps[0] : 0, v_scale = in ? exps[args.n * a.kv_heads * args.chunks] : 0;
            }
            checks = is_v ? cleans : mask || (short_boxes >> box0 & box_bits);
            if (!checks) return;
#pragma unroll
            for (int i = 0; i < WORDS; ++i) {
                const int key = i * 32 + lane;
                t_key[i] = (int64_t)__shfl_sync(0xffffffffu, tokens, box0 + (key >> lg_rows)) + (key & (rows_box - 1));
                keep[i] = t_key[i] < a.nk && (!mask || mask[t_key[i]]);
            }
        };
        if (tiles > 0) look_up(0);
        for (int j = 0; j < tiles; ++j) {
            const int st = j % STAGES, ph = j / STAGES, slot = j % kMaskSlots;
            const int token = __shfl_sync(0xffffffffu, tokens, ((j & (batch - 1)) << lg_boxes) + (lane & (boxes - 1)));
            uint32_t w[WORDS];
            bool hidden = false;
#pragma unroll
            for (int i = 0; i < WORDS; ++i) w[i] = 0xffffffffu;
            if (checks) {
#pragma unroll
                for (int i = 0; i < WORDS; ++i) {
                    w[i] = __ballot_sync(0xffffffffu, keep[i] != 0);
                    hidden |= t_key[i] < a.nk && !keep[i];
                }
                hidden = __any_sync(0xffffffffu, hidden);
            }
            if (j >= STAGES && !warp_wait((is_v ? kVEmpty : kKEmpty) + st, ph - 1, 38)) break;
            if (is_v) {
                load(&map_v, sv + st * OP, OP, kVFull + st, kh, token, boxes, rows_box);
            } else {
                if (lane == 0) {  // handed on with K, then with S
#pragma unroll
                    for (int i = 0; i < WORDS; ++i) valid[slot][i] = w[i];
                }
                if (SPLIT) {
                    if (lane < 4) k_unscale[slot][lane] = pow2((float)-k_exp), v_exp[slot][lane] = (float)v_scale;
                    __syncwarp();
                }
                load(&map_k, sk + st * OP, OP, kKFull + st, kh, token, boxes, rows_box);
            }
            done = j + 1;
            if (((j + 1) & (batch - 1)) == 0) {
                tokens = tokens_next;
                short_boxes = cut(tokens);
                if (j + 1 + batch < tiles) tokens_next = first_token(j + 1 + batch);
            }
            if (j + 1 < tiles) look_up(j + 1);
            if (is_v && cleans) {
                if (hidden) {
                    if (!warp_wait(kVFull + st, ph, 37)) break;
#pragma unroll
                    for (int i = 0; i < WORDS; ++i)
                        for (uint32_t gone = ~w[i]; gone; gone &= gone - 1) {
                            const int r = i * 32 + __ffs(gone) - 1;
#pragma unroll
                            for (int p = 0; p < PANELS; ++p)
                                *reinterpret_cast<uint32_t*>(gbase + st * OP + p * kPanel + r * 128 + lane * 4) = 0;
                        }
                    fence_proxy_async_smem();
                    __syncwarp();
                }
                if (lane == 0) mbar_arrive(bar(kVClean + st));
            }
        }
        if (lane == 0) issued[is_v] = done;
    } else if (tiles > 0) {
        // ---------------------------------------------------------------- MMA issuer
        // The whole warp walks the loop, so that descriptors stay in uniform registers; one lane issues.
        const bool leader = elect_one();
        const int k_steps = (a.dim + 15) / 16;
        const uint32_t idesc_s = idesc_16(BF16, KEYS, a.scale < 0.0f, false);
        const uint32_t idesc_o = idesc_16(BF16, k_steps * 16, false, true);
        const uint64_t q_desc = sw128_desc(sq), k_desc = sw128_desc(sk), v_desc = sw128_desc_mn(sv, kPanel);
        auto scores = [&](int j) {  // S of tile j, when what its columns held is used up
            const int st = j % STAGES, b = j % NS;
            if (!warp_wait(kKFull + st, j / STAGES, 29)) return false;
            if (OWN_P && j >= 1 && !warp_wait(kSEmpty, j - 1, 30)) return false;
            if (!OWN_P && j >= 2 && !warp_wait(kOFull + (j & 1), (j - 2) >> 1, 30)) return false;
            tc_fence_after();
            if (leader) {
#pragma unroll
                for (int p = SPLIT ? 0 : 2; p < 3; ++p) {  // lo·hi, hi·lo, hi·hi
                    const uint64_t qa = q_desc + (p == 0 ? PANELS * kQPanel >> 4 : 0);
                    const uint64_t ka = k_desc + ((uint32_t)st * OP >> 4) + (p == 1 ? PANELS * kPanel >> 4 : 0);
#pragma unroll
                    for (int s = 0; s < 4 * PANELS; ++s)
                        if (s < k_steps)
                            mma_16_ss(tmem + b * KEYS, qa + ((s >> 2) * kQPanel + (s & 3) * 32 >> 4),
                                      ka + ((s >> 2) * kPanel + (s & 3) * 32 >> 4), idesc_s,
                                      (p > (SPLIT ? 0 : 2) || s > 0) ? 1u : 0u);
                }
                mma_commit(bar(kKEmpty + st));
                mma_commit(bar(kSFull + b));
                mbar_arrive(bar(kSFull + b));  // the producer's bits of valid keys, seen here, go on with S
            }
            __syncwarp();
            return true;
        };
        bool ok = warp_wait(kQFull, 0, 28) && scores(0) && (NS == 1 || tiles == 1 || scores(1));
        for (int j = 0; ok && j < tiles; ++j) {
            const int st = j % STAGES, ph = j / STAGES;
            if (OWN_P && j + 1 < tiles) ok = scores(j + 1);
            if (ok) ok = warp_wait(kPFull + j % NS, j / NS, 33);
            if (ok) ok = warp_wait(kVFull + st, ph, 31);
            if (ok && cleans) ok = warp_wait(kVClean + st, ph, 32);
            if (ok && SPLIT && j > 0) ok = warp_wait(kOEmpty, j - 1, 36);
            if (!ok) break;
            tc_fence_after();
            if (leader) {
#pragma unroll
                for (int p = SPLIT ? 0 : 2; p < 3; ++p) {
                    const uint64_t va = v_desc + ((uint32_t)st * OP >> 4) + (p == 1 ? PANELS * kPanel >> 4 : 0);
                    const uint32_t pa = tmem + PCOL + j % NS * KEYS + (p == 0 ? 32 : 0);
#pragma unroll
                    for (int s = 0; s < KEYS / 16; ++s) {
                        const bool fresh = s == 0 && (SPLIT ? p == 0 : j == 0);
                        mma_16_ts(tmem + kColO, pa + s * 8,
                                  va + (uint32_t)(s * 2048 >> 4), idesc_o, fresh ? 0u : 1u);
                    }
                }
                mma_commit(bar(kVEmpty + st));
                mma_commit(bar(kOFull + (j & 1)));
            }
            __syncwarp();
            if (!OWN_P && j + 2 < tiles) ok = scores(j + 2);
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (*abort_p)  // the same for all: nobody waits any more
        settle(smem_u32(bars), {kFin, kQFull, kKFull, kVFull, SPLIT, STAGES}, issued, args.err);
    if (warp == 5) tmem_dealloc(tmem, TMEM);
}

// ------------------------------------------------------------------------------------ f32 operands

struct SplitArgs {
    const float* x[2];    // k, v
    int64_t stride[2];    // elements between rows
    __half* parts[2];     // [2][n][rows][heads][dim]
    int32_t* exps;        // [2][n][heads][chunks]
    int64_t n, rows;
    int heads, dim, chunks;
    const uint8_t* mask;  // rows that count
};

constexpr int kSplitRows = 64;
constexpr int kSplitThreads = 256;

// One pass over k and v: 16 rows of a head get the power of two that their largest finite magnitude asks for, and are
// written as two parts. A CTA takes 64 rows of as many whole heads as 32 lanes hold, eight channels a lane; a thread
// has eight rows in registers while shared memory joins the magnitudes. Rows that the mask hides become zero.
__global__ void __launch_bounds__(kSplitThreads, 2) attention_split_kernel(const __grid_constant__ SplitArgs a) {
    cudaGridDependencySynchronize();
    constexpr int WARPS = kSplitThreads / 32, MINE = kSplitRows / WARPS, CHUNKS = kSplitRows / kChunk;
    __shared__ uint32_t tops[CHUNKS][32];
    const int t = blockIdx.y & 1, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int lanes = a.dim / 8, per = 32 / lanes, at = lane / lanes, head0 = (int)(blockIdx.y >> 1) * per;
    const int64_t item = blockIdx.z, r0 = (int64_t)blockIdx.x * kSplitRows;
    const bool on = at < per && head0 + at < a.heads;
    const int ch = head0 * a.dim + lane * 8;
    if (threadIdx.x < CHUNKS * 32) tops[warp][lane] = 0;
    __syncthreads();
    Raw8f raw[MINE];  // rows warp, warp + 8, …: two of each 16
#pragma unroll
    for (int i = 0; i < MINE; ++i) {
        const int64_t r = r0 + warp + i * WARPS, row = item * a.rows + r;
        raw[i] = Raw8f{};
        if (on && r < a.rows && (!a.mask || a.mask[row])) raw[i] = load_raw8(a.x[t] + row * a.stride[t] + ch);
    }
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
        uint32_t top = 0;
#pragma unroll
        for (int i = c * (MINE / CHUNKS); i < (c + 1) * (MINE / CHUNKS); ++i) {
            float v[8];
            widen8<float>(raw[i], v);
#pragma unroll
            for (int e = 0; e < 8; ++e) top = larger(top, v[e]);
        }
        if (on && top) atomicMax(&tops[c][at], top);
    }
    __syncthreads();
    const int64_t width = (int64_t)a.heads * a.dim, plane = a.n * a.rows * width;
#pragma unroll
    for (int i = 0; i < MINE; ++i) {
        const int64_t r = r0 + warp + i * WARPS;
        if (!on || r >= a.rows) continue;
        const float f = pow2((float)scale_exponent(tops[i / (MINE / CHUNKS)][at]));
        float v[8];
        widen8<float>(raw[i], v);
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) split2(v[2 * e] * f, v[2 * e + 1] * f, hi[e], lo[e]);
        uint4* out = reinterpret_cast<uint4*>(a.parts[t] + (item * a.rows + r) * width + ch);
        out[0] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        out[plane / 8] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
    }
    const int chunk = (int)(r0 / kChunk) + warp, head = head0 + lane;
    if (warp < CHUNKS && lane < per && head < a.heads && chunk < a.chunks)
        a.exps[((t * a.n + item) * a.heads + head) * a.chunks + chunk] = scale_exponent(tops[warp][lane]);
}

// A map over [items][rows][heads][dim] 16-bit values, boxes of 64 channels × one head × box_rows rows.
void encode_heads(CUtensorMap* map, const void* base, bool bf16, int64_t items, int64_t rows, int64_t heads,
                  int64_t dim, int64_t stride, int box_rows) {
    const uint64_t dims[4] = {(uint64_t)dim, (uint64_t)heads, (uint64_t)rows, (uint64_t)items};
    const uint64_t strides[3] = {(uint64_t)dim * 2, (uint64_t)stride * 2, (uint64_t)(rows * stride) * 2};
    const uint32_t box[4] = {64, 1, (uint32_t)box_rows, 1};
    encode_tensor_map_16(map, base, bf16, 4, dims, strides, box);
}

template <class OUT, int PANELS>
void launch_typed(mbx_ctx* ctx, const TcArgs& t, const CUtensorMap (&maps)[3]) {
    const int64_t ctas = t.n * t.a.heads * t.a.q_blocks * t.a.splits;
    MBX_REQUIRE(ctas < (int64_t(1) << 31), "block_attention: too many query blocks");
    constexpr int smem = smem_of<PANELS, is_f32<OUT>()>();
    ensure_smem_limit((const void*)attention_tc_kernel<OUT, PANELS>, smem, "attention_tc");
    launch_after(ctx, "attention_tc", attention_tc_kernel<OUT, PANELS>, dim3((unsigned)ctas), kThreads, smem, maps[0], maps[1],
                 maps[2], t);
}

}  // namespace

size_t attention_split_bytes(const BlockShape& s) {
    return align256(4 * 2 * (size_t)(s.n * s.kv_heads * ((s.nk + kChunk - 1) / kChunk))) +
           2 * align256(2 * 2 * (size_t)(s.n * s.nk * s.kv_heads * s.dim));
}

void launch_attention_tc(mbx_ctx* ctx, const AttnArgs& a, int dtype, int64_t n, void* split) {
    TcArgs t{a, nullptr, 0, n, ctx->dev_err};
    CUtensorMap maps[3];
    const bool bf16 = dtype == MBX_DTYPE_BF16;
    const int rows_box = std::min(a.block_k, dtype != MBX_DTYPE_F32 && a.dim <= 64 ? keys_of<1, false>() : keys_of<2, false>());
    if (dtype == MBX_DTYPE_F32) {
        SplitArgs s{};
        s.chunks = (int)((a.nk + kChunk - 1) / kChunk);
        const size_t exps_bytes = align256(4 * 2 * (size_t)(n * a.kv_heads * s.chunks));
        const size_t part_bytes = align256(2 * 2 * (size_t)(n * a.nk * a.kv_heads * a.dim));
        s.exps = static_cast<int32_t*>(split);
        s.n = n, s.rows = a.nk, s.heads = a.kv_heads, s.dim = a.dim, s.mask = a.mask;
        s.x[0] = static_cast<const float*>(a.k), s.x[1] = static_cast<const float*>(a.v);
        s.stride[0] = a.k_stride, s.stride[1] = a.v_stride;
        for (int i = 0; i < 2; ++i)
            s.parts[i] = reinterpret_cast<__half*>(static_cast<uint8_t*>(split) + exps_bytes + i * part_bytes);
        const int per = 32 / (a.dim / 8);  // heads of a CTA
        const dim3 grid((unsigned)((a.nk + kSplitRows - 1) / kSplitRows),
                        (unsigned)(2 * ((a.kv_heads + per - 1) / per)), (unsigned)n);
        launch_after(ctx, "attention_split", attention_split_kernel, grid, kSplitThreads, 0, s);
        t.exps = s.exps, t.chunks = s.chunks;
        for (int i = 1; i < 3; ++i)
            encode_heads(&maps[i], s.parts[i - 1], false, 2 * n, a.nk, a.kv_heads, a.dim, (int64_t)a.kv_heads * a.dim,
                         rows_box);
        maps[0] = maps[1];  // q is split where it is used
    } else {
        encode_heads(&maps[0], a.q, bf16, n, a.nq, a.heads, a.dim, a.q_stride, kRows);
        encode_heads(&maps[1], a.k, bf16, n, a.nk, a.kv_heads, a.dim, a.k_stride, rows_box);
        encode_heads(&maps[2], a.v, bf16, n, a.nk, a.kv_heads, a.dim, a.v_stride, rows_box);
    }
    if (dtype == MBX_DTYPE_F32) return a.dim > 64 ? launch_typed<float, 2>(ctx, t, maps) : launch_typed<float, 1>(ctx, t, maps);
    if (dtype == MBX_DTYPE_F16) return a.dim > 64 ? launch_typed<__half, 2>(ctx, t, maps) : launch_typed<__half, 1>(ctx, t, maps);
    a.dim > 64 ? launch_typed<__nv_bfloat16, 2>(ctx, t, maps) : launch_typed<__nv_bfloat16, 1>(ctx, t, maps);
}

}  // namespace mbx
