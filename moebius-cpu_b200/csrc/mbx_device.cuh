// Device-side helpers shared by the kernels.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace mbx {

// x·σ(x) = x / (1 + e^−x), the reference's SiLU (src/engine/math.rs:34-36),
// evaluated with the hardware exponential and the approximate divide (within
// a few ulp); e^−x overflowing to +inf gives the correctly signed zero limit.
__device__ __forceinline__ float dev_silu(float x) { return __fdividef(x, 1.0f + __expf(-x)); }

// Loads of data read once (the read-only path); stores are plain so the
// result stays in L2 for the consumer kernel that usually follows.
template <class T>
__device__ __forceinline__ T ldg_stream(const T* p) {
    return __ldg(p);
}

template <class T>
__device__ __forceinline__ void stg_stream(T* p, const T& v) {
    *p = v;
}

// Thread mapping for per-item, per-channel streaming kernels over one item of
// hw pixels × cv channel vectors: each thread keeps one channel vector j (so its
// per-channel operands live in registers) and walks pixels p, p + rows_step, ...
// Returns false for threads with no channel vector (cv does not divide the block).
struct ChanStationary {
    int j;          // channel vector of this thread
    int64_t p0;     // first pixel
    int64_t step;   // pixel stride
    __device__ __forceinline__ bool init(int cv) {
        if (cv <= (int)blockDim.x) {
            const int rows = blockDim.x / cv;
            const int r = threadIdx.x / cv;
            if (r >= rows) return false;
            j = threadIdx.x - r * cv;
            p0 = (int64_t)blockIdx.x * rows + r;
            step = (int64_t)gridDim.x * rows;
        } else {
            j = threadIdx.x;  // caller loops j += blockDim.x
            p0 = blockIdx.x;
            step = gridDim.x;
        }
        return true;
    }
};

__device__ __forceinline__ float4 f4_fma(float4 a, float4 b, float4 c) {
    return make_float4(fmaf(a.x, b.x, c.x), fmaf(a.y, b.y, c.y), fmaf(a.z, b.z, c.z), fmaf(a.w, b.w, c.w));
}

// Two f32 in one register pair: sm_100 adds both, or multiplies and adds both, in one instruction, each as if alone.
__device__ __forceinline__ uint64_t pair(float lo, float hi) {
    uint64_t v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(lo), "f"(hi));
    return v;
}
__device__ __forceinline__ void unpair(uint64_t v, float& lo, float& hi) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}

// Eight consecutive elements of any of the storage types as f32, and back (rounded to nearest):
// one or two 16-byte accesses, so p must be 16-byte aligned.
struct Raw8f {
    float4 a, b;
};
template <class T>
struct Raw8 {
    using type = uint4;
};
template <>
struct Raw8<float> {
    using type = Raw8f;
};

__device__ __forceinline__ Raw8f load_raw8(const float* p) {
    return Raw8f{__ldg(reinterpret_cast<const float4*>(p)), __ldg(reinterpret_cast<const float4*>(p) + 1)};
}
template <class T>
__device__ __forceinline__ uint4 load_raw8(const T* p) {
    return __ldg(reinterpret_cast<const uint4*>(p));
}

template <class T>
__device__ __forceinline__ void widen8(const typename Raw8<T>::type& r, float (&v)[8]);
template <>
__device__ __forceinline__ void widen8<float>(const Raw8f& r, float (&v)[8]) {
    v[0] = r.a.x, v[1] = r.a.y, v[2] = r.a.z, v[3] = r.a.w;
    v[4] = r.b.x, v[5] = r.b.y, v[6] = r.b.z, v[7] = r.b.w;
}
template <>
__device__ __forceinline__ void widen8<__half>(const uint4& r, float (&v)[8]) {
    const uint32_t u[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
        v[2 * i] = f.x, v[2 * i + 1] = f.y;
    }
}
template <>
__device__ __forceinline__ void widen8<__nv_bfloat16>(const uint4& r, float (&v)[8]) {
    const uint32_t u[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(u[i] << 16);
        v[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
    }
}

__device__ __forceinline__ void store8(float* p, const float (&v)[8]) {
    reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}
__device__ __forceinline__ void store8(__half* p, const float (&v)[8]) {
    __half2 h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
    *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(h);
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, const float (&v)[8]) {
    __nv_bfloat162 h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
    *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(h);
}

}  // namespace mbx
