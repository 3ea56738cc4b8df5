// Loads and stores of short runs of elements as fp32, for the kernels that take several element types.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <cstdint>

#include "../../include/mindiesd_b200.h"

namespace sdb {

// kBytes (2, 4, 8 or 16) consecutive bytes at an address that is a multiple of kBytes.
template <int kBytes>
struct Raw;
template <>
struct Raw<16> { using type = uint4; };
template <>
struct Raw<8> { using type = uint2; };
template <>
struct Raw<4> { using type = uint32_t; };
template <>
struct Raw<2> { using type = uint16_t; };
template <>
struct Raw<1> { using type = uint8_t; };

__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(float v) { return v; }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }

// kE elements of T at p as one or more accesses of at most 16 bytes; p is aligned to min(16, kE * sizeof(T)).
template <typename T, int kE>
struct Run {
    static constexpr int kBytes = kE * static_cast<int>(sizeof(T));
    static constexpr int kPiece = kBytes < 16 ? kBytes : 16;
    static constexpr int kPieces = kBytes / kPiece;
    using Piece = typename Raw<kPiece>::type;
    union Data {
        Piece piece[kPieces];
        T elem[kE];
        __device__ __forceinline__ Data() {}
    } d;
    __device__ __forceinline__ void load(const T* p) {
#pragma unroll
        for (int i = 0; i < kPieces; ++i) d.piece[i] = __ldg(reinterpret_cast<const Piece*>(p) + i);
    }
    __device__ __forceinline__ void store(T* p) const {
#pragma unroll
        for (int i = 0; i < kPieces; ++i) reinterpret_cast<Piece*>(p)[i] = d.piece[i];
    }
    __device__ __forceinline__ float get(int i) const { return to_f32(d.elem[i]); }
    __device__ __forceinline__ void set(int i, float v) { d.elem[i] = from_f32<T>(v); }
};

__device__ __forceinline__ uint4 load_shared16(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
    return v;
}

__device__ __forceinline__ void store_shared16(uint32_t addr, const uint4& v) {
    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

// Maximum that keeps a NaN (fmaxf drops it).
__device__ __forceinline__ float max_nan(float a, float b) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}

// Two values as e4m3, the first in the low byte; beyond 448 in magnitude they become +-448, NaN stays NaN.
__device__ __forceinline__ uint16_t e4m3x2(float lo, float hi) {
    uint16_t h;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(h) : "f"(hi), "f"(lo));
    return h;
}

}  // namespace sdb
