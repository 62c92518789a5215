// Element types, 16-byte vector accesses and division by run-time constants
// for the generation operators (rotary.cu, kv_cache.cu, paged_attention.cu).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace chm {

// n / d for 0 <= n < 2^31 and a divisor fixed for the launch:
// floor(n * m / 2^(32 + s)) with m = ceil(2^(32 + s) / d), s = ceil(log2 d) - 1.
// The error of m, below 1 / 2^(32 + s) * d <= 2^-31 of a unit of the quotient
// per n, cannot reach the next multiple for n < 2^31.
struct FastDiv {
    uint32_t d, m, s;
    FastDiv() = default;
    explicit FastDiv(uint32_t div) : d(div), m(0), s(0) {
        if (div > 1) {
            uint32_t l = 0;
            while ((1ull << l) < div) ++l;
            s = l - 1;
            m = (uint32_t)(((1ull << (32 + s)) + div - 1) / div);
        }
    }
    __device__ __forceinline__ uint32_t div(uint32_t n) const { return d == 1 ? n : __umulhi(n, m) >> s; }
};

template <typename T>
__device__ __forceinline__ float to_float(T x);
template <>
__device__ __forceinline__ float to_float<float>(float x) {
    return x;
}
template <>
__device__ __forceinline__ float to_float<__half>(__half x) {
    return __half2float(x);
}
template <>
__device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 x) {
    return __bfloat162float(x);
}

// Round to nearest even (fp16: values past its range become infinite).
template <typename T>
__device__ __forceinline__ T from_float(float x);
template <>
__device__ __forceinline__ float from_float<float>(float x) {
    return x;
}
template <>
__device__ __forceinline__ __half from_float<__half>(float x) {
    return __float2half_rn(x);
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) {
    return __float2bfloat16_rn(x);
}

// V consecutive elements in one access (V * sizeof(T) a power of two, at most
// 16 bytes, and the address a multiple of it).
template <typename T, int V>
struct alignas(sizeof(T) * V) Pack {
    T v[V];
};

__host__ __device__ inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

inline bool valid_float_type(int32_t t) { return t == CHM_FP32 || t == CHM_FP16 || t == CHM_BF16; }
inline int type_bytes(int32_t t) { return t == CHM_FP32 ? 4 : t == CHM_FP16 || t == CHM_BF16 ? 2 : 1; }

}  // namespace chm
