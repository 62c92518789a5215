// Quantising a paged key-value cache as it is written, and reading it back
// (chm_cache_write, chm_cache_read).
//
// Per vector: scale = RN32(max |x| / top), code = RN(x / scale) with the
// quotient taken exactly.  The fp32 product x * (1 / scale) is within 2 ulp of
// the quotient, so it gives the same code unless it lies that near to the
// middle between two codes; those few values are decided in 64 bits, where a
// quotient of two fp32 numbers cannot round onto a middle that it is not on.
#include <cuda_fp8.h>

#include <cstdio>

#include "kv_cache.cuh"

namespace chm {

constexpr int kCacheThreads = 256;

struct CacheArgs {
    chm_kv_cache c;
    const void* in[2];   // k, v vectors (write: source, read: destination)
    int64_t vec_t[2], vec_h[2];
    const int64_t* slots;
    int64_t num_slots;
    int64_t vectors;  // tokens * heads
    FastDiv by_heads, by_page;
    bool wide;  // 16-byte accesses of the vectors
};

template <typename T>
__device__ __forceinline__ void load8(const T* p, bool wide, float (&x)[8]) {
    constexpr int kV = 16 / sizeof(T);
    if (wide) {
#pragma unroll
        for (int i = 0; i < 8; i += kV) {
            const Pack<T, kV> w = *reinterpret_cast<const Pack<T, kV>*>(p + i);
#pragma unroll
            for (int j = 0; j < kV; ++j) x[i + j] = to_float<T>(w.v[j]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = to_float<T>(p[i]);
    }
}

template <typename T>
__device__ __forceinline__ void store8(T* p, bool wide, const float (&x)[8]) {
    constexpr int kV = 16 / sizeof(T);
    if (wide) {
#pragma unroll
        for (int i = 0; i < 8; i += kV) {
            Pack<T, kV> w;
#pragma unroll
            for (int j = 0; j < kV; ++j) w.v[j] = from_float<T>(x[i + j]);
            *reinterpret_cast<Pack<T, kV>*>(p + i) = w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) p[i] = from_float<T>(x[i]);
    }
}

// x / s rounded to the nearest integer, ties to even (|x / s| < 128).
__device__ __forceinline__ int int8_code(float x, float s, float inv) {
    const float q = x * inv;
    const float r = rintf(q);
    if (fabsf(q - r) > 0.4999f) return __double2int_rn((double)x / (double)s);
    return (int)r;
}

// x / s rounded to the nearest e4m3 number, ties to even, as its byte.
__device__ __forceinline__ uint32_t e4m3_code(float x, float s, float inv) {
    float q = x * inv;
    // middles: below 2^-6 odd multiples of 2^-10 (decided in 64 bits always),
    // above it the numbers whose last 20 fraction bits are 0x80000
    const uint32_t low = __float_as_uint(q) & 0xFFFFFu;
    if (low - 0x7FFFCu <= 8u || (fabsf(q) < 0.015625f && q != 0.0f)) {
        const double d = (double)x / (double)s;
        q = (float)d;  // to odd: a quotient beside a middle must not land on it
        const uint32_t bits = __float_as_uint(q);
        if ((double)q != d && !(bits & 1)) q = __uint_as_float(fabs((double)q) < fabs(d) ? bits + 1 : bits - 1);
    }
    return __nv_cvt_float_to_fp8(q, __NV_SATFINITE, __NV_E4M3);
}

// A group of LPV lanes holds a vector, 8 elements a lane.
template <typename T, int KIND, int LPV>
__global__ void __launch_bounds__(kCacheThreads) cache_write_kernel(const CacheArgs a) {
    const int lane = threadIdx.x % LPV;
    const int64_t vec = (int64_t)blockIdx.x * (kCacheThreads / LPV) + threadIdx.x / LPV;
    const int side = blockIdx.y;
    const uint32_t t = vec < a.vectors ? a.by_heads.div((uint32_t)vec) : 0u;
    const uint32_t h = (uint32_t)vec - t * a.c.heads;
    const int64_t slot = vec < a.vectors ? a.slots[t] : -1;
    const bool on = slot >= 0 && slot < a.num_slots;
    const bool mine = on && lane * 8 < a.c.dim;
    float x[8] = {};
    if (mine)
        load8<T>(static_cast<const T*>(a.in[side]) + t * a.vec_t[side] + h * a.vec_h[side] + lane * 8, a.wide, x);
    const int64_t page = slot / a.c.page_size;
    const int64_t within = slot - page * a.c.page_size;
    char* base = static_cast<char*>(side ? a.c.v : a.c.k);
    const int64_t at = page * a.c.page_stride + h * a.c.head_stride + within * a.c.token_stride + lane * 8;
    if (KIND == CHM_FP16) {
        if (mine) store8<__half>(reinterpret_cast<__half*>(base) + at, true, x);
    } else if (KIND == CHM_BF16) {
        if (mine) store8<__nv_bfloat16>(reinterpret_cast<__nv_bfloat16*>(base) + at, true, x);
    } else {
        // as integers: an infinity or a NaN is above every finite value
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[i]) & 0x7FFFFFFFu);
#pragma unroll
        for (int m = LPV / 2; m > 0; m >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, m, LPV));
        const float amax = __uint_as_float(top);
        // FLT_MAX / top rounded down is the largest scale: the top code never reads back as an infinity
        float s = fminf(__fdiv_rn(amax, KIND == CHM_INT8 ? 127.0f : 448.0f),
                        KIND == CHM_INT8 ? 0x1.0204060000000p+121f : 0x1.2492480000000p+119f);
        bool zero = false;
        if (top >= 0x7F800000u) s = __uint_as_float(0x7FC00000u), zero = true;
        if (amax < 1.262177448e-29f) s = 0.0f, zero = true;  // 2^-96
        uint32_t w[2] = {0u, 0u};
        if (!zero) {
            const float inv = __frcp_rn(s);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint32_t code = KIND == CHM_INT8 ? (uint32_t)int8_code(x[i], s, inv) & 0xFFu : e4m3_code(x[i], s, inv);
                w[i >> 2] |= code << (8 * (i & 3));
            }
        }
        if (mine) *reinterpret_cast<uint2*>(base + at) = make_uint2(w[0], w[1]);
        if (on && lane == 0) (side ? a.c.v_scale : a.c.k_scale)[(page * a.c.heads + h) * a.c.page_size + within] = s;
    }
}

template <typename T, int KIND, int LPV>
__global__ void __launch_bounds__(kCacheThreads) cache_read_kernel(const CacheArgs a) {
    const int lane = threadIdx.x % LPV;
    const int64_t vec = (int64_t)blockIdx.x * (kCacheThreads / LPV) + threadIdx.x / LPV;
    const int side = blockIdx.y;
    if (vec >= a.vectors || lane * 8 >= a.c.dim) return;
    const uint32_t t = a.by_heads.div((uint32_t)vec);
    const uint32_t h = (uint32_t)vec - t * a.c.heads;
    const int64_t slot = a.slots[t];
    float x[8] = {};
    if (slot >= 0 && slot < a.num_slots) {
        const int64_t page = slot / a.c.page_size;
        const int64_t within = slot - page * a.c.page_size;
        const char* base = static_cast<const char*>(side ? a.c.v : a.c.k);
        const int64_t at = page * a.c.page_stride + h * a.c.head_stride + within * a.c.token_stride + lane * 8;
        if (KIND == CHM_FP16) {
            load8<__half>(reinterpret_cast<const __half*>(base) + at, true, x);
        } else if (KIND == CHM_BF16) {
            load8<__nv_bfloat16>(reinterpret_cast<const __nv_bfloat16*>(base) + at, true, x);
        } else {
            const float s = (side ? a.c.v_scale : a.c.k_scale)[(page * a.c.heads + h) * a.c.page_size + within];
            const uint2 w = *reinterpret_cast<const uint2*>(base + at);
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                const uint32_t two = ((i < 4 ? w.x : w.y) >> (8 * (i & 3))) & 0xFFFFu;
                float2 y;
                if (KIND == CHM_INT8)
                    y = make_float2((float)(int8_t)(two & 0xFFu), (float)(int8_t)(two >> 8));
                else
                    y = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)two, __NV_E4M3)));
                x[i] = y.x * s, x[i + 1] = y.y * s;
            }
        }
    }
    T* out = static_cast<T*>(const_cast<void*>(a.in[side])) + t * a.vec_t[side] + h * a.vec_h[side] + lane * 8;
    store8<T>(out, a.wide, x);
}

template <typename T, int KIND, bool WRITE>
static void launch_cache(const CacheArgs& a, cudaStream_t st) {
    const int lpv = a.c.dim <= 64 ? 8 : a.c.dim <= 128 ? 16 : 32;
    const int per = kCacheThreads / lpv;
    const dim3 grid((unsigned)((a.vectors + per - 1) / per), 2);
#define CHM_CACHE_GO(L)                                                      \
    if (WRITE)                                                               \
        cache_write_kernel<T, KIND, L><<<grid, kCacheThreads, 0, st>>>(a);   \
    else                                                                     \
        cache_read_kernel<T, KIND, L><<<grid, kCacheThreads, 0, st>>>(a)
    if (lpv == 8) {
        CHM_CACHE_GO(8);
    } else if (lpv == 16) {
        CHM_CACHE_GO(16);
    } else {
        CHM_CACHE_GO(32);
    }
#undef CHM_CACHE_GO
}

template <typename T, bool WRITE>
static void dispatch_kind(const CacheArgs& a, cudaStream_t st) {
    switch (a.c.type) {
        case CHM_FP16: return launch_cache<T, CHM_FP16, WRITE>(a, st);
        case CHM_BF16: return launch_cache<T, CHM_BF16, WRITE>(a, st);
        case CHM_INT8: return launch_cache<T, CHM_INT8, WRITE>(a, st);
        default: return launch_cache<T, CHM_E4M3, WRITE>(a, st);
    }
}

template <bool WRITE>
static chm_status run_cache(const chm_kv_cache* cache, const chm_heads* k, const chm_heads* v, int32_t type,
                            int64_t tokens, const int64_t* slots, cudaStream_t st) {
    const char* who = WRITE ? "cache_write" : "cache_read";
    CHM_TRY(check_cache(cache, who));
    auto bad = [&](const char* why) {
        char msg[160];
        snprintf(msg, sizeof(msg), "%s: %s", who, why);
        set_last_message(msg);
        return CHM_ERR_INVALID;
    };
    if (!k || !v || !valid_float_type(type)) return bad("fp32, fp16 or bf16 keys and values");
    if (tokens < 0) return bad("negative size");
    if (k->heads != cache->heads || v->heads != cache->heads) return bad("heads differ from the cache's");
    if (tokens == 0) return CHM_OK;
    if (!k->data || !v->data || !slots) return bad("null keys, values or slots");
    if (tokens > INT32_MAX / cache->heads) return bad("more than 2^31 - 1 vectors");
    CacheArgs a{};
    a.c = *cache;
    const chm_heads* kv[2] = {k, v};
    const int run = 16 / type_bytes(type);
    a.wide = true;
    for (int i = 0; i < 2; ++i) {
        a.in[i] = kv[i]->data;
        a.vec_t[i] = kv[i]->token_stride;
        a.vec_h[i] = kv[i]->head_stride;
        a.wide = a.wide && aligned16(kv[i]->data) && a.vec_t[i] % run == 0 && a.vec_h[i] % run == 0;
    }
    a.slots = slots;
    a.num_slots = cache->num_pages * cache->page_size;
    a.vectors = tokens * cache->heads;
    a.by_heads = FastDiv((uint32_t)cache->heads);
    a.by_page = FastDiv((uint32_t)cache->page_size);
    if (type == CHM_FP32)
        dispatch_kind<float, WRITE>(a, st);
    else if (type == CHM_FP16)
        dispatch_kind<__half, WRITE>(a, st);
    else
        dispatch_kind<__nv_bfloat16, WRITE>(a, st);
    return launch_status(WRITE ? "cache_write_kernel" : "cache_read_kernel");
}

}  // namespace chm

extern "C" chm_status chm_cache_write(const chm_kv_cache* cache, const chm_heads* k, const chm_heads* v, int32_t type,
                                      int64_t tokens, const int64_t* slots, void* stream) {
    return chm::run_cache<true>(cache, k, v, type, tokens, slots, (cudaStream_t)stream);
}

extern "C" chm_status chm_cache_read(const chm_kv_cache* cache, const int64_t* slots, int64_t tokens,
                                     const chm_heads* k, const chm_heads* v, int32_t type, void* stream) {
    return chm::run_cache<false>(cache, k, v, type, tokens, slots, (cudaStream_t)stream);
}
