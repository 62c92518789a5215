// Quantising a paged key-value cache as it is written, and reading it back
// (chm_cache_write, chm_cache_read).
//
// Per vector: scale = RN32(max |x| / top), code = RN(x / scale) with the
// quotient taken exactly: x times the reciprocal of the scale (off by less than
// 3.7e-7 of itself) may lie on the other side of a middle between two codes.
// - fp32 vectors: the product with the reciprocal made 2^-21 smaller and larger
//   encloses the quotient; where both round to the same code that is it, else
//   (about one value in 2^16) the remainder decides.
// - 16-bit vectors: top * x / max |x| is on a middle, or 2^-19 of it away (the
//   middle has at most 8 bits, the maximum 11).  Values away from it do not mind a
//   factor 1 +- 2^-21.  Those on it lie where the rounding of the scale puts them:
//   above where it was rounded down, below where up, which that factor does for all
//   of the vector at once.  Where the scale is exact, so is the quotient on a
//   middle, and the product corrected by its remainder gives it.
//   One bf16 value in a hundred or so is on a middle; the way of fp32 vectors took
//   most warps through the remainder (32,768 tokens of 8 heads of 128 to e4m3: 63 us
//   against 48).
//
// Both directions move their bytes once; the bound is HBM, and next to it, for
// codes, the instructions per value (134 per warp and vector of 128 to write, 90 to
// read; the integer pipe, at half rate, is busy for two thirds of the writing).  One
// B200, us on the device: 32,768 tokens of 8 heads of 128 bf16 values written to e4m3 in
// 43 to 47 (203 MB, 4.3 to 4.7 TB/s) and read back in 35 (5.8 TB/s), the two calls in 83;
// 8,192 to a bf16 cache in 13 and back in 10 (67 MB each), the two calls in 25.
#include <cuda_fp8.h>

#include <type_traits>

#include "kv_cache.cuh"

namespace chm {

constexpr int kCacheThreads = 128;
// Vectors per thread and side: one, until there are so many vectors that more loads on their
// way count for more than more warps.  Device time of one against several:
//   writing (2): 32 tokens of 8 heads of 128 bf16 values 1.9 / 2.3 us, 8,192 to e4m3 11.8 / 12.0,
//     32,768 to e4m3 49 / 47;
//   reading (4): 1.8 / 2.6, 2,048 from e4m3 3.7 / 4.1, 8,192 8.6 / 8.5, 32,768 40 / 35.
// (32,768 written and read back: 80 us; 1 and 4: 82, 2 and 3: 82, 2 and 2: 84, 256 threads: 2 to
// 7 more.)
constexpr int kWriteUnroll = 2, kReadUnroll = 4;
constexpr int64_t kWriteMany = 131072, kReadMany = 65536;

struct CacheArgs {
    chm_kv_cache c;
    const void* vec[2];  // k, v vectors (write: source, read: destination)
    int64_t vec_t[2], vec_h[2];
    const int64_t* slots;
    int64_t num_slots;
    int64_t vectors;  // tokens * heads
    FastDiv by_heads, by_page;
    // 8,192 tokens of 8 heads of 128 bf16 values to int8 11.6 us, and back 8.2:
    bool wide;   // 16-byte accesses of the vectors where they start there (else 14.3 and 47)
    bool small;  // slots below 2^31: 32-bit division (else 12.3 and 9.5)
};

// Eight elements as they are in memory.
template <typename T>
struct Eight {
    uint32_t w[2 * sizeof(T)];

    __device__ __forceinline__ void load(const T* p, bool wide) {
        if (wide) {
#pragma unroll
            for (int i = 0; i < (int)sizeof(T) / 2; ++i) {
                const uint4 x = reinterpret_cast<const uint4*>(p)[i];
                w[4 * i] = x.x, w[4 * i + 1] = x.y, w[4 * i + 2] = x.z, w[4 * i + 3] = x.w;
            }
        } else if (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i % (2 * sizeof(T))] = reinterpret_cast<const uint32_t*>(p)[i];
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                w[i] = reinterpret_cast<const uint16_t*>(p)[2 * i] |
                       (uint32_t) reinterpret_cast<const uint16_t*>(p)[2 * i + 1] << 16;
        }
    }
    __device__ __forceinline__ void store(T* p, bool wide) const {
        if (wide) {
#pragma unroll
            for (int i = 0; i < (int)sizeof(T) / 2; ++i)
                reinterpret_cast<uint4*>(p)[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
        } else if (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < 8; ++i) reinterpret_cast<uint32_t*>(p)[i] = w[i % (2 * sizeof(T))];
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) reinterpret_cast<uint16_t*>(p)[i] = (uint16_t)(w[i / 2] >> (16 * (i & 1)));
        }
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (auto& x : w) x = 0;
    }
    __device__ __forceinline__ float2 pair(int i) const;
    __device__ __forceinline__ void set(int i, float a, float b);
    // The largest magnitude's bits, as an integer (an infinity or a NaN is above
    // every finite number): two at once for 16-bit types.
    __device__ __forceinline__ uint32_t top() const {
        uint32_t m = 0;
#pragma unroll
        for (auto x : w) m = sizeof(T) == 4 ? max(m, x & 0x7FFFFFFFu) : __vmaxu2(m, x & 0x7FFF7FFFu);
        return m;
    }
    static __device__ __forceinline__ float magnitude(uint32_t bits);  // of one value
};
template <>
__device__ __forceinline__ float2 Eight<float>::pair(int i) const {
    return make_float2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
}
template <>
__device__ __forceinline__ float2 Eight<__half>::pair(int i) const {
    return __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
}
template <>
__device__ __forceinline__ float2 Eight<__nv_bfloat16>::pair(int i) const {
    return make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xFFFF0000u));
}
template <>
__device__ __forceinline__ void Eight<float>::set(int i, float a, float b) {
    w[2 * i] = __float_as_uint(a), w[2 * i + 1] = __float_as_uint(b);
}
template <>
__device__ __forceinline__ void Eight<__half>::set(int i, float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    w[i] = *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ void Eight<__nv_bfloat16>::set(int i, float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    w[i] = *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ float Eight<float>::magnitude(uint32_t m) {
    return __uint_as_float(m);
}
template <>
__device__ __forceinline__ float Eight<__half>::magnitude(uint32_t m) {
    return __half2float(__ushort_as_half((unsigned short)m));
}
template <>
__device__ __forceinline__ float Eight<__nv_bfloat16>::magnitude(uint32_t m) {
    return __uint_as_float(m << 16);
}

// Four values as codes, the quotient by f's inverse rounded once.
template <int KIND>
__device__ __forceinline__ uint32_t four_codes(const float* x, float f) {
    if (KIND == CHM_INT8) {
        // 1.5 * 2^23 leaves the integer, to nearest and ties to even, in the low bits
        uint32_t b[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) b[i] = __float_as_uint(__fmaf_rn(x[i], f, 12582912.0f));
        return __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
    }
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(x[0] * f, x[1] * f), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(x[2] * f, x[3] * f), __NV_SATFINITE, __NV_E4M3);
    return __byte_perm(lo, hi, 0x5410);
}

// The code of x where the two that enclose the quotient differ: they are neighbours,
// and the remainder x - middle * scale (exact: one rounding of fma, the middle has few
// bits) tells the side; on the middle the even code.
template <int KIND>
__device__ __forceinline__ uint32_t nearer_code(float x, float s, uint32_t lo, uint32_t hi) {
    float a, b;
    if (KIND == CHM_INT8) {
        a = fabsf((float)(int8_t)lo), b = fabsf((float)(int8_t)hi);
    } else {
        const float2 y = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(lo | hi << 8), __NV_E4M3)));
        a = fabsf(y.x), b = fabsf(y.y);
    }
    const float r = __fmaf_rn(-0.5f * (a + b), s, fabsf(x));
    return r > 0.0f || (r == 0.0f && (lo & 1)) ? hi : lo;
}

__device__ __forceinline__ float reciprocal(float x) {  // within 1 ulp
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// Where a slot's vector is: its element offset (this lane's eight), and its scale.
struct Place {
    int64_t at, scale;
};
__device__ __forceinline__ Place place_of(const CacheArgs& a, int64_t slot, uint32_t h, int lane) {
    const int64_t page = a.small ? (int64_t)a.by_page.div((uint32_t)slot) : slot / a.c.page_size;
    const int64_t within = slot - page * a.c.page_size;
    return Place{page * a.c.page_stride + h * a.c.head_stride + within * a.c.token_stride + lane * 8,
                 (page * a.c.heads + h) * a.c.page_size + within};
}

// A group of LPV lanes holds a vector, 8 elements a lane.
template <typename T, int KIND, int LPV, int U>
__global__ void __launch_bounds__(kCacheThreads) cache_write_kernel(const CacheArgs a) {
    constexpr int kPer = kCacheThreads / LPV;
    const int lane = threadIdx.x % LPV;
    const int64_t first = (int64_t)blockIdx.x * (kPer * U) + threadIdx.x / LPV;
    Eight<T> x[U][2];
    Place place[U];
    bool on[U];
#pragma unroll
    for (int j = 0; j < U; ++j) {
        const int64_t vec = first + j * kPer;
        on[j] = vec < a.vectors;
        const uint32_t t = on[j] ? a.by_heads.div((uint32_t)vec) : 0u;
        const uint32_t h = (uint32_t)vec - t * a.c.heads;
        const int64_t slot = on[j] ? a.slots[t] : -1;
        on[j] = slot >= 0 && slot < a.num_slots;
        if (on[j]) place[j] = place_of(a, slot, h, lane);
#pragma unroll
        for (int side = 0; side < 2; ++side) {
            if (on[j] && lane * 8 < a.c.dim)
                x[j][side].load(static_cast<const T*>(a.vec[side]) + t * a.vec_t[side] + h * a.vec_h[side] + lane * 8,
                                a.wide);
            else
                x[j][side].clear();
        }
    }
#pragma unroll
    for (int j = 0; j < U; ++j) {
        float largest[2];
        if (KIND == CHM_INT8 || KIND == CHM_E4M3) {
            uint32_t top[2] = {x[j][0].top(), x[j][1].top()};
            if (sizeof(T) == 2) {  // both vectors' in one word
                top[0] = __vmaxu2(__byte_perm(top[0], top[1], 0x5410), __byte_perm(top[0], top[1], 0x7632));
#pragma unroll
                for (int m = LPV / 2; m > 0; m >>= 1) top[0] = __vmaxu2(top[0], __shfl_xor_sync(0xffffffffu, top[0], m, LPV));
                top[1] = top[0] >> 16;
                top[0] &= 0xFFFFu;
            } else {
#pragma unroll
                for (int side = 0; side < 2; ++side)
#pragma unroll
                    for (int m = LPV / 2; m > 0; m >>= 1)
                        top[side] = max(top[side], __shfl_xor_sync(0xffffffffu, top[side], m, LPV));
            }
            largest[0] = Eight<T>::magnitude(top[0]), largest[1] = Eight<T>::magnitude(top[1]);
        }
#pragma unroll
        for (int side = 0; side < 2; ++side) {
            char* base = static_cast<char*>(side ? a.c.v : a.c.k);
            const bool mine = on[j] && lane * 8 < a.c.dim;
            if (KIND == CHM_FP16 || KIND == CHM_BF16) {
                using H = typename std::conditional<KIND == CHM_FP16, __half, __nv_bfloat16>::type;
                Eight<H> y;
                if (std::is_same<T, H>::value) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) y.w[i] = x[j][side].w[i];
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float2 p = x[j][side].pair(i);
                        y.set(i, p.x, p.y);
                    }
                }
                if (mine) y.store(reinterpret_cast<H*>(base) + place[j].at, true);
                continue;
            }
            const float amax = largest[side];
            // amax / top to nearest: a product with its inverse and one step by the remainder
            // (Markstein's division) give it for every fp32 amax of this range (checked for all
            // fractions)
            constexpr float kTop = KIND == CHM_INT8 ? 127.0f : 448.0f, kInv = 1.0f / kTop;
            const float near = amax * kInv;
            float s = fminf(__fmaf_rn(__fmaf_rn(-near, kTop, amax), kInv, near),
                            KIND == CHM_INT8 ? 0x1.0204060000000p+121f : 0x1.2492480000000p+119f);
            const bool odd = !(amax <= 3.402823466e38f), none = amax < 1.262177448e-29f;  // 2^-96
            if (odd) s = __uint_as_float(0x7FC00000u);
            if (none) s = 0.0f;
            uint32_t w[2] = {0u, 0u};
            if (!odd && !none) {
                const float inv = reciprocal(s);
                float f[8];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 p = x[j][side].pair(i);
                    f[2 * i] = p.x, f[2 * i + 1] = p.y;
                }
                const float below = inv * 0.99999952316284f, past = inv * 1.00000047683716f;  // 1 -+ 2^-21
                if (sizeof(T) == 2) {
                    const float off = __fmaf_rn(-s, kTop, amax);  // above 0: the scale was rounded down
                    if (off == 0.0f) {
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const float q = f[i] * inv;
                            f[i] = __fmaf_rn(__fmaf_rn(-q, s, f[i]), inv, q);
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < 8; ++i) f[i] *= off > 0.0f ? past : below;
                    }
                    w[0] = four_codes<KIND>(f, 1.0f);
                    w[1] = four_codes<KIND>(f + 4, 1.0f);
                } else {
                    uint32_t v[2];
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        w[i] = four_codes<KIND>(f + 4 * i, below);
                        v[i] = four_codes<KIND>(f + 4 * i, past);
                    }
                    unsigned long long differ = (unsigned long long)(w[1] ^ v[1]) << 32 | (w[0] ^ v[0]);
                    while (differ) {
                        const int e = (__ffsll((long long)differ) - 1) >> 3;
                        differ &= ~(0xFFull << (8 * e));
                        const int at = 8 * (e & 3);
                        const uint32_t lo = (e < 4 ? w[0] : w[1]) >> at & 0xFFu, hi = (e < 4 ? v[0] : v[1]) >> at & 0xFFu;
                        float y = f[0];
#pragma unroll
                        for (int k = 1; k < 8; ++k) y = e == k ? f[k] : y;
                        const uint32_t flip = (nearer_code<KIND>(y, s, lo, hi) ^ lo) << at;
                        if (e < 4)
                            w[0] ^= flip;
                        else
                            w[1] ^= flip;
                    }
                }
            }
            if (mine) *reinterpret_cast<uint2*>(base + place[j].at) = make_uint2(w[0], w[1]);
            if (on[j] && lane == 0) (side ? a.c.v_scale : a.c.k_scale)[place[j].scale] = s;
        }
    }
}

template <typename T, int KIND, int LPV, int U>
__global__ void __launch_bounds__(kCacheThreads) cache_read_kernel(const CacheArgs a) {
    constexpr int kPer = kCacheThreads / LPV;
    constexpr bool kCodes = KIND == CHM_INT8 || KIND == CHM_E4M3;
    using H = typename std::conditional<KIND == CHM_FP16, __half, __nv_bfloat16>::type;
    const int lane = threadIdx.x % LPV;
    const int64_t first = (int64_t)blockIdx.x * (kPer * U) + threadIdx.x / LPV;
    if (lane * 8 >= a.c.dim) return;
    Eight<H> held[U][2];
    uint2 codes[U][2];
    float scale[U][2];
    uint32_t t[U], h[U];
#pragma unroll
    for (int j = 0; j < U; ++j) {
        const int64_t vec = first + j * kPer;
        t[j] = vec < a.vectors ? a.by_heads.div((uint32_t)vec) : 0u;
        h[j] = (uint32_t)vec - t[j] * a.c.heads;
        const int64_t slot = vec < a.vectors ? a.slots[t[j]] : -1;
        const bool on = slot >= 0 && slot < a.num_slots;
        Place p{};
        if (on) p = place_of(a, slot, h[j], lane);
#pragma unroll
        for (int side = 0; side < 2; ++side) {
            const char* base = static_cast<const char*>(side ? a.c.v : a.c.k);
            held[j][side].clear();
            codes[j][side] = make_uint2(0, 0);
            scale[j][side] = 0.0f;
            if (on && kCodes) {
                codes[j][side] = *reinterpret_cast<const uint2*>(base + p.at);
                scale[j][side] = (side ? a.c.v_scale : a.c.k_scale)[p.scale];
            } else if (on) {
                held[j][side].load(reinterpret_cast<const H*>(base) + p.at, true);
            }
        }
    }
#pragma unroll
    for (int j = 0; j < U; ++j) {
        if (first + j * kPer >= a.vectors) continue;
#pragma unroll
        for (int side = 0; side < 2; ++side) {
            Eight<T> y;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float2 f;
                if (kCodes) {
                    const uint32_t two = (i < 2 ? codes[j][side].x : codes[j][side].y) >> (16 * (i & 1)) & 0xFFFFu;
                    if (KIND == CHM_INT8)
                        f = make_float2((float)(int8_t)(two & 0xFFu), (float)(int8_t)(two >> 8));
                    else
                        f = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)two, __NV_E4M3)));
                    f.x *= scale[j][side], f.y *= scale[j][side];
                } else {
                    f = held[j][side].pair(i);
                }
                if (std::is_same<T, H>::value && !kCodes)
                    y.w[i] = held[j][side].w[i];
                else
                    y.set(i, f.x, f.y);
            }
            y.store(static_cast<T*>(const_cast<void*>(a.vec[side])) + t[j] * a.vec_t[side] + h[j] * a.vec_h[side] +
                        lane * 8,
                    a.wide);
        }
    }
}

template <typename T, int KIND, int LPV, bool WRITE>
static void launch_lanes(const CacheArgs& a, cudaStream_t st) {
    constexpr int kMany = WRITE ? kWriteUnroll : kReadUnroll;
    const bool many = a.vectors >= (WRITE ? kWriteMany : kReadMany);
    const int per = kCacheThreads / LPV * (many ? kMany : 1);
    const unsigned grid = (unsigned)((a.vectors + per - 1) / per);
    if constexpr (WRITE) {
        if (many)
            cache_write_kernel<T, KIND, LPV, kMany><<<grid, kCacheThreads, 0, st>>>(a);
        else
            cache_write_kernel<T, KIND, LPV, 1><<<grid, kCacheThreads, 0, st>>>(a);
    } else {
        if (many)
            cache_read_kernel<T, KIND, LPV, kMany><<<grid, kCacheThreads, 0, st>>>(a);
        else
            cache_read_kernel<T, KIND, LPV, 1><<<grid, kCacheThreads, 0, st>>>(a);
    }
}

template <typename T, int KIND, bool WRITE>
static void launch_cache(const CacheArgs& a, cudaStream_t st) {
    if (a.c.dim <= 64)
        launch_lanes<T, KIND, 8, WRITE>(a, st);
    else if (a.c.dim <= 128)
        launch_lanes<T, KIND, 16, WRITE>(a, st);
    else
        launch_lanes<T, KIND, 32, WRITE>(a, st);
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
        a.vec[i] = kv[i]->data;
        a.vec_t[i] = kv[i]->token_stride;
        a.vec_h[i] = kv[i]->head_stride;
        a.wide = a.wide && aligned16(kv[i]->data) && a.vec_t[i] % run == 0 && a.vec_h[i] % run == 0;
    }
    a.slots = slots;
    a.num_slots = cache->num_pages * cache->page_size;
    a.vectors = tokens * cache->heads;
    a.small = a.num_slots <= INT32_MAX;
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
