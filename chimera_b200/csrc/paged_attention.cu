// Attention of one new token per sequence over a paged key-value cache
// (chm_paged_attention).
//
// out = sum_j p_j v_j / sum_j p_j with p_j = exp(scale <q, k_j> - m), one pass
// over the tokens with a running maximum m.  Every key and value is read once,
// for all the query heads that share it, so the bound is HBM.
//
// The products run on mma.sync m16n8k16 with the tokens (for the scores) and
// the elements of the value vector (for the output) as the 16 rows and the
// query heads of one key head as the 8 columns:
//   S^T [tokens x heads] = K [tokens x dim] Q^T,   O^T [dim x heads] += V^T P^T.
// Both contractions may take their index in any order, so a thread's 16-byte
// loads are its operand registers as they come: no shared memory, no barrier.
#include <cmath>
#include <cstdio>

#include "kv_cache.cuh"

namespace chm {

constexpr int kAttWarps = 4;
constexpr int kAttThreads = kAttWarps * 32;
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.69314718055994530942f;

struct AttArgs {
    chm_kv_cache c;
    const void* q;
    void* out;
    int64_t q_b, q_h, out_b, out_h;
    int32_t q_type;
    int32_t batch, q_heads, group;  // group: query heads per key head
    int32_t blocks;                 // blocks of 8 * NT query heads per key head
    const int32_t* tables;
    int64_t table_stride;
    int32_t capacity;  // table_width * page_size
    const int32_t* lens;
    const int32_t* starts;
    float scale_log2;
    float* lse;
    FastDiv by_page;
};

__device__ __forceinline__ uint4 ldg16(const void* p) {
    uint4 r;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
                 : "l"(p));
    return r;
}

__device__ __forceinline__ uint2 ldg8(const void* p) {
    uint2 r;
    asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0,%1}, [%2];" : "=r"(r.x), "=r"(r.y) : "l"(p));
    return r;
}

template <bool HALF>
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                    uint32_t b1) {
    if (HALF)
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// 8x8 transpose of 16-bit elements across the warp.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
}

__device__ __forceinline__ float exp2_fast(float x) {
    float r;
    asm("ex2.approx.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

template <bool HALF>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
    if (HALF) {
        const __half2 h = __floats2half2_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}

template <bool HALF>
__device__ __forceinline__ float2 unpack16(uint32_t x) {
    if (HALF) return __half22float2(*reinterpret_cast<const __half2*>(&x));
    return make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xFFFF0000u));
}

// Two 8-bit codes as bf16 pairs, exactly.  int8: `y` holds the codes in the
// low bytes of its halves; 128 + (code & 127) less 128, or 256 for a negative
// code.  e4m3: the codes in the high bytes; a bf16 with an exponent 120 too
// low, times 2^120 (subnormal codes come out of the product exactly too).
template <int KIND>
__device__ __forceinline__ uint32_t codes_to_bf16(uint32_t y) {
    __nv_bfloat162 r;
    if (KIND == CHM_INT8) {
        const uint32_t a = (y & 0x007F007Fu) | 0x43004300u;
        const uint32_t b = (y & 0x00800080u) | 0x43004300u;
        r = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
    } else {
        const uint32_t a = (y & 0x80008000u) | ((y >> 4) & 0x07F007F0u);
        const uint32_t b = 0x7B807B80u;
        r = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
    }
    return *reinterpret_cast<const uint32_t*>(&r);
}

// What one lane knows of one token of a step: where it is, and its scales.
struct TokenInfo {
    int64_t at;  // element offset of its vector, -1: none
    float ks, vs;
};

// One sequence's attended range and the walk over its table.
struct Sequence {
    int first, end;  // positions
    const int32_t* table;
};

template <int KIND>
__device__ __forceinline__ TokenInfo token_info(const AttArgs& a, const Sequence& s, int pos, int head, bool& bad) {
    TokenInfo r{-1, 0.0f, 0.0f};
    if (pos < s.end) {
        const uint32_t pi = a.by_page.div((uint32_t)pos);
        const uint32_t within = (uint32_t)pos - pi * (uint32_t)a.c.page_size;
        const int64_t page = s.table[pi];
        if (page < 0 || page >= a.c.num_pages) {
            bad = true;
        } else {
            r.at = page * a.c.page_stride + (int64_t)head * a.c.head_stride + (int64_t)within * a.c.token_stride;
            if (KIND == CHM_INT8 || KIND == CHM_E4M3) {
                const int64_t i = (page * a.c.heads + head) * a.c.page_size + within;
                r.ks = a.c.k_scale[i];
                r.vs = a.c.v_scale[i];
            }
        }
    }
    return r;
}

// DMAX: dim rounded up to 64, 128 or 256; NT: blocks of 8 query heads.
template <int DMAX, int KIND, int NT>
__global__ void __launch_bounds__(kAttThreads) paged_attention_kernel(const AttArgs a) {
    constexpr bool kWide = KIND == CHM_FP16 || KIND == CHM_BF16;  // 16-bit cache
    constexpr bool kHalf = KIND == CHM_FP16;                      // type of the products
    constexpr int kBytes = kWide ? 2 : 1;
    constexpr int kU = kWide ? 1 : 2;        // groups of 16 tokens per warp and step
    constexpr int kTok = 16 * kU;
    constexpr int kKC = DMAX * kBytes / 64;  // 16-byte runs of a key per thread
    constexpr int kSteps = DMAX / 16;        // products along dim
    constexpr int kE = DMAX / 8;             // value elements per thread and token
    constexpr int kVC = kE * kBytes / 8;     // 8-byte runs of a value per thread
    constexpr int kM = kE / 2;               // 16-row blocks of the output
    constexpr int kHeads = 8 * NT;
    constexpr int kRow = DMAX + 4;
    __shared__ uint4 s_q[2][NT][kSteps / 2][32];  // high and low part of q as operand registers
    __shared__ float s_o[kAttWarps][kHeads][kRow];
    __shared__ float s_m[kAttWarps][kHeads], s_l[kAttWarps][kHeads];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int seg = blockIdx.x, b = blockIdx.y;
    const int head = seg / a.blocks;
    const int h0 = head * a.group + (seg - head * a.blocks) * kHeads;  // first query head
    const int nh = min(kHeads, (head + 1) * a.group - h0);
    const int dim = a.c.dim;

    Sequence s;
    s.table = a.tables + b * a.table_stride;
    s.first = a.starts ? min(max(a.starts[b], 0), a.capacity) : 0;
    s.end = a.lens[b];
    bool bad = s.end > a.capacity;
    if (bad) s.end = 0;

    // q: lane (g, t) of run i holds the 8 elements that its key runs meet
    const bool split_q = !kWide && a.q_type == CHM_FP16;
    for (int i = threadIdx.x; i < NT * (kSteps / 2) * 32; i += kAttThreads) {
        const int ln = i & 31, run = (i >> 5) % (kSteps / 2), nt = (i >> 5) / (kSteps / 2);
        const int hh = nt * 8 + (ln >> 2);
        const int d0 = kWide ? run * 32 + (ln & 3) * 8 : (run >> 1) * 64 + (ln & 3) * 16 + (run & 1) * 8;
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float x[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int d = d0 + 2 * j + e;
                x[e] = 0.0f;
                if (hh < nh && d < dim) {
                    const int64_t at = b * a.q_b + (h0 + hh) * a.q_h + d;
                    x[e] = a.q_type == CHM_FP16 ? __half2float(static_cast<const __half*>(a.q)[at])
                                                : __bfloat162float(static_cast<const __nv_bfloat16*>(a.q)[at]);
                }
            }
            hi[j] = pack16<kHalf>(x[0], x[1]);
            const float2 r = unpack16<kHalf>(hi[j]);
            lo[j] = pack16<kHalf>(x[0] - r.x, x[1] - r.y);
        }
        s_q[0][nt][run][ln] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        s_q[1][nt][run][ln] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
    }
    __syncthreads();

    float o[NT][kM][4] = {};
    float m[NT][2], l[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) m[n][0] = m[n][1] = -INFINITY, l[n][0] = l[n][1] = 0.0f;

    for (int base = s.first + warp * kTok; base < s.end; base += kAttWarps * kTok) {
        const TokenInfo info = token_info<KIND>(a, s, base + lane % kTok, head, bad);
        // ---- scores
        float sc[NT][kU][4] = {};
#pragma unroll
        for (int u = 0; u < kU; ++u) {
            uint4 kr[2][kKC];
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const int64_t at = __shfl_sync(0xffffffffu, info.at, u * 16 + r * 8 + g);
                const char* p = static_cast<const char*>(a.c.k) + at * kBytes + t * 16;
#pragma unroll
                for (int c = 0; c < kKC; ++c) {
                    kr[r][c] = make_uint4(0, 0, 0, 0);
                    if (at >= 0 && (c * 64 + t * 16) < dim * kBytes) kr[r][c] = ldg16(p + c * 64);
                }
            }
#pragma unroll
            for (int c = 0; c < kKC; ++c) {
                const uint32_t w0[4] = {kr[0][c].x, kr[0][c].y, kr[0][c].z, kr[0][c].w};
                const uint32_t w1[4] = {kr[1][c].x, kr[1][c].y, kr[1][c].z, kr[1][c].w};
                // pairs of the run: 4 words of a 16-bit cache, 8 pairs of codes
#pragma unroll
                for (int j = 0; j < (kWide ? 1 : 2); ++j) {
                    uint32_t p0[4], p1[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        if (kWide) {
                            p0[i] = w0[i], p1[i] = w1[i];
                        } else {
                            const uint32_t x0 = w0[j * 2 + (i >> 1)], x1 = w1[j * 2 + (i >> 1)];
                            const uint32_t sel = KIND == CHM_INT8 ? ((i & 1) ? 0x4342 : 0x4140) : ((i & 1) ? 0x3424 : 0x1404);
                            p0[i] = codes_to_bf16<KIND>(__byte_perm(x0, 0, sel));
                            p1[i] = codes_to_bf16<KIND>(__byte_perm(x1, 0, sel));
                        }
                    }
                    const int run = kWide ? c : c * 2 + j;
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        uint4 bq = s_q[0][n][run][lane];
                        mma<kHalf>(sc[n][u], p0[0], p1[0], p0[1], p1[1], bq.x, bq.y);
                        mma<kHalf>(sc[n][u], p0[2], p1[2], p0[3], p1[3], bq.z, bq.w);
                        if (!kWide && split_q) {
                            bq = s_q[1][n][run][lane];
                            mma<kHalf>(sc[n][u], p0[0], p1[0], p0[1], p1[1], bq.x, bq.y);
                            mma<kHalf>(sc[n][u], p0[2], p1[2], p0[3], p1[3], bq.z, bq.w);
                        }
                    }
                }
            }
        }
        // ---- running maximum; it follows the scores only when one passes it by more than 2^8
        float vs[kU][2];
        bool above = false;
#pragma unroll
        for (int u = 0; u < kU; ++u)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const int src = u * 16 + r * 8 + g;
                const bool on = base + src < s.end;
                float f = a.scale_log2;
                if (!kWide) {
                    f *= __shfl_sync(0xffffffffu, info.ks, src);
                    vs[u][r] = __shfl_sync(0xffffffffu, info.vs, src);
                }
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float& x = sc[n][u][r * 2 + e];
                        x = on ? x * f : -INFINITY;
                        above = above || x > m[n][e] + 8.0f;
                    }
            }
        if (__any_sync(0xffffffffu, above)) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float top = m[n][e];
#pragma unroll
                    for (int u = 0; u < kU; ++u) top = fmaxf(top, fmaxf(sc[n][u][e], sc[n][u][2 + e]));
#pragma unroll
                    for (int x = 4; x < 32; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
                    const float f = top == m[n][e] ? 1.0f : exp2_fast(m[n][e] - top);
                    m[n][e] = top;
                    l[n][e] *= f;
#pragma unroll
                    for (int i = 0; i < kM; ++i) o[n][i][e] *= f, o[n][i][2 + e] *= f;
                }
        }
        // ---- probabilities as the operand of the second product
        uint32_t ph[NT][kU][2], pl[NT][kU][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const float m0 = m[n][0] == -INFINITY ? 0.0f : m[n][0], m1 = m[n][1] == -INFINITY ? 0.0f : m[n][1];
#pragma unroll
            for (int u = 0; u < kU; ++u)
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    float p0 = exp2_fast(sc[n][u][r * 2] - m0), p1 = exp2_fast(sc[n][u][r * 2 + 1] - m1);
                    l[n][0] += p0, l[n][1] += p1;
                    if (!kWide) p0 *= vs[u][r], p1 *= vs[u][r];
                    const uint32_t hi = pack16<kHalf>(p0, p1);
                    const float2 h = unpack16<kHalf>(hi);
                    ph[n][u][r] = transpose8(hi);
                    pl[n][u][r] = transpose8(pack16<kHalf>(p0 - h.x, p1 - h.y));
                }
        }
        // ---- values
#pragma unroll
        for (int u = 0; u < kU; ++u) {
            uint32_t vr[4][kVC * 2];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int64_t at = __shfl_sync(0xffffffffu, info.at, u * 16 + (i >> 1) * 8 + 2 * t + (i & 1));
                const char* p = static_cast<const char*>(a.c.v) + at * kBytes;
                if (kVC >= 2) {
#pragma unroll
                    for (int c = 0; c < kVC / 2; ++c) {
                        uint4 x = make_uint4(0, 0, 0, 0);
                        const int off = c * 128 + g * 16;
                        if (at >= 0 && off < dim * kBytes) x = ldg16(p + off);
                        vr[i][c * 4] = x.x, vr[i][c * 4 + 1] = x.y, vr[i][c * 4 + 2] = x.z, vr[i][c * 4 + 3] = x.w;
                    }
                } else {
                    uint2 x = make_uint2(0, 0);
                    if (at >= 0 && g * 8 < dim) x = ldg8(p + g * 8);
                    vr[i][0] = x.x, vr[i][1] = x.y;
                }
            }
#pragma unroll
            for (int i = 0; i < kM; ++i) {
                uint32_t f[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) {  // row block r & 1, tokens r >> 1
                    const int x = i + (r & 1) * kM;
                    const uint32_t* v0 = vr[(r >> 1) * 2];
                    const uint32_t* v1 = vr[(r >> 1) * 2 + 1];
                    if (kWide) {
                        f[r] = __byte_perm(v0[x / 2], v1[x / 2], (x & 1) ? 0x7632 : 0x5410);
                    } else {
                        const int e = x & 3;
                        // the codes in the low (int8) or high (e4m3) bytes of the halves
                        const uint32_t sel = KIND == CHM_INT8 ? (uint32_t)(e | (4 + e) << 8) : (uint32_t)(e << 4 | (4 + e) << 12);
                        f[r] = codes_to_bf16<KIND>(__byte_perm(v0[x / 4], v1[x / 4], sel));
                    }
                }
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    mma<kHalf>(o[n][i], f[0], f[1], f[2], f[3], ph[n][u][0], ph[n][u][1]);
                    mma<kHalf>(o[n][i], f[0], f[1], f[2], f[3], pl[n][u][0], pl[n][u][1]);
                }
            }
        }
    }

    // ---- the warps' parts joined
    bad = __syncthreads_or(bad);
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            float sum = l[n][e];
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
            const int hh = n * 8 + 2 * t + e;
            if (g == 0) s_m[warp][hh] = m[n][e], s_l[warp][hh] = sum;
#pragma unroll
            for (int half = 0; half < 2; ++half)
#pragma unroll
                for (int i = 0; i < kM; ++i) {
                    const int x = i + half * kM;
                    const int d = kWide ? (x / 8) * 64 + g * 8 + x % 8
                                        : kE >= 16 ? (x / 16) * 128 + g * 16 + x % 16 : g * 8 + x;
                    s_o[warp][hh][d] = o[n][i][half * 2 + e];
                }
        }
    __syncthreads();
    for (int i = threadIdx.x; i < nh * dim; i += kAttThreads) {
        const int hh = i / dim, d = i - hh * dim;
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < kAttWarps; ++w) top = fmaxf(top, s_m[w][hh]);
        float sum = 0.0f, acc = 0.0f;
#pragma unroll
        for (int w = 0; w < kAttWarps; ++w) {
            const float f = s_m[w][hh] == -INFINITY ? 0.0f : exp2_fast(s_m[w][hh] - top);
            sum += f * s_l[w][hh];
            acc += f * s_o[w][hh][d];
        }
        float y = sum == 0.0f ? 0.0f : acc / sum;
        float e = sum == 0.0f ? -INFINITY : (top + log2f(sum)) * kLn2;
        if (bad) y = e = __int_as_float(0x7FC00000);
        const int64_t at = b * a.out_b + (h0 + hh) * a.out_h + d;
        if (a.q_type == CHM_FP16)
            static_cast<__half*>(a.out)[at] = __float2half_rn(y);
        else
            static_cast<__nv_bfloat16*>(a.out)[at] = __float2bfloat16_rn(y);
        if (d == 0 && a.lse) a.lse[(int64_t)b * a.q_heads + h0 + hh] = e;
    }
}

template <int DMAX, int KIND, int NT>
static void launch_attention(AttArgs a, cudaStream_t st) {
    a.blocks = (a.group + 8 * NT - 1) / (8 * NT);
    const dim3 grid((unsigned)(a.c.heads * a.blocks), (unsigned)a.batch);
    paged_attention_kernel<DMAX, KIND, NT><<<grid, kAttThreads, 0, st>>>(a);
}

template <int KIND>
static void dispatch_dim(const AttArgs& a, cudaStream_t st) {
    // more than 8 query heads per key head take two blocks of 8 at a time, so
    // that up to 16 read the cache once; at dim 256 the registers hold one block
    if (a.c.dim > 128) return launch_attention<256, KIND, 1>(a, st);
    if (a.c.dim > 64) {
        if (a.group > 8) return launch_attention<128, KIND, 2>(a, st);
        return launch_attention<128, KIND, 1>(a, st);
    }
    if (a.group > 8) return launch_attention<64, KIND, 2>(a, st);
    return launch_attention<64, KIND, 1>(a, st);
}

static chm_status refuse_attention(const char* why) {
    char msg[160];
    snprintf(msg, sizeof(msg), "paged_attention: %s", why);
    set_last_message(msg);
    return CHM_ERR_INVALID;
}

}  // namespace chm

extern "C" size_t chm_paged_attention_workspace_bytes(const chm_kv_cache* cache, int64_t batch, int32_t q_heads,
                                                      int32_t table_width) {
    (void)cache, (void)batch, (void)q_heads, (void)table_width;
    return 256;
}

extern "C" chm_status chm_paged_attention(const chm_kv_cache* cache, const chm_heads* q, const chm_heads* out,
                                          int32_t type, int64_t batch, const int32_t* tables, int64_t table_stride,
                                          int32_t table_width, const int32_t* lens, const int32_t* starts,
                                          float scale, float* lse, void* workspace, size_t workspace_bytes,
                                          void* stream) {
    using namespace chm;
    CHM_TRY(check_cache(cache, "paged_attention"));
    if (!q || !out) return refuse_attention("null queries or output");
    if (type != CHM_FP16 && type != CHM_BF16) return refuse_attention("queries are fp16 or bf16");
    if (type_bytes(cache->type) == 2 && cache->type != type)
        return refuse_attention("queries have the type of a 16-bit cache");
    if (batch < 0 || table_width < 0) return refuse_attention("negative size");
    if (q->heads < 1 || q->heads != out->heads || q->heads % cache->heads)
        return refuse_attention("query heads must be a multiple of the cache's heads");
    if (batch > 65535) return refuse_attention("at most 65535 sequences");
    if ((int64_t)table_width * cache->page_size > (1 << 30)) return refuse_attention("a table spans at most 2^30 tokens");
    if (batch == 0) return CHM_OK;
    if (!q->data || !out->data || !lens || (table_width > 0 && !tables)) return refuse_attention("null pointer");
    if (!workspace || workspace_bytes < chm_paged_attention_workspace_bytes(cache, batch, q->heads, table_width))
        return CHM_ERR_CAPACITY;
    AttArgs a{};
    a.c = *cache;
    a.q = q->data;
    a.out = out->data;
    a.q_b = q->batch_stride, a.q_h = q->head_stride, a.out_b = out->batch_stride, a.out_h = out->head_stride;
    a.q_type = type;
    a.batch = (int32_t)batch;
    a.q_heads = q->heads;
    a.group = q->heads / cache->heads;
    a.tables = tables;
    a.table_stride = table_stride;
    a.capacity = table_width * cache->page_size;
    a.lens = lens;
    a.starts = starts;
    a.scale_log2 = scale * kLog2e;
    a.lse = lse;
    a.by_page = FastDiv((uint32_t)cache->page_size);
    cudaStream_t st = (cudaStream_t)stream;
    switch (cache->type) {
        case CHM_FP16: dispatch_dim<CHM_FP16>(a, st); break;
        case CHM_BF16: dispatch_dim<CHM_BF16>(a, st); break;
        case CHM_INT8: dispatch_dim<CHM_INT8>(a, st); break;
        default: dispatch_dim<CHM_E4M3>(a, st); break;
    }
    return launch_status("paged_attention_kernel");
}
