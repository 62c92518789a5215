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
// runs are its operand registers as they come: each lane copies its own runs
// into a ring of its own in shared memory, steps ahead, and reads them back;
// no layout to swizzle, no barrier.
#include <algorithm>
#include <cmath>
#include <cstdio>

#include "kv_cache.cuh"

namespace chm {

constexpr int kAttWarps = 4;
constexpr int kAttThreads = kAttWarps * 32;
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.69314718055994530942f;

struct Plan;
struct Boundary;

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
    int32_t capacity;     // table_width * page_size
    int32_t unit_tokens;  // tokens per unit of work
    FastDiv by_unit;
    Plan* plan;
    Boundary* boundaries;
    float* parts;
    const int32_t* lens;
    const int32_t* starts;
    float scale_log2;
    float* lse;
    FastDiv by_page;
};

// Asynchronous copies of N bytes into shared memory; zeros where `on` is false.
template <int N>
__device__ __forceinline__ void copy_async(uint32_t to, const void* from, bool on) {
    const int bytes = on ? N : 0;
    if (N == 16)
        asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
    else
        asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(to), "l"(from), "n"(N), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// Until all but the newest N groups of this thread's copies have landed.
template <int N>
__device__ __forceinline__ void copies_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
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

// ---- how the work is split ------------------------------------------------------
//
// A segment is one sequence's tokens for one block of query heads that share a
// key head.  It is cut into tiles (a step of all warps), and the tiles of all
// segments, in the order (sequence, block, tile), are dealt out evenly: with
// `per` = ceil(units / blocks), block c takes units [c * per, (c + 1) * per).
// So the lengths, which only the device knows, do not matter to the balance, a
// long sequence spreads over the device and short ones stay whole.  A segment
// that crosses a block boundary leaves a part (unnormalised output, maximum,
// sum) per block in the workspace, and attention_join_kernel adds them in order.
struct Plan {
    int per;    // units per block
    int total;  // units
};
struct Boundary {  // the first segment of a block
    int seq, seg;
    int first, units;  // its first unit, its units
};

struct Range {
    int first, end;  // positions attended to
    int units;
    bool bad;  // the length does not fit the table
};

__device__ __forceinline__ Range sequence_range(const AttArgs& a, int b) {
    Range r;
    r.first = a.starts ? min(max(a.starts[b], 0), a.capacity) : 0;
    r.end = a.lens[b];
    r.bad = r.end > a.capacity;
    if (r.bad) r.end = 0;
    r.units = max(1, (int)a.by_unit.div((uint32_t)(max(r.end - r.first, 0) + a.unit_tokens - 1)));
    return r;
}

// The parts of a segment of 8 * NT heads: `slots` of [heads][DMAX + 2] floats,
// the last two the maximum and the sum.  Block c uses slot 2c for the segment
// that holds its first unit and 2c + 1 for its last.
template <int DMAX>
__device__ __forceinline__ float* part_row(float* parts, int slot, int heads, int hh) {
    return parts + ((int64_t)slot * heads + hh) * (DMAX + 4);
}

__device__ __forceinline__ void store_row(const AttArgs& a, int b, int head, int d, float y) {
    const int64_t at = b * a.out_b + head * a.out_h + d;
    if (a.q_type == CHM_FP16)
        static_cast<__half*>(a.out)[at] = __float2half_rn(y);
    else
        static_cast<__nv_bfloat16*>(a.out)[at] = __float2bfloat16_rn(y);
}

// DMAX: dim rounded up to 64, 128 or 256; NT: blocks of 8 query heads.
template <int DMAX, int KIND, int NT>
struct Shape {
    static constexpr bool kWide = KIND == CHM_FP16 || KIND == CHM_BF16;  // 16-bit cache
    static constexpr int kBytes = kWide ? 2 : 1;
    static constexpr int kU = DMAX * kBytes <= 128 ? 2 : 1;  // groups of 16 tokens per warp and step
    static constexpr int kTok = 16 * kU;
    static constexpr int kTile = kAttWarps * kTok;
    static constexpr int kHeads = 8 * NT;
    // blocks per SM that the registers (the output tiles) leave room for
    static constexpr int kResident = DMAX * kBytes > 256 ? 1 : DMAX > 128 || NT > 1 ? 2 : 3;
    // A warp's copies in flight: kStages steps of keys and of values, which fill
    // the shared memory that the resident blocks have, about 190 KB per SM.
    static constexpr int kSlot = kTok * DMAX * kBytes;
    static constexpr int kStages = (kResident == 3 ? 8192 : kResident == 2 ? 12288 : 16384) / kSlot;
    // shared memory: q as operand registers (high and low part), rings, scales;
    // at a segment's end the warps' parts take the place of the rings
    static constexpr int kQ = 2 * NT * (DMAX / 32) * 512;
    static constexpr int kRing = kAttWarps * kStages * 2 * kSlot;
    static constexpr int kScales = kWide ? 0 : kAttWarps * kStages * 2 * kTok * 4;
    static constexpr int kRow = DMAX + 4;
    static constexpr int kOut = kAttWarps * kHeads * (kRow + 2) * 4;
    static_assert(kOut <= kRing, "the warps' parts fit in the rings");
    static constexpr int kShared = kQ + kRing + kScales;
    static_assert(kResident * (kShared + 1024) <= 227 * 1024, "the resident blocks' shared memory");
};

template <int DMAX, int KIND, int NT>
__global__ void __launch_bounds__(kAttThreads, Shape<DMAX, KIND, NT>::kResident)
    paged_attention_kernel(const AttArgs a) {
    using S = Shape<DMAX, KIND, NT>;
    constexpr bool kWide = S::kWide;
    constexpr bool kHalf = KIND == CHM_FP16;  // type of the products
    constexpr int kBytes = S::kBytes, kU = S::kU, kTok = S::kTok, kTile = S::kTile, kHeads = S::kHeads;
    constexpr int kStages = S::kStages, kSlot = S::kSlot;
    constexpr int kKC = DMAX * kBytes / 64;     // 16-byte runs of a key per thread
    constexpr int kRuns = DMAX / 32;            // operand runs of q
    constexpr int kE = DMAX / 8;                // value elements per thread and token
    constexpr int kVB = kE * kBytes < 16 ? 8 : 16;  // bytes of a run of a value
    constexpr int kVC = kE * kBytes / kVB;      // runs of a value per thread
    constexpr int kM = kE / 2;                  // 16-row blocks of the output
    constexpr int kRow = S::kRow;
    static_assert(S::kResident >= 1 && kStages >= 1, "shape");
    extern __shared__ __align__(16) uint8_t smem[];
    uint4(*s_q)[NT][kRuns][32] = reinterpret_cast<uint4(*)[NT][kRuns][32]>(smem);
    float(*s_o)[kHeads][kRow] = reinterpret_cast<float(*)[kHeads][kRow]>(smem + S::kQ);
    float(*s_m)[kHeads] = reinterpret_cast<float(*)[kHeads]>(smem + S::kQ + kAttWarps * kHeads * kRow * 4);
    float(*s_l)[kHeads] = s_m + kAttWarps;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int dim = a.c.dim;
    // This warp's ring: per stage the keys' runs, then the values', each lane's
    // own 16 bytes in a row of 512, so that a lane reads back what it copied.
    const uint8_t* const ring = smem + S::kQ + warp * (kStages * 2 * kSlot);
    const float* const scales = reinterpret_cast<const float*>(smem + S::kQ + S::kRing) + warp * (kStages * 2 * kTok);
    const uint32_t ring_at = (uint32_t)__cvta_generic_to_shared(ring) + lane * 16;
    const uint32_t ring_v = (uint32_t)__cvta_generic_to_shared(ring) + lane * kVB;
    const uint32_t scales_at = (uint32_t)__cvta_generic_to_shared(scales) + lane * 4;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    // ---- this block's units (every warp works them out for itself)
    const int segs = a.c.heads * a.blocks;
    int total = 0;
    for (int b = lane; b < a.batch; b += 32) total += sequence_range(a, b).units;
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) total += __shfl_xor_sync(0xffffffffu, total, x);
    total *= segs;
    const int per = (total + (int)gridDim.x - 1) / (int)gridDim.x;
    int u = blockIdx.x * per;
    const int u1 = min(u + per, total);
    if (blockIdx.x == 0 && threadIdx.x == 0) *a.plan = Plan{per, total};
    if (u >= u1) return;
    int b = 0, before = 0;  // the sequence that holds unit u, the units of those before it
    for (int base = 0; base < a.batch; base += 32) {
        const int n = base + lane < a.batch ? sequence_range(a, base + lane).units * segs : 0;
        int sum = n;
#pragma unroll
        for (int x = 1; x < 32; x <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, sum, x);
            if (lane >= x) sum += y;
        }
        const uint32_t past = __ballot_sync(0xffffffffu, base + lane < a.batch && before + sum > u);
        if (past) {
            const int at = __ffs(past) - 1;
            b = base + at;
            before += __shfl_sync(0xffffffffu, sum - n, at);
            break;
        }
        before += __shfl_sync(0xffffffffu, sum, 31);
    }
    Range r = sequence_range(a, b);
    const bool split_q = !kWide && a.q_type == CHM_FP16;
    const char* const kbase = static_cast<const char*>(a.c.k);
    const char* const vbase = static_cast<const char*>(a.c.v);

    for (int piece = 0; u < u1; ++piece) {
        const int in_seq = u - before;
        const int seg = in_seq / r.units;
        const int unit0 = in_seq - seg * r.units;
        const int unit1 = min(r.units, unit0 + (u1 - u));
        const bool whole = unit1 - unit0 == r.units;
        if (piece == 0 && threadIdx.x == 0) a.boundaries[blockIdx.x] = Boundary{b, seg, u - unit0, r.units};
        const int head = seg / a.blocks;
        const int h0 = head * a.group + (seg - head * a.blocks) * kHeads;  // first query head
        const int nh = min(kHeads, (head + 1) * a.group - h0);
        const int32_t* table = a.tables + b * a.table_stride;
        const int first = r.first + unit0 * a.unit_tokens;
        const int end = unit1 == r.units ? r.end : r.first + unit1 * a.unit_tokens;
        bool bad = r.bad;

        // Token `pos` of the range, one per lane: its page, then its place and scales.
        auto page_of = [&](int pos) { return pos < end ? table[a.by_page.div((uint32_t)pos)] : 0; };
        int64_t at = -1;  // element offset of this lane's token of the newest step, -1: none
        auto place = [&](int pos, int page, int stage) {
            at = -1;
            int64_t scale = -1;
            if (pos < end) {
                if (page < 0 || page >= a.c.num_pages) {
                    bad = true;
                } else {
                    const uint32_t within = (uint32_t)pos - a.by_page.div((uint32_t)pos) * (uint32_t)a.c.page_size;
                    at = page * a.c.page_stride + (int64_t)head * a.c.head_stride +
                         (int64_t)within * a.c.token_stride;
                    if (!kWide) scale = ((int64_t)page * a.c.heads + head) * a.c.page_size + within;
                }
            }
            if (!kWide && lane < kTok) {
                const int64_t x = max(scale, (int64_t)0);
                copy_async<4>(scales_at + stage * (2 * kTok * 4), a.c.k_scale + x, scale >= 0);
                copy_async<4>(scales_at + stage * (2 * kTok * 4) + kTok * 4, a.c.v_scale + x, scale >= 0);
            }
        };
        auto copy_keys = [&](int stage) {
            const uint32_t to = ring_at + stage * 2 * kSlot;
#pragma unroll
            for (int i = 0; i < kU; ++i)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int64_t x = __shfl_sync(0xffffffffu, at, i * 16 + h * 8 + g);
                    const char* p = kbase + max(x, (int64_t)0) * kBytes + t * 16;
#pragma unroll
                    for (int c = 0; c < kKC; ++c) {
                        const bool in = c * 64 + t * 16 < dim * kBytes;
                        copy_async<16>(to + ((i * 2 + h) * kKC + c) * 512, in ? p + c * 64 : p, x >= 0 && in);
                    }
                }
        };
        auto copy_values = [&](int stage) {
            const uint32_t to = ring_v + stage * 2 * kSlot + kSlot;
#pragma unroll
            for (int i = 0; i < kU; ++i)
#pragma unroll
                for (int h = 0; h < 4; ++h) {
                    const int64_t x = __shfl_sync(0xffffffffu, at, i * 16 + (h >> 1) * 8 + 2 * t + (h & 1));
                    const char* p = vbase + max(x, (int64_t)0) * kBytes;
#pragma unroll
                    for (int c = 0; c < kVC; ++c) {
                        const int off = c * 128 + g * kVB;
                        const bool in = off < dim * kBytes;
                        copy_async<kVB>(to + ((i * 4 + h) * kVC + c) * (32 * kVB), in ? p + off : p, x >= 0 && in);
                    }
                }
        };

        int pos = first + warp * kTok + lane % kTok;  // this lane's token of the newest step
        int base = first + warp * kTok;               // the oldest step's first
        int next_page = page_of(pos);
#pragma unroll
        for (int i = 0; i < kStages; ++i) {
            const int page = next_page;
            next_page = page_of(pos + kTile);
            if (base + i * kTile < end) {
                place(pos, page, i);
                copy_keys(i);
                copies_commit();
                copy_values(i);
                copies_commit();
            } else {
                copies_commit();
                copies_commit();
            }
            pos += kTile;
        }

        // q: lane (g, t) of a run holds the 8 elements that its key runs meet
        for (int i = threadIdx.x; i < NT * kRuns * 32; i += kAttThreads) {
            const int ln = i & 31, run = (i >> 5) % kRuns, nt = (i >> 5) / kRuns;
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
                        const int64_t qa = b * a.q_b + (h0 + hh) * a.q_h + d;
                        x[e] = a.q_type == CHM_FP16 ? __half2float(static_cast<const __half*>(a.q)[qa])
                                                    : __bfloat162float(static_cast<const __nv_bfloat16*>(a.q)[qa]);
                    }
                }
                hi[j] = pack16<kHalf>(x[0], x[1]);
                const float2 y = unpack16<kHalf>(hi[j]);
                lo[j] = pack16<kHalf>(x[0] - y.x, x[1] - y.y);
            }
            s_q[0][nt][run][ln] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
            s_q[1][nt][run][ln] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
        }
        __syncthreads();

        float o[NT][kM][4] = {};
        float m[NT][2], l[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) m[n][0] = m[n][1] = -INFINITY, l[n][0] = l[n][1] = 0.0f;

        // The copies run kStages steps ahead: a step's keys and values are copied into the
        // slots that the step kStages before it has just been read from.
        int stage = 0;
        for (; base < end; base += kTile) {
            const uint8_t* const keys = ring + stage * 2 * kSlot + lane * 16;
            const uint8_t* const values = ring + stage * 2 * kSlot + kSlot + lane * kVB;
            const bool more = base + kStages * kTile < end;
            const int page = next_page;
            next_page = page_of(pos + kTile);
            copies_wait<2 * kStages - 1>();
            __syncwarp();
            // ---- scores
            float sc[NT][kU][4] = {};
#pragma unroll
            for (int i = 0; i < kU; ++i)
#pragma unroll
                for (int c = 0; c < kKC; ++c) {
                    const uint4 r0 = *reinterpret_cast<const uint4*>(keys + (i * 2 * kKC + c) * 512);
                    const uint4 r1 = *reinterpret_cast<const uint4*>(keys + ((i * 2 + 1) * kKC + c) * 512);
                    const uint32_t w0[4] = {r0.x, r0.y, r0.z, r0.w}, w1[4] = {r1.x, r1.y, r1.z, r1.w};
                    // pairs of the run: 4 words of a 16-bit cache, 8 pairs of codes
#pragma unroll
                    for (int j = 0; j < (kWide ? 1 : 2); ++j) {
                        uint32_t p0[4], p1[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            if (kWide) {
                                p0[e] = w0[e], p1[e] = w1[e];
                            } else {
                                const uint32_t x0 = w0[j * 2 + (e >> 1)], x1 = w1[j * 2 + (e >> 1)];
                                const uint32_t sel =
                                    KIND == CHM_INT8 ? ((e & 1) ? 0x4342 : 0x4140) : ((e & 1) ? 0x3424 : 0x1404);
                                p0[e] = codes_to_bf16<KIND>(__byte_perm(x0, 0, sel));
                                p1[e] = codes_to_bf16<KIND>(__byte_perm(x1, 0, sel));
                            }
                        }
                        const int run = kWide ? c : c * 2 + j;
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            uint4 bq = s_q[0][n][run][lane];
                            mma<kHalf>(sc[n][i], p0[0], p1[0], p0[1], p1[1], bq.x, bq.y);
                            mma<kHalf>(sc[n][i], p0[2], p1[2], p0[3], p1[3], bq.z, bq.w);
                            if (!kWide && split_q) {
                                bq = s_q[1][n][run][lane];
                                mma<kHalf>(sc[n][i], p0[0], p1[0], p0[1], p1[1], bq.x, bq.y);
                                mma<kHalf>(sc[n][i], p0[2], p1[2], p0[3], p1[3], bq.z, bq.w);
                            }
                        }
                    }
                }
            // ---- running maximum; it follows the scores only when one passes it by more than 2^8
            float vscale[kU][2];
            bool above = false;
#pragma unroll
            for (int i = 0; i < kU; ++i)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int src = i * 16 + h * 8 + g;
                    const bool on = base + src < end;
                    float f = a.scale_log2;
                    if (!kWide) {
                        f *= scales[stage * 2 * kTok + src];
                        vscale[i][h] = scales[stage * 2 * kTok + kTok + src];
                    }
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            float& x = sc[n][i][h * 2 + e];
                            x = on ? x * f : -INFINITY;
                            above = above || x > m[n][e] + 8.0f;
                        }
                }
            if (!kWide) __syncwarp();  // the scales are read; the next step's take their place
            if (more) {
                place(pos, page, stage);
                copy_keys(stage);
            }
            copies_commit();
            pos += kTile;
            if (__any_sync(0xffffffffu, above)) {
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float top = m[n][e];
#pragma unroll
                        for (int i = 0; i < kU; ++i) top = fmaxf(top, fmaxf(sc[n][i][e], sc[n][i][2 + e]));
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
                for (int i = 0; i < kU; ++i)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        float p0 = exp2_fast(sc[n][i][h * 2] - m0), p1 = exp2_fast(sc[n][i][h * 2 + 1] - m1);
                        l[n][0] += p0, l[n][1] += p1;
                        if (!kWide) p0 *= vscale[i][h], p1 *= vscale[i][h];
                        const uint32_t hi = pack16<kHalf>(p0, p1);
                        const float2 y = unpack16<kHalf>(hi);
                        ph[n][i][h] = transpose8(hi);
                        pl[n][i][h] = transpose8(pack16<kHalf>(p0 - y.x, p1 - y.y));
                    }
            }
            // ---- values
            copies_wait<2 * kStages - 1>();
#pragma unroll
            for (int i = 0; i < kU; ++i) {
                uint32_t vr[4][kVC * kVB / 4];
#pragma unroll
                for (int h = 0; h < 4; ++h)
#pragma unroll
                    for (int c = 0; c < kVC; ++c) {
                        const uint8_t* x = values + ((i * 4 + h) * kVC + c) * (32 * kVB);
                        if (kVB == 16) {
                            const uint4 w = *reinterpret_cast<const uint4*>(x);
                            vr[h][c * 4] = w.x, vr[h][c * 4 + 1] = w.y, vr[h][c * 4 + 2] = w.z, vr[h][c * 4 + 3] = w.w;
                        } else {
                            const uint2 w = *reinterpret_cast<const uint2*>(x);
                            vr[h][0] = w.x, vr[h][1] = w.y;
                        }
                    }
#pragma unroll
                for (int j = 0; j < kM; ++j) {
                    uint32_t f[4];
#pragma unroll
                    for (int h = 0; h < 4; ++h) {  // row block h & 1, tokens h >> 1
                        const int x = j + (h & 1) * kM;
                        const uint32_t* v0 = vr[(h >> 1) * 2];
                        const uint32_t* v1 = vr[(h >> 1) * 2 + 1];
                        if (kWide) {
                            f[h] = __byte_perm(v0[x / 2], v1[x / 2], (x & 1) ? 0x7632 : 0x5410);
                        } else {
                            // the codes in the low (int8) or high (e4m3) bytes of the halves
                            const int e = x & 3;
                            const uint32_t sel =
                                KIND == CHM_INT8 ? (uint32_t)(e | (4 + e) << 8) : (uint32_t)(e << 4 | (4 + e) << 12);
                            f[h] = codes_to_bf16<KIND>(__byte_perm(v0[x / 4], v1[x / 4], sel));
                        }
                    }
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        mma<kHalf>(o[n][j], f[0], f[1], f[2], f[3], ph[n][i][0], ph[n][i][1]);
                        mma<kHalf>(o[n][j], f[0], f[1], f[2], f[3], pl[n][i][0], pl[n][i][1]);
                    }
                }
            }
            if (more) copy_values(stage);
            copies_commit();
            stage = stage + 1 == kStages ? 0 : stage + 1;
        }
        copies_wait<0>();

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
                for (int x = 0; x < kE; x += 4) {
                    const int d = kWide ? (x / 8) * 64 + g * 8 + x % 8
                                        : kE >= 16 ? (x / 16) * 128 + g * 16 + x % 16 : g * 8 + x;
                    const int j = x % kM, k = x / kM * 2 + e;
                    *reinterpret_cast<float4*>(&s_o[warp][hh][d]) =
                        make_float4(o[n][j][k], o[n][j + 1][k], o[n][j + 2][k], o[n][j + 3][k]);
                }
            }
        __syncthreads();
        for (int hh = warp; hh < nh; hh += kAttWarps) {
            float top = -INFINITY, sum = 0.0f, f[kAttWarps];
#pragma unroll
            for (int w = 0; w < kAttWarps; ++w) top = fmaxf(top, s_m[w][hh]);
#pragma unroll
            for (int w = 0; w < kAttWarps; ++w) {
                f[w] = s_m[w][hh] == -INFINITY ? 0.0f : exp2_fast(s_m[w][hh] - top);
                sum += f[w] * s_l[w][hh];
            }
            if (bad) sum = __int_as_float(0x7FC00000);
            float* part = part_row<DMAX>(a.parts, 2 * blockIdx.x + (piece > 0), kHeads, hh);
            for (int d = lane; d < dim; d += 32) {
                float acc = 0.0f;
#pragma unroll
                for (int w = 0; w < kAttWarps; ++w) acc += f[w] * s_o[w][hh][d];
                if (whole)
                    store_row(a, b, h0 + hh, d, sum == 0.0f ? 0.0f : bad ? sum : acc / sum);
                else
                    part[d] = acc;
            }
            if (lane == 0) {
                if (!whole)
                    part[DMAX] = top, part[DMAX + 1] = sum;
                else if (a.lse)
                    a.lse[(int64_t)b * a.q_heads + h0 + hh] = sum == 0.0f ? -INFINITY : (top + log2f(sum)) * kLn2;
            }
        }
        __syncthreads();  // the parts are read; the next segment's copies take their place
        u += unit1 - unit0;
        if (u == before + r.units * segs && u < u1) {
            before = u;
            r = sequence_range(a, ++b);
        }
    }
}

// Block (c, h): if the first segment of block c + 1 began in block c, head h of
// that segment from its parts, in the order of the blocks.
constexpr int kJoinThreads = 128;

template <int DMAX, int NT>
__global__ void __launch_bounds__(kJoinThreads) attention_join_kernel(const AttArgs a) {
    constexpr int kHeads = 8 * NT;
    constexpr int kWarps = kJoinThreads / 32;
    constexpr int kV = DMAX / 32;  // elements per lane
    __shared__ float s_acc[kWarps][DMAX];
    __shared__ float s_top[kWarps], s_sum[kWarps];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int per = a.plan->per;
    const int c = blockIdx.x + 1;
    if (c * (int64_t)per >= a.plan->total) return;
    const Boundary s = a.boundaries[c];
    const int c0 = s.first / per, c1 = (s.first + s.units - 1) / per;
    if (s.first == c * per || c != c0 + 1) return;
    const int head = s.seg / a.blocks;
    const int h0 = head * a.group + (s.seg - head * a.blocks) * kHeads;
    const int hh = blockIdx.y;
    if (h0 + hh >= (head + 1) * a.group) return;
    // each warp: every kWarps-th part, with a running maximum
    float top = -INFINITY, sum = 0.0f, acc[kV] = {};
#pragma unroll 4
    for (int i = c0 + warp; i <= c1; i += kWarps) {
        const int slot = 2 * i + (i == c0 && c0 * per != s.first);
        const float* part = part_row<DMAX>(a.parts, slot, kHeads, hh);
        const float m = part[DMAX], l = part[DMAX + 1];
        const float now = fmaxf(top, m);
        const float f = top == now ? 1.0f : exp2_fast(top - now);
        const float w = m == -INFINITY ? 0.0f : exp2_fast(m - now);
        top = now;
        sum = sum * f + l * w;
#pragma unroll
        for (int v = 0; v < kV; ++v) acc[v] = acc[v] * f + part[v * 32 + lane] * w;
    }
#pragma unroll
    for (int v = 0; v < kV; ++v) s_acc[warp][v * 32 + lane] = acc[v];
    if (lane == 0) s_top[warp] = top, s_sum[warp] = sum;
    __syncthreads();
    top = -INFINITY, sum = 0.0f;
    float f[kWarps];
#pragma unroll
    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, s_top[w]);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
        f[w] = s_top[w] == -INFINITY ? 0.0f : exp2_fast(s_top[w] - top);
        sum += f[w] * s_sum[w];
    }
    for (int d = threadIdx.x; d < a.c.dim; d += kJoinThreads) {
        float y = 0.0f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) y += f[w] * s_acc[w][d];
        store_row(a, s.seq, h0 + hh, d, sum == 0.0f ? 0.0f : sum != sum ? sum : y / sum);
    }
    if (threadIdx.x == 0 && a.lse)
        a.lse[(int64_t)s.seq * a.q_heads + h0 + hh] = sum == 0.0f ? -INFINITY : (top + log2f(sum)) * kLn2;
}

static int sm_count() {
    static int cached[64];
    int dev = 0, n = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev >= 64) {
        cudaGetLastError();
        return 148;
    }
    if (cached[dev] > 0) return cached[dev];
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) {
        cudaGetLastError();
        return 148;
    }
    return cached[dev] = n;
}

struct Layout {
    int blocks;       // thread blocks of the main kernel
    int unit_tokens;  // tokens per unit
    bool joins;       // whether a segment can be split
};

template <int DMAX, int KIND, int NT>
struct Launch {
    using S = Shape<DMAX, KIND, NT>;

    static Layout layout(const AttArgs& a) {
        Layout y;
        // up to 4 tiles a segment stays whole: a second launch costs more than they do
        const int whole = 4 * S::kTile;
        y.unit_tokens = a.capacity <= whole ? whole : S::kTile;
        y.joins = a.capacity > whole;
        const int64_t segs = (int64_t)a.c.heads * ((a.group + S::kHeads - 1) / S::kHeads);
        const int64_t units = a.batch * segs * std::max<int64_t>(1, ((int64_t)a.capacity + y.unit_tokens - 1) / y.unit_tokens);
        y.blocks = (int)std::min<int64_t>(units, (int64_t)sm_count() * S::kResident);
        return y;
    }
    // Units are counted in 32 bits.
    static bool fits(const AttArgs& a) {
        const Layout y = layout(a);
        const int64_t segs = (int64_t)a.c.heads * ((a.group + S::kHeads - 1) / S::kHeads);
        const int64_t per_seq = std::max<int64_t>(1, ((int64_t)a.capacity + y.unit_tokens - 1) / y.unit_tokens);
        return segs * per_seq <= (INT32_MAX - (1 << 16)) / std::max(1, a.batch);
    }
    template <typename A>
    static void carve(A& arena, const Layout& y, AttArgs* a) {
        auto plan = arena.template take<Plan>(1);
        auto bounds = arena.template take<Boundary>(y.blocks);
        auto parts = arena.template take<float>(y.joins ? (size_t)2 * y.blocks * S::kHeads * (DMAX + 4) : 0);
        if (a) {
            a->plan = (Plan*)plan;
            a->boundaries = (Boundary*)bounds;
            a->parts = (float*)parts;
        }
    }
    static size_t workspace(const AttArgs& a) {
        Counter c;
        carve(c, layout(a), nullptr);
        return c.s.off;
    }
    struct Counter {
        Sizer s;
        template <typename T>
        void* take(size_t n) {
            s.take<T>(n);
            return nullptr;
        }
    };
    static chm_status run(AttArgs a, void* ws, size_t ws_bytes, cudaStream_t st) {
        const Layout y = layout(a);
        Arena arena(ws, ws_bytes);
        carve(arena, y, &a);
        if (arena.overflow) return CHM_ERR_CAPACITY;
        a.blocks = (a.group + S::kHeads - 1) / S::kHeads;
        a.unit_tokens = y.unit_tokens;
        a.by_unit = FastDiv((uint32_t)y.unit_tokens);
        static bool set[64];  // per device: the kernel may take this much shared memory
        int dev = 0;
        CHM_CUDA(cudaGetDevice(&dev));
        if (dev >= 64 || !set[dev]) {
            CHM_CUDA(cudaFuncSetAttribute(paged_attention_kernel<DMAX, KIND, NT>,
                                          cudaFuncAttributeMaxDynamicSharedMemorySize, S::kShared));
            if (dev < 64) set[dev] = true;
        }
        paged_attention_kernel<DMAX, KIND, NT><<<(unsigned)y.blocks, kAttThreads, S::kShared, st>>>(a);
        CHM_TRY(launch_status("paged_attention_kernel"));
        if (!y.joins || y.blocks < 2) return CHM_OK;
        // The join's blocks start while the main kernel's last ones run, and wait for its end.
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3((unsigned)(y.blocks - 1), (unsigned)std::min(S::kHeads, a.group));
        cfg.blockDim = dim3(kJoinThreads);
        cfg.stream = st;
        cudaLaunchAttribute attr{};
        attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr.val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = &attr;
        cfg.numAttrs = 1;
        CHM_CUDA(cudaLaunchKernelEx(&cfg, attention_join_kernel<DMAX, NT>, (const AttArgs)a));
        return CHM_OK;
    }
};

// Calls f on the Launch<> for a cache's type, dim and sharing.  More than 8
// query heads per key head take two blocks of 8 at a time, so that up to 16
// read the cache once; at dim 256 the registers hold one block.
template <int KIND, typename F>
static auto with_kind(const AttArgs& a, F f) {
    if (a.c.dim > 128) return f(Launch<256, KIND, 1>{});
    if (a.c.dim > 64) return a.group > 8 ? f(Launch<128, KIND, 2>{}) : f(Launch<128, KIND, 1>{});
    return a.group > 8 ? f(Launch<64, KIND, 2>{}) : f(Launch<64, KIND, 1>{});
}

template <typename F>
static auto with_launch(const AttArgs& a, F f) {
    switch (a.c.type) {
        case CHM_FP16: return with_kind<CHM_FP16>(a, f);
        case CHM_BF16: return with_kind<CHM_BF16>(a, f);
        case CHM_INT8: return with_kind<CHM_INT8>(a, f);
        default: return with_kind<CHM_E4M3>(a, f);
    }
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
    using namespace chm;
    if (check_cache(cache, "paged_attention") != CHM_OK) return 0;
    if (batch < 0 || batch > 65535 || q_heads < 1 || q_heads % cache->heads || table_width < 0 ||
        (int64_t)table_width * cache->page_size > (1 << 30))
        return 0;
    AttArgs a{};
    a.c = *cache;
    a.batch = (int32_t)batch;
    a.group = q_heads / cache->heads;
    a.capacity = table_width * cache->page_size;
    return with_launch(a, [&](auto l) { return l.workspace(a); });
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
    if (!with_launch(a, [&](auto l) { return l.fits(a); })) return refuse_attention("too much work for one call");
    return with_launch(a, [&](auto l) { return l.run(a, workspace, workspace_bytes, st); });
}
