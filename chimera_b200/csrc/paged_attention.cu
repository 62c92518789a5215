// Attention of one new token per sequence over a paged key-value cache
// (chm_paged_attention).
//
// out = sum_j p_j v_j / sum_j p_j with p_j = exp(scale <q, k_j> - m), one pass
// over the tokens with a running maximum m.  Every key and value is read once,
// for all the query heads that share it, so the bound is HBM: 2 G flops per
// element read for G heads, where the device has time for 500 per bf16 element.
//
// The products run on mma.sync m16n8k16 with the tokens (for the scores) and
// the elements of the value vector (for the output) as the 16 rows and the
// query heads of one key head as the 8 columns:
//   S^T [tokens x heads] = K [tokens x dim] Q^T,   O^T [dim x heads] += V^T P^T.
// Both contractions may take their index in any order, so a thread's 16-byte
// runs are its operand registers as they come; 8-bit codes become fp16 numbers in
// registers.  (tcgen05 would take K and V from shared memory only: codes would go
// there a second time, and values transposed.  At 8 cycles per product the tensor
// cores are busy for 9 to 20% of the time as it is.)  Each warp copies its runs
// into a ring of its own in shared memory ahead of their use.
//
// One B200, us on the device: 64 sequences of up to 4,096 tokens (32 query heads on
// 8 key heads of 128, bf16) 94 for 546 MB, 5.8 TB/s; one sequence of 262,144 tokens
// (28 on 4 of 128, int8) 58 for 277 MB, 4.8 TB/s; 128 documents of up to 2,000
// tokens (20 on 4 of 64, e4m3) 35 for 72 MB (as calls among others 99, 65 and 37).
// A call that joins parts costs 6 for one sequence of no tokens and
// 14 for 128 of them: two launches, some 3 us from a block's start to its first
// product, 1 to 2 at each segment's end.  Beside that, 16-bit caches wait for memory;
// 8-bit ones are bound by the instructions of 10 to 12 warps per SM (0.56 issued per
// cycle; more warps, fewer instructions or shorter chains of products did not change
// the time).
#include <algorithm>
#include <cmath>
#include <cstdio>

#include <cuda_fp8.h>

#include "kv_cache.cuh"

namespace chm {

constexpr int kAttWarps = 4;
constexpr int kAttThreads = kAttWarps * 32;
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.69314718055994530942f;
constexpr uint32_t kNowhere = 0xFFFFFFFFu;

struct Plan {
    int per;    // units per block
    int total;  // units
};
struct Boundary {  // the segment that holds a block's first unit
    int seq, seg;
    int first, units;  // its first unit, its units
};

struct AttArgs {
    chm_kv_cache c;
    uint32_t page16, head16, token16;  // the cache's strides in 16 bytes
    const void* q;
    void* out;
    int64_t q_b, q_h, out_b, out_h;
    int32_t q_type;
    bool q_wide;                    // q in 16-byte loads
    int32_t batch, q_heads, group;  // group: query heads per key head
    int32_t blocks;                 // blocks of 8 * NT query heads per key head
    const int32_t* tables;
    int64_t table_stride;
    int32_t capacity;     // table_width * page_size
    int32_t unit_tokens;  // tokens per unit of work
    int32_t start_units;  // units that a segment counts before its tokens
    FastDiv by_unit, by_page;
    const int32_t* lens;
    const int32_t* starts;
    float scale_log2;
    float* lse;
    Plan* plan;
    int32_t* before;  // units before each sequence
    Boundary* boundaries;
    float* parts;
    int32_t main_blocks; // of the main kernel
    bool join_segments;  // the join's blocks stand for segments, not boundaries
};

// Asynchronous copies of N bytes into shared memory, `OFF` bytes past `from`;
// the second form writes zeros where `on` is false.
template <int N, int OFF>
__device__ __forceinline__ void copy_async(uint32_t to, const void* from) {
    if (N == 16)
        asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1 + %2], 16;" ::"r"(to), "l"(from), "n"(OFF) : "memory");
    else
        asm volatile("cp.async.ca.shared.global [%0], [%1 + %2], %3;" ::"r"(to), "l"(from), "n"(OFF), "n"(N) : "memory");
}
template <int N>
__device__ __forceinline__ void copy_async_if(uint32_t to, const void* from, bool on) {
    const int bytes = on ? N : 0;
    if (N == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
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

// 2^x, log2 x; results below 2^-126 are zero.
__device__ __forceinline__ float exp2_fast(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float log2_fast(float x) {
    float r;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
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

// int8 codes as fp16, exactly: the byte with its sign bit turned, u = code + 128,
// under the exponent of 1024 is 1024 + u; less 1152 it is the code.
__device__ __forceinline__ uint32_t int8_half2(uint32_t x) {
    const uint32_t c = 0x64806480u;
    const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&x), *reinterpret_cast<const __half2*>(&c));
    return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t e4m3_half2(uint32_t x) {
    const __half2_raw r = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)x, __NV_E4M3);
    return (uint32_t)r.x | (uint32_t)r.y << 16;
}

// Four codes of a word as two fp16 pairs.
template <int KIND>
__device__ __forceinline__ void codes_of_word(uint32_t x, uint32_t& lo, uint32_t& hi) {
    if (KIND == CHM_INT8) {
        x ^= 0x80808080u;
        lo = int8_half2(__byte_perm(x, 0x64646464u, 0x4140));
        hi = int8_half2(__byte_perm(x, 0x64646464u, 0x4342));
    } else {
        lo = e4m3_half2(x & 0xFFFFu);
        hi = e4m3_half2(x >> 16);
    }
}

// Byte e of two words as an fp16 pair.
template <int KIND>
__device__ __forceinline__ uint32_t codes_of_pair(uint32_t x, uint32_t y, int e) {
    if (KIND == CHM_INT8) return int8_half2((__byte_perm(x, y, (uint32_t)(e | (4 + e) << 8)) & 0x00FF00FFu) ^ 0x64806480u);
    return e4m3_half2(__byte_perm(x, y, (uint32_t)(e | (4 + e) << 4)) & 0xFFFFu);
}

// ---- how the work is split ------------------------------------------------------
//
// A segment is one sequence's tokens for one block of query heads that share a
// key head.  It is cut into units of a tile (a step of all warps), and the units
// of all segments, in the order (sequence, block, unit), are dealt out evenly:
// with `per` = ceil(units / blocks), block c takes [c * per, (c + 1) * per).  So
// the lengths, which only the device knows, do not matter to the balance, a long
// sequence spreads over the device and short ones stay whole.  A segment counts
// kStartUnits more, before its first tile, for what its start and end cost: blocks
// with many short segments were the last to finish (64 sequences up to 4,096
// tokens: 110 us with none, 104 / 102 / 101 / 102 with 1 / 2 / 3 / 5; 128 long
// documents e4m3: 43.5, 39.3 / 39.3 / 39.5 / 41.3).  A segment that
// crosses from one block to the next leaves a part (unnormalised output,
// reference exponent, sum) per block in the workspace, and attention_join_kernel
// adds them in order.

constexpr int kStartUnits = 2;

struct Range {
    int first, end;  // positions attended to
    int units;
    bool bad;  // the length does not fit the table
};

__device__ __forceinline__ Range range_of(const AttArgs& a, int start, int len) {
    Range r;
    r.first = min(max(start, 0), a.capacity);
    r.end = max(len, 0);  // so that end - first stays within 32 bits
    r.bad = r.end > a.capacity;
    if (r.bad) r.end = 0;
    r.units = a.start_units + max(1, (int)a.by_unit.div((uint32_t)(max(r.end - r.first, 0) + a.unit_tokens - 1)));
    return r;
}
__device__ __forceinline__ Range sequence_range(const AttArgs& a, int b) {
    return range_of(a, a.starts ? a.starts[b] : 0, a.lens[b]);
}

// Where the units of up to 128 sequences lie, worked out by a warp: lane i has
// those of sequences i, 32 + i, 64 + i and 96 + i, and the sums up to them.
struct Deal {
    int n[4], sum[4];
    int total;

    __device__ __forceinline__ Deal(const AttArgs& a, int segs, int lane) {
        int len[4], start[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int i = k * 32 + lane;
            len[k] = i < a.batch ? a.lens[i] : 0;
            start[k] = a.starts && i < a.batch ? a.starts[i] : 0;
        }
#pragma unroll
        for (int k = 0; k < 4; ++k)
            sum[k] = n[k] = k * 32 + lane < a.batch ? range_of(a, start[k], len[k]).units * segs : 0;
#pragma unroll
        for (int x = 1; x < 32; x <<= 1)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int y = __shfl_up_sync(0xffffffffu, sum[k], x);
                if (lane >= x) sum[k] += y;
            }
        total = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int all = __shfl_sync(0xffffffffu, sum[k], 31);
            sum[k] += total;
            total += all;
        }
    }
    // The sequence that holds unit u < total, and the units before it.
    __device__ __forceinline__ int find(int u, int& before) const {
        int b = 0;
#pragma unroll
        for (int k = 3; k >= 0; --k) {
            const uint32_t past = __ballot_sync(0xffffffffu, sum[k] > u);
            if (past) {
                const int at = __ffs(past) - 1;
                b = k * 32 + at;
                before = __shfl_sync(0xffffffffu, sum[k] - n[k], at);
            }
        }
        return b;
    }
    __device__ __forceinline__ int before(int b) const {
        int y = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int x = __shfl_sync(0xffffffffu, sum[k] - n[k], b & 31);
            if (b >> 5 == k) y = x;
        }
        return y;
    }
};

// Rows of parts: DMAX output elements, then the reference and the sum.  Block c
// has slot 2c for the segment that holds its first unit and 2c + 1 for its last.
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

// Element d of the output over tokens [first, end) where the products came out NaN beside
// a finite sum of probabilities.  An infinite value makes them so: the low term of its weight
// may be 0 or negative, and a weight that 16 bits do not hold is 0.  The probability itself is
// positive, so with infinities of one sign among the values the element is that infinity; with
// both, or a NaN, it is NaN.  64 sequences up to 4,096 tokens of bf16 with an infinite
// channel take 390 us in place of 95, with all values NaN 109.
template <int KIND>
__device__ __noinline__ float infinite_element(const AttArgs& a, int b, int head, int first, int end, int d) {
    constexpr bool kWide = KIND == CHM_FP16 || KIND == CHM_BF16;
    constexpr int kAhead = 8;  // values on their way: loads without branches, past the end the last token's
    const int32_t* const table = a.tables + b * a.table_stride;
    const char* const values = static_cast<const char*>(a.c.v) + (head * a.c.head_stride + d) * (kWide ? 2 : 1);
    bool plus = false, minus = false;
    for (int j = first; j < end; j += kAhead) {
        uint16_t x[kAhead];
        float by[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            const uint32_t at = (uint32_t)min(j + k, end - 1), turn = a.by_page.div(at);
            const uint32_t within = at - turn * (uint32_t)a.c.page_size;
            // (inside the cache, or the sum were NaN; a table that changes meanwhile stays inside too)
            const int64_t page = min(max((int64_t)table[turn], (int64_t)0), a.c.num_pages - 1);
            const char* from = values + (page * a.c.page_stride + within * a.c.token_stride) * (kWide ? 2 : 1);
            x[k] = kWide ? *reinterpret_cast<const uint16_t*>(from) : *reinterpret_cast<const uint8_t*>(from);
            by[k] = kWide ? 1.0f : a.c.v_scale[(page * a.c.heads + head) * a.c.page_size + within];
        }
        bool nan = false;
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            float y;
            if (KIND == CHM_BF16)
                y = __uint_as_float((uint32_t)x[k] << 16);
            else if (KIND == CHM_FP16)
                y = __half2float(__ushort_as_half(x[k]));
            else if (KIND == CHM_INT8)
                y = by[k] * (float)(int8_t)x[k];
            else
                y = by[k] * __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)x[k], __NV_E4M3)));
            plus = plus || y == INFINITY;
            minus = minus || y == -INFINITY;
            nan = nan || y != y;
        }
        if (nan || (plus && minus)) break;
        if (j + kAhead >= end && plus != minus) return plus ? INFINITY : -INFINITY;
    }
    return __int_as_float(0x7FC00000);
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
    // A warp's ring: kSlots copies of a step's keys or of its values, in turn, are on their
    // way or in use.  8 KB per warp stream at 6.7 TB/s with 12 warps per SM; 12 KB cost the
    // long sequence 66 us in place of 64.
    static constexpr int kSlot = kTok * DMAX * kBytes;
    static constexpr int kSlots = (kResident == 3 ? 8192 : kResident == 2 ? 16384 : 32768) / kSlot;
    static_assert(kSlots % 2 == 0, "keys take even slots, values odd ones");
    static constexpr int kScaleSlots = kSlots / 2 + 1;  // steps whose scales are on their way or in use
    // shared memory: q as operand registers, two factors of its rows, rings, scales, the warps' parts
    static constexpr int kQ = NT * (DMAX / 32) * 512 + kHeads * 8;
    static constexpr int kRing = kAttWarps * kSlots * kSlot;
    static constexpr int kScales = kWide ? 0 : kAttWarps * kScaleSlots * 2 * kTok * 4;
    static constexpr int kRow = DMAX + 4;
    static constexpr int kOut = kAttWarps * kHeads * (kRow + 2) * 4;
    static constexpr int kShared = kQ + kRing + kScales + kOut;
    static_assert(kResident * (kShared + 1024) <= 227 * 1024, "the resident blocks' shared memory");
};

template <int DMAX, int KIND, int NT>
__global__ void __launch_bounds__(kAttThreads, Shape<DMAX, KIND, NT>::kResident)
    paged_attention_kernel(const __grid_constant__ AttArgs a) {
    using S = Shape<DMAX, KIND, NT>;
    constexpr bool kWide = S::kWide;
    constexpr bool kHalf = KIND != CHM_BF16;  // fp16 products; 8-bit codes are fp16 numbers
    constexpr int kBytes = S::kBytes, kU = S::kU, kTok = S::kTok, kTile = S::kTile, kHeads = S::kHeads;
    constexpr int kSlots = S::kSlots, kSlot = S::kSlot, kScaleSlots = S::kScaleSlots;
    constexpr int kKC = DMAX * kBytes / 64;         // 16-byte runs of a key per thread
    constexpr int kRuns = DMAX / 32;                // operand runs of q
    constexpr int kE = DMAX / 8;                    // value elements per thread and token
    constexpr int kVB = kE * kBytes < 16 ? 8 : 16;  // bytes of a run of a value
    constexpr int kVC = kE * kBytes / kVB;          // runs of a value per thread
    constexpr int kVT = kVB == 16 ? 4 : 8;          // tokens per copy of values
    constexpr int kM = kE / 2;                      // 16-row blocks of the output
    constexpr int kRow = S::kRow;
    // Weights are exp2(score - ref), where ref trails the largest exponent (score, plus the
    // log2 of the value's scale) by kLead and moves only when one passes it by kRoom.  fp16
    // weights (their high part) so stay below 2^15, and the smallest step of their low part,
    // 2^-24, is 2^-35 of the largest: many small ones are not lost.  bf16 has fp32's range.
    constexpr float kLead = kHalf ? 11.0f : 0.0f, kRoom = kHalf ? 15.0f : 8.0f;
    // A value's scale counts as at least 2^-80: without values exp2(score - ref) is then below
    // 2^95 and its sum over 2^30 tokens finite, and the smallest scale that is written, 2^-105,
    // still has weights that fp16 holds.  So does an infinite one: its products are infinite
    // whatever the reference, which would take the others' probabilities with it.  References
    // may so differ by 200 beside sums of up to 2^95: a sum takes the factor between two of
    // them, which may be below 2^-126, in two halves.
    constexpr float kLeast = -80.0f;
    extern __shared__ __align__(16) uint8_t smem[];
    uint4(*s_q)[kRuns][32] = reinterpret_cast<uint4(*)[kRuns][32]>(smem);
    float* const s_f = reinterpret_cast<float*>(smem + NT * kRuns * 512);
    uint8_t* const s_parts = smem + S::kQ + S::kRing + S::kScales;
    float(*s_o)[kHeads][kRow] = reinterpret_cast<float(*)[kHeads][kRow]>(s_parts);
    float(*s_m)[kHeads] = reinterpret_cast<float(*)[kHeads]>(s_parts + kAttWarps * kHeads * kRow * 4);
    float(*s_l)[kHeads] = s_m + kAttWarps;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int dim = a.c.dim;
    // This warp's ring: the keys of a step, its values, the next step's keys and so on, a slot
    // each.  Keys: a lane's own 16 bytes in a row of 512.  Values: eight lanes copy 128
    // bytes of a token (a row of four tokens, or of eight 64-byte ones, is one copy of 512);
    // by lane they would go to memory a sector at a time, which halves the bandwidth (3.7
    // against 6.7 TB/s).  Lane (g, t) then finds its run in line t, 16-byte places turned by
    // 2t so that neither side has bank conflicts.
    const uint8_t* const ring = smem + S::kQ + warp * (kSlots * kSlot);
    const float* const scales = reinterpret_cast<const float*>(smem + S::kQ + S::kRing) + warp * (kScaleSlots * 2 * kTok);
    const uint32_t ring_k = (uint32_t)__cvta_generic_to_shared(ring) + lane * 16;
    const int vt = kVB == 16 ? lane >> 3 : lane >> 2;  // the token a lane copies, of kVT
    const int vc = kVB == 16 ? lane & 7 : lane & 3;    // and its 16 bytes of it
    const uint32_t ring_v = (uint32_t)__cvta_generic_to_shared(ring) +
                            (kVB == 16 ? vt * 8 + (vc ^ (2 * vt)) : (vt >> 1) * 8 + (((vt & 1) * 4 + vc) ^ (vt & 6))) * 16;
    // where lane (g, t) reads the values of its first and second token of eight
    const int run_v0 = kVB == 16 ? (t * 8 + (g ^ (2 * t))) * 16 : t * 128 + ((g >> 1) ^ (2 * t)) * 16 + (g & 1) * 8;
    const int run_v1 = kVB == 16 ? run_v0 : t * 128 + ((4 + (g >> 1)) ^ (2 * t)) * 16 + (g & 1) * 8;
    const uint32_t scales_at = (uint32_t)__cvta_generic_to_shared(scales) + lane * 4;
    const char* const kbase = static_cast<const char*>(a.c.k) + t * 16;
    const char* const vbase = static_cast<const char*>(a.c.v) + vc * 16;
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

    struct Piece {
        int b, h0, nh;  // its sequence, first query head, query heads
        int head;       // key head
        int first, end;
        bool whole, bad;
    } now{}, next{};
    // Token `pos` of the range, one per lane: its page, then its place and scales.
    auto page_of = [&](const Piece& it, int pos) {
        return pos < it.end ? a.tables[it.b * a.table_stride + a.by_page.div((uint32_t)pos)] : 0;
    };
    uint32_t at = kNowhere;  // of this lane's token of the newest step, in 16 bytes
    bool full = false;       // all the step's tokens are there, in their whole width
    auto place = [&](Piece& it, int pos, int page, int slot) {
        at = kNowhere;
        int64_t scale = 0;
        if (pos < it.end) {
            if (page < 0 || page >= a.c.num_pages) {
                it.bad = true;
            } else {
                const uint32_t within = (uint32_t)pos - a.by_page.div((uint32_t)pos) * (uint32_t)a.c.page_size;
                at = (uint32_t)page * a.page16 + (uint32_t)it.head * a.head16 + within * a.token16;
                if (!kWide) scale = ((int64_t)page * a.c.heads + it.head) * a.c.page_size + within;
            }
        }
        if (!kWide && lane < kTok) {
            copy_async_if<4>(scales_at + slot * (2 * kTok * 4), a.c.k_scale + scale, at != kNowhere);
            copy_async_if<4>(scales_at + slot * (2 * kTok * 4) + kTok * 4, a.c.v_scale + scale, at != kNowhere);
        }
        full = __all_sync(0xffffffffu, at != kNowhere) && dim == DMAX;
    };
    auto copy_keys = [&](int slot) {
        const uint32_t to = ring_k + slot * kSlot;
#pragma unroll
        for (int i = 0; i < 2 * kU; ++i) {
            const uint32_t x = __shfl_sync(0xffffffffu, at, i * 8 + g);
            const char* p = kbase + (uint64_t)x * 16;
            if (full) {
                copy_async<16, 0>(to + i * kKC * 512, p);
                if (kKC > 1) copy_async<16, 64>(to + (i * kKC + 1) * 512, p);
                if (kKC > 2) copy_async<16, 128>(to + (i * kKC + 2) * 512, p);
                if (kKC > 3) copy_async<16, 192>(to + (i * kKC + 3) * 512, p);
                if (kKC > 4) {
                    copy_async<16, 256>(to + (i * kKC + 4) * 512, p);
                    copy_async<16, 320>(to + (i * kKC + 5) * 512, p);
                    copy_async<16, 384>(to + (i * kKC + 6) * 512, p);
                    copy_async<16, 448>(to + (i * kKC + 7) * 512, p);
                }
            } else {
#pragma unroll
                for (int c = 0; c < kKC; ++c) {
                    const bool on = x != kNowhere && c * 64 + t * 16 < dim * kBytes;
                    copy_async_if<16>(to + (i * kKC + c) * 512, on ? p + c * 64 : kbase, on);
                }
            }
        }
    };
    auto copy_values = [&](int slot) {
        const uint32_t to = ring_v + slot * kSlot;
#pragma unroll
        for (int i = 0; i < kTok / kVT; ++i) {
            // 128-byte runs: tokens 2t or 2t + 1 of eight, as lanes t need them together
            const int src = kVB == 16 ? (i >> 1) * 8 + 2 * vt + (i & 1) : i * 8 + vt;
            const uint32_t x = __shfl_sync(0xffffffffu, at, src);
            const char* p = vbase + (uint64_t)x * 16;
            if (full) {
                copy_async<16, 0>(to + i * kVC * 512, p);
                if (kVC > 1) copy_async<16, 128>(to + (i * kVC + 1) * 512, p);
                if (kVC > 2) {
                    copy_async<16, 256>(to + (i * kVC + 2) * 512, p);
                    copy_async<16, 384>(to + (i * kVC + 3) * 512, p);
                }
            } else {
#pragma unroll
                for (int c = 0; c < kVC; ++c) {
                    const bool on = x != kNowhere && c * 128 + vc * 16 < dim * kBytes;
                    copy_async_if<16>(to + (i * kVC + c) * 512, on ? p + c * 128 : vbase, on);
                }
            }
        }
    };

    int pos = 0;           // this lane's token of the newest step
    int next_page = 0;     // and its page, of the step after
    int newest = 0;        // the newest step's first token
    bool live = false;     // whether that step has tokens
    int scale_in = 0;      // where the newest step's scales go
    // The next step of `it`: where its tokens are, its scales and keys on their way.
    auto next_keys = [&](Piece& it, int slot) {
        pos += kTile, newest += kTile;
        live = newest < it.end;
        scale_in = scale_in + 1 == kScaleSlots ? 0 : scale_in + 1;
        if (live) {
            const int page = next_page;
            next_page = page_of(it, pos + kTile);
            place(it, pos, page, scale_in);
            copy_keys(slot);
        }
        copies_commit();
    };
    auto its_values = [&](int slot) {
        if (live) copy_values(slot);
        copies_commit();
    };

    // ---- segment by segment; the next one's first copies are on their way while this one's
    // parts are joined
    for (int piece = -1;; ++piece) {
        float o[NT][kM][4] = {};
        float m[NT][2], l[NT][2];  // references and sums of this lane's columns
#pragma unroll
        for (int n = 0; n < NT; ++n) m[n][0] = m[n][1] = -INFINITY, l[n][0] = l[n][1] = 0.0f;
        if (piece >= 0) {
            float qf[NT][2], qg[NT][2];
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    qf[n][e] = kWide ? a.scale_log2 : s_f[n * 8 + 2 * t + e];
                    qg[n][e] = kWide ? 1.0f : s_f[kHeads + n * 8 + 2 * t + e];
                }

            // The copies run kSlots / 2 steps ahead: keys that have been read make room for those
            // of the step that far ahead, its values for its values.
            int slot = 0, scale_out = 0;
            for (int base = now.first + warp * kTok; base < now.end; base += kTile) {
                const uint8_t* const keys = ring + slot * kSlot + lane * 16;
                copies_wait<kSlots - 1>();
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
                                if (kWide)
                                    p0[e] = w0[e], p1[e] = w1[e];
                                else if (e % 2 == 0) {
                                    codes_of_word<KIND>(w0[j * 2 + e / 2], p0[e], p0[e + 1]);
                                    codes_of_word<KIND>(w1[j * 2 + e / 2], p1[e], p1[e + 1]);
                                }
                            }
                            const int run = kWide ? c : c * 2 + j;
#pragma unroll
                            for (int n = 0; n < NT; ++n) {
                                const uint4 bq = s_q[n][run][lane];
                                mma<kHalf>(sc[n][i], p0[0], p1[0], p0[1], p1[1], bq.x, bq.y);
                                mma<kHalf>(sc[n][i], p0[2], p1[2], p0[3], p1[3], bq.z, bq.w);
                            }
                        }
                    }
                // ---- scaled: by half of q's factor, the key's scale, the other half, so that neither
                // passes fp32's range where the score does not; tokens past the end get weight zero
#pragma unroll
                for (int i = 0; i < kU; ++i)
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int e = 0; e < 4; ++e) sc[n][i][e] *= qf[n][e & 1];
                float vs[kU][2], lv[kU][2];
                if (!kWide) {
#pragma unroll
                    for (int i = 0; i < kU; ++i)
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const int src = i * 16 + h * 8 + g;
                            const float ks = scales[scale_out * 2 * kTok + src];
                            vs[i][h] = scales[scale_out * 2 * kTok + kTok + src];
                            const float x = log2_fast(fabsf(vs[i][h]));
                            lv[i][h] = x < INFINITY ? fmaxf(x, kLeast) : kLeast;
#pragma unroll
                            for (int n = 0; n < NT; ++n)
#pragma unroll
                                for (int e = 0; e < 2; ++e) sc[n][i][h * 2 + e] = sc[n][i][h * 2 + e] * ks * qg[n][e];
                        }
                    scale_out = scale_out + 1 == kScaleSlots ? 0 : scale_out + 1;
                }
                bool above = false;
                if (base + kTok > now.end) {
#pragma unroll
                    for (int i = 0; i < kU; ++i)
#pragma unroll
                        for (int h = 0; h < 2; ++h)
                            if (base + i * 16 + h * 8 + g >= now.end) {
#pragma unroll
                                for (int n = 0; n < NT; ++n) sc[n][i][h * 2] = sc[n][i][h * 2 + 1] = -INFINITY;
                            }
                }
#pragma unroll
                for (int i = 0; i < kU; ++i)
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            above = above || (kWide ? sc[n][i][e] : sc[n][i][e] + lv[i][e >> 1]) > m[n][e & 1] + kRoom;
                __syncwarp();  // all lanes have read the keys and scales
                next_keys(now, slot);
                slot = slot + 1 == kSlots ? 0 : slot + 1;
                // ---- the reference follows the largest exponent
                if (__any_sync(0xffffffffu, above)) {
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            float top = m[n][e] + kLead;
#pragma unroll
                            for (int i = 0; i < kU; ++i)
#pragma unroll
                                for (int h = 0; h < 2; ++h)
                                    top = fmaxf(top, kWide ? sc[n][i][h * 2 + e] : sc[n][i][h * 2 + e] + lv[i][h]);
#pragma unroll
                            for (int x = 4; x < 32; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
                            top -= kLead;
                            const float half = top > m[n][e] ? exp2_fast(0.5f * (m[n][e] - top)) : 1.0f, f = half * half;
                            m[n][e] = fmaxf(top, m[n][e]);
                            l[n][e] = l[n][e] * half * half;
#pragma unroll
                            for (int i = 0; i < kM; ++i) o[n][i][e] *= f, o[n][i][2 + e] *= f;
                        }
                }
                // ---- weights as the operand of the second product, in 16-bit terms: bf16 three, for
                // fp32's 24 bits (two, 16 bits, rounded 3 times as many outputs the other way than the
                // plain form; 64 sequences up to 4,096 tokens take 94.1 us with three, 93.9 with two, 16
                // heads per key head 35.6 and 34.9), fp16 two, 22 bits down to 2^-36 of the largest
                uint32_t ph[NT][kU][2], pl[NT][kU][2], pt[NT][kU][2];
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const float m0 = m[n][0] == -INFINITY ? 0.0f : m[n][0], m1 = m[n][1] == -INFINITY ? 0.0f : m[n][1];
#pragma unroll
                    for (int i = 0; i < kU; ++i)
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            float p0 = exp2_fast(sc[n][i][h * 2] - m0), p1 = exp2_fast(sc[n][i][h * 2 + 1] - m1);
                            l[n][0] += p0, l[n][1] += p1;
                            if (!kWide) p0 *= vs[i][h], p1 *= vs[i][h];
                            const uint32_t hi = pack16<kHalf>(p0, p1);
                            const float2 y = unpack16<kHalf>(hi);
                            ph[n][i][h] = transpose8(hi);
                            const uint32_t lo = pack16<kHalf>(p0 - y.x, p1 - y.y);
                            pl[n][i][h] = transpose8(lo);
                            if (!kHalf) {
                                const float2 z = unpack16<kHalf>(lo);
                                pt[n][i][h] = transpose8(pack16<kHalf>(p0 - y.x - z.x, p1 - y.y - z.y));
                            }
                        }
                }
                // ---- values
                const uint8_t* const values = ring + slot * kSlot;
                copies_wait<kSlots - 1>();
                __syncwarp();
#pragma unroll
                for (int i = 0; i < kU; ++i) {
                    uint32_t vr[4][kVC * kVB / 4];
#pragma unroll
                    for (int h = 0; h < 4; ++h)
#pragma unroll
                        for (int c = 0; c < kVC; ++c) {
                            if (kVB == 16) {
                                const uint4 w = *reinterpret_cast<const uint4*>(values + ((i * 4 + h) * kVC + c) * 512 + run_v0);
                                vr[h][c * 4] = w.x, vr[h][c * 4 + 1] = w.y, vr[h][c * 4 + 2] = w.z, vr[h][c * 4 + 3] = w.w;
                            } else {
                                const uint2 w = *reinterpret_cast<const uint2*>(values + (i * 2 + (h >> 1)) * 512 +
                                                                                (h & 1 ? run_v1 : run_v0));
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
                            if (kWide)
                                f[h] = __byte_perm(v0[x / 2], v1[x / 2], (x & 1) ? 0x7632 : 0x5410);
                            else
                                f[h] = codes_of_pair<KIND>(v0[x / 4], v1[x / 4], x & 3);
                        }
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            mma<kHalf>(o[n][j], f[0], f[1], f[2], f[3], ph[n][i][0], ph[n][i][1]);
                            mma<kHalf>(o[n][j], f[0], f[1], f[2], f[3], pl[n][i][0], pl[n][i][1]);
                            if (!kHalf) mma<kHalf>(o[n][j], f[0], f[1], f[2], f[3], pt[n][i][0], pt[n][i][1]);
                        }
                    }
                }
                __syncwarp();
                its_values(slot);
                slot = slot + 1 == kSlots ? 0 : slot + 1;
            }
            copies_wait<0>();
        }
        // ---- the next segment
        const bool last = u >= u1;
        if (!last) {
            if (u == before + r.units * segs) {
                before = u;
                r = sequence_range(a, ++b);
            }
            const int in_seq = u - before;
            const int seg = in_seq / r.units;
            const int unit0 = in_seq - seg * r.units;
            const int unit1 = min(r.units, unit0 + (u1 - u));
            if (threadIdx.x == 0) {
                if (piece < 0) a.boundaries[blockIdx.x] = Boundary{b, seg, u - unit0, r.units};
                if (in_seq == 0) a.before[b] = before;
            }
            next.b = b;
            next.head = seg / a.blocks;
            next.h0 = next.head * a.group + (seg - next.head * a.blocks) * kHeads;
            next.nh = min(kHeads, (next.head + 1) * a.group - next.h0);
            next.first = r.first + max(unit0 - a.start_units, 0) * a.unit_tokens;
            next.end = unit1 == r.units ? r.end : r.first + max(unit1 - a.start_units, 0) * a.unit_tokens;
            next.whole = unit1 - unit0 == r.units;
            next.bad = r.bad;
            u += unit1 - unit0;
        }
        // ---- this segment's warps' parts to shared memory
        if (piece >= 0) {
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
        }
        if (!last) {
            newest = next.first + warp * kTok - kTile;
            pos = newest + lane % kTok;
            next_page = page_of(next, pos + kTile);
            scale_in = -1;
#pragma unroll
            for (int n = 0; n < kSlots; ++n) {
                if (n % 2 == 0)
                    next_keys(next, n);
                else
                    its_values(n);
            }
        }
        if (piece >= 0) {
            const bool bad = __syncthreads_or(now.bad);
            for (int hh = warp; hh < now.nh; hh += kAttWarps) {
                float top = -INFINITY, sum = 0.0f, f[kAttWarps];
#pragma unroll
                for (int w = 0; w < kAttWarps; ++w) top = fmaxf(top, s_m[w][hh]);
#pragma unroll
                for (int w = 0; w < kAttWarps; ++w) {
                    const float half = s_m[w][hh] == -INFINITY ? 0.0f : exp2_fast(0.5f * (s_m[w][hh] - top));
                    f[w] = half * half;
                    sum += s_l[w][hh] * half * half;
                }
                if (bad) sum = __int_as_float(0x7FC00000);
                float* part = part_row<DMAX>(a.parts, 2 * blockIdx.x + (piece > 0), kHeads, hh);
                float acc[DMAX / 32];
                bool odd = false;
#pragma unroll
                for (int v = 0; v < DMAX / 32; ++v) {
                    acc[v] = 0.0f;
#pragma unroll
                    for (int w = 0; w < kAttWarps; ++w) acc[v] += f[w] * s_o[w][hh][v * 32 + lane];
                    odd = odd || acc[v] != acc[v];
                }
                if (__any_sync(0xffffffffu, odd) && sum == sum) {
#pragma unroll
                    for (int v = 0; v < DMAX / 32; ++v)
                        if (acc[v] != acc[v] && v * 32 + lane < dim)
                            acc[v] = infinite_element<KIND>(a, now.b, now.head, now.first, now.end, v * 32 + lane);
                }
#pragma unroll
                for (int v = 0; v < DMAX / 32; ++v) {
                    const int d = v * 32 + lane;
                    if (d >= dim) continue;
                    if (now.whole)
                        store_row(a, now.b, now.h0 + hh, d, sum == 0.0f ? 0.0f : bad ? sum : acc[v] / sum);
                    else
                        part[d] = acc[v];
                }
                if (lane == 0) {
                    if (!now.whole)
                        part[DMAX] = top, part[DMAX + 1] = sum;
                    else if (a.lse)
                        a.lse[(int64_t)now.b * a.q_heads + now.h0 + hh] = sum == 0.0f ? -INFINITY : (top + log2f(sum)) * kLn2;
                }
            }
        }
        if (last) break;
        // q: lane (g, t) of a run holds the 8 elements that its key runs meet.  For an 8-bit
        // cache a row is brought by a power of two to a largest element below 2^14, so that
        // fp16 holds it (exactly but for elements below 2^-28 of the largest).
        {
            constexpr int kLanes = DMAX / 8;  // lanes per row
            const int d0 = (lane % kLanes) * 8;
#pragma unroll
            for (int h = 0; h < kHeads; h += kAttWarps * (32 / kLanes)) {
                const int hh = h + warp * (32 / kLanes) + lane / kLanes;
                float x[8] = {};
                const int64_t qa = next.b * a.q_b + (next.h0 + hh) * a.q_h + d0;
                if (hh < next.nh && d0 < dim) {
                    uint32_t w[4];
                    if (a.q_wide) {
                        const uint4 y = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.q) + qa);
                        w[0] = y.x, w[1] = y.y, w[2] = y.z, w[3] = y.w;
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            w[e] = static_cast<const uint16_t*>(a.q)[qa + 2 * e] |
                                   (uint32_t) static_cast<const uint16_t*>(a.q)[qa + 2 * e + 1] << 16;
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float2 y = a.q_type == CHM_FP16 ? unpack16<true>(w[e]) : unpack16<false>(w[e]);
                        x[2 * e] = y.x, x[2 * e + 1] = y.y;
                    }
                }
                float f = a.scale_log2, f2 = 1.0f;
                if (!kWide) {
                    float top = 0.0f;
#pragma unroll
                    for (int e = 0; e < 8; ++e) top = isfinite(x[e]) ? fmaxf(top, fabsf(x[e])) : top;
#pragma unroll
                    for (int y = kLanes / 2; y > 0; y >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, y));
                    const int y = top > 0.0f ? 13 - ilogbf(top) : 0;  // -114 to 146: in two halves
                    const float up = exp2f((float)(y / 2)), up2 = exp2f((float)(y - y / 2));
#pragma unroll
                    for (int e = 0; e < 8; ++e) x[e] = x[e] * up * up2;
                    f *= exp2f((float)-(y / 2));
                    f2 = exp2f((float)-(y - y / 2));
                }
                uint32_t w[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) w[e] = pack16<kHalf>(x[2 * e], x[2 * e + 1]);
                const int run = kWide ? d0 / 32 : d0 / 64 * 2 + (d0 / 8) % 2;
                const int tt = kWide ? d0 / 8 % 4 : d0 / 16 % 4;
                if (hh < kHeads) {
                    s_q[hh / 8][run][hh % 8 * 4 + tt] = make_uint4(w[0], w[1], w[2], w[3]);
                    if (d0 == 0) s_f[hh] = f, s_f[kHeads + hh] = f2;
                }
            }
        }
        __syncthreads();
        now = next;
    }
}

// Block (x, y): some heads, a row of threads each, of a segment that several blocks had,
// from its parts in the order of the blocks.  x stands for a segment or, where there are
// fewer, for the boundary before block x + 1 (then the segment's first boundary does it).
// Which parts there are follows from the lengths: up to 128 sequences that is worked out
// while the main kernel's last blocks run (one sequence of 600 tokens 7.7 us against 8.8,
// 16 of them 12.7 against 13.1), else read from what the main kernel left.
constexpr int kJoinThreads = 256;

template <int DMAX, int NT>
__global__ void __launch_bounds__(kJoinThreads) attention_join_kernel(const AttArgs a) {
    constexpr int kHeads = 8 * NT;
    constexpr int kV = DMAX / 32;   // elements per lane
    constexpr int kAhead = kV > 4 ? 4 : 8;  // parts on their way per warp
    __shared__ float s_acc[kJoinThreads / 32][DMAX];
    __shared__ float s_sum[kJoinThreads / 32], s_top[kJoinThreads / 32];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;  // of this row of threads
    const int segs = a.c.heads * a.blocks;
    const bool early = a.batch <= 128;
    Plan plan{1, 0};
    Boundary s{0, 0, 0, 1};
    bool any = true;
    if (early) {
        const Deal deal(a, segs, lane);
        plan = Plan{(deal.total + a.main_blocks - 1) / a.main_blocks, deal.total};
        if (a.join_segments) {
            s.seq = blockIdx.x / segs;
            s.first = deal.before(s.seq);
        } else {
            const int64_t u = (blockIdx.x + 1) * (int64_t)plan.per;
            any = u < plan.total;
            if (any) s.seq = deal.find((int)u, s.first);
        }
        s.units = sequence_range(a, s.seq).units;
        s.seg = a.join_segments ? blockIdx.x - s.seq * segs : ((int)(blockIdx.x + 1) * plan.per - s.first) / s.units;
        s.first += s.seg * s.units;
    }
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (!early) {
        plan = *a.plan;
        if (a.join_segments) {
            s.seq = blockIdx.x / segs;
            s.seg = blockIdx.x - s.seq * segs;
            s.units = sequence_range(a, s.seq).units;
            s.first = a.before[s.seq] + s.seg * s.units;
        } else {
            any = (blockIdx.x + 1) * (int64_t)plan.per < plan.total;
            if (any) s = a.boundaries[blockIdx.x + 1];
        }
    }
    if (!any) return;
    const int c0 = s.first / plan.per, c1 = (s.first + s.units - 1) / plan.per;
    // a boundary: one inside the segment, and its first
    if (c0 == c1 || (!a.join_segments && c0 != (int)blockIdx.x)) return;
    const int head = s.seg / a.blocks;
    const int h0 = head * a.group + (s.seg - head * a.blocks) * kHeads;
    const int hh = blockIdx.y * blockDim.y + threadIdx.y;
    if (hh >= kHeads || h0 + hh >= (head + 1) * a.group) return;
    const int odd = c0 * plan.per != s.first;  // whether the first part is its block's second slot
    auto part = [&](int i) { return part_row<DMAX>(a.parts, 2 * i + (i == c0 ? odd : 0), kHeads, hh); };
    // each warp takes every warps-th part, kAhead of them on their way at once
    float top = -INFINITY, sum = 0.0f, acc[kV] = {};
    for (int i = c0 + warp; i <= c1; i += warps * kAhead) {
        float x[kAhead][kV], m[kAhead], l[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            const bool on = i + j * warps <= c1;
            const float* p = part(on ? i + j * warps : i);
            m[j] = on ? p[DMAX] : -INFINITY;
            l[j] = on ? p[DMAX + 1] : 0.0f;
#pragma unroll
            for (int v = 0; v < kV; ++v) x[j][v] = on ? p[v * 32 + lane] : 0.0f;
        }
        float now = top;
#pragma unroll
        for (int j = 0; j < kAhead; ++j) now = fmaxf(now, m[j]);
        const float half = top == now ? 1.0f : exp2_fast(0.5f * (top - now)), f = half * half;
        top = now;
        sum = sum * half * half;
#pragma unroll
        for (int v = 0; v < kV; ++v) acc[v] *= f;
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            const float half = m[j] == -INFINITY ? 0.0f : exp2_fast(0.5f * (m[j] - top)), w = half * half;
            sum += l[j] * half * half;
#pragma unroll
            for (int v = 0; v < kV; ++v) acc[v] += x[j][v] * w;
        }
    }
    if (warps > 1) {
#pragma unroll
        for (int v = 0; v < kV; ++v) s_acc[warp][v * 32 + lane] = acc[v];
        if (lane == 0) s_sum[warp] = sum, s_top[warp] = top;
        __syncthreads();
        if (warp > 0) return;
        float all = top;
        for (int w = 1; w < warps; ++w) all = fmaxf(all, s_top[w]);
        sum = 0.0f;
#pragma unroll
        for (int v = 0; v < kV; ++v) acc[v] = 0.0f;
        for (int w = 0; w < warps; ++w) {
            const float half = s_top[w] == -INFINITY ? 0.0f : exp2_fast(0.5f * (s_top[w] - all)), f = half * half;
            sum += s_sum[w] * half * half;
#pragma unroll
            for (int v = 0; v < kV; ++v) acc[v] += f * s_acc[w][v * 32 + lane];
        }
        top = all;
    }
#pragma unroll
    for (int v = 0; v < kV; ++v) {
        const int d = v * 32 + lane;
        if (d >= a.c.dim) continue;
        if (acc[v] != acc[v] && sum == sum) {  // an infinite part, its factor 0 maybe: as infinite_element
            bool plus = false, minus = false, none = false;
            for (int i = c0; i <= c1; ++i) {
                const float y = part(i)[d];
                plus = plus || y == INFINITY;
                minus = minus || y == -INFINITY;
                none = none || y != y;
            }
            if (!none && plus != minus) acc[v] = plus ? INFINITY : -INFINITY;
        }
        store_row(a, s.seq, h0 + hh, d, sum == 0.0f ? 0.0f : sum != sum ? sum : acc[v] / sum);
    }
    if (lane == 0 && a.lse)
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
    int segs;         // segments per sequence
    int unit_tokens;  // tokens per unit
    int start_units;
    int64_t units;    // at most
    bool joins;       // whether a segment can be split
};

template <int DMAX, int KIND, int NT>
struct Launch {
    using S = Shape<DMAX, KIND, NT>;

    static Layout layout(const AttArgs& a) {
        Layout y;
        y.segs = a.c.heads * ((a.group + S::kHeads - 1) / S::kHeads);
        // Up to 4 tiles, or 8 where there are segments enough for the device, a segment stays
        // whole: a second launch and the parts cost more than the balance gains.  Device time
        // of 1 / 16 / 64 / 128 sequences (32 query heads on 8 of 128, bf16): 2 tiles 6.2 / 6.3 /
        // 14 / 20 us whole, 7.0 / 10.4 / 16 / 23 split; 4 tiles 7.7 / 8.1 / 19 / 31 and 7.1 / 10.3 /
        // 18 / 33; 8 tiles 11.0 / 11.2 / 32 / 52 and 7.6 / 12.4 / 31 / 52, of 32 and 48 sequences
        // 13.6 and 17.4 whole, 16.5 and 21.8 split.  So one sequence of 4 tiles loses 0.6 us by
        // the rule and 64 lose 1; 16 and 128 gain 2.  Whole segments are one unit whatever their
        // length, and a block takes a whole number of them: past a round of the resident blocks
        // (444 segments, 55 sequences of 8 key heads) the time steps up, 48 sequences of 256 tokens
        // 11.8 us, 56 of them 17.8.
        const int whole = ((int64_t)a.batch * y.segs >= 128 ? 8 : 4) * S::kTile;
        y.unit_tokens = a.capacity <= whole ? whole : S::kTile;
        y.joins = a.capacity > whole;
        y.start_units = y.joins ? kStartUnits : 0;  // else a segment is one unit
        y.units = (int64_t)a.batch * y.segs * (y.start_units + std::max(1, (a.capacity + y.unit_tokens - 1) / y.unit_tokens));
        y.blocks = (int)std::min<int64_t>(y.units, (int64_t)sm_count() * S::kResident);
        return y;
    }
    struct Counter {
        Sizer s;
        template <typename T>
        void* take(size_t n) {
            s.take<T>(n);
            return nullptr;
        }
    };
    template <typename A>
    static void carve(A& arena, const Layout& y, AttArgs* a, int batch) {
        auto plan = arena.template take<Plan>(1);
        auto before = arena.template take<int32_t>(batch);
        auto bounds = arena.template take<Boundary>(y.blocks);
        auto parts = arena.template take<float>(y.joins ? (size_t)2 * y.blocks * S::kHeads * (DMAX + 4) : 0);
        if (a) {
            a->plan = (Plan*)plan;
            a->before = (int32_t*)before;
            a->boundaries = (Boundary*)bounds;
            a->parts = (float*)parts;
        }
    }
    // Units are counted in 32 bits.
    static bool too_much(const Layout& y) {
        if (y.units <= INT32_MAX - (1 << 20)) return false;
        set_last_message("paged_attention: too much work for one call");
        return true;
    }
    static size_t workspace(const AttArgs& a) {
        const Layout y = layout(a);
        if (too_much(y)) return 0;
        Counter c;
        carve(c, y, nullptr, a.batch);
        return c.s.off;
    }
    static chm_status run(AttArgs a, void* ws, size_t ws_bytes, cudaStream_t st) {
        const Layout y = layout(a);
        if (too_much(y)) return CHM_ERR_INVALID;
        Arena arena(ws, ws_bytes);
        carve(arena, y, &a, a.batch);
        if (arena.overflow) return CHM_ERR_CAPACITY;
        if (a.c.num_pages == 0) {  // copies of nothing still name an address
            a.c.k = a.c.v = ws;
            a.c.k_scale = a.c.v_scale = (float*)ws;
        }
        a.blocks = (a.group + S::kHeads - 1) / S::kHeads;
        a.unit_tokens = y.unit_tokens;
        a.start_units = y.start_units;
        a.by_unit = FastDiv((uint32_t)y.unit_tokens);
        const int64_t segments = (int64_t)a.batch * y.segs;
        a.join_segments = segments < y.blocks;
        a.main_blocks = y.blocks;
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
        // A warp has 8 parts on their way: warps enough for eight rounds of the most a segment
        // can have, and a row of one warp for each head where one is enough.
        const int64_t most = std::min<int64_t>(y.blocks, y.units / segments);
        const int warps = (int)std::min<int64_t>(kJoinThreads / 32, (most + 63) / 64), heads = std::min(S::kHeads, a.group);
        const int rows = warps == 1 ? std::min(heads, 8) : 1;
        cfg.gridDim = dim3((unsigned)(a.join_segments ? segments : y.blocks - 1), (unsigned)((heads + rows - 1) / rows));
        cfg.blockDim = dim3((unsigned)(32 * warps), (unsigned)rows);
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
// read the cache once: 32 sequences of 4,096 tokens, 2 key heads of 128, bf16, 16 /
// 9 query heads each 36 / 34 us, by single blocks 38 / 37; 128 sequences of 128
// tokens 13 against 17 (one of 8,192 tokens 14 against 12).  At dim 256 the
// registers hold one block.
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

// Whether 32 bits of 16 bytes reach every vector of the cache.
static bool spans_64gb(const chm_kv_cache& c) {
    const unsigned __int128 n = (unsigned __int128)(uint64_t)std::max<int64_t>(c.num_pages - 1, 0) * (uint64_t)c.page_stride +
                                (unsigned __int128)(uint64_t)(c.heads - 1) * (uint64_t)c.head_stride +
                                (unsigned __int128)(uint64_t)(c.page_size - 1) * (uint64_t)c.token_stride;
    return n * type_bytes(c.type) / 16 < kNowhere;
}

static chm_status refuse_attention(const char* why) {
    char msg[160];
    snprintf(msg, sizeof(msg), "paged_attention: %s", why);
    set_last_message(msg);
    return CHM_ERR_INVALID;
}

// What is wrong with a call's sizes, or NULL.
static const char* bad_sizes(const chm_kv_cache& c, int64_t batch, int32_t q_heads, int32_t table_width) {
    if (batch < 0 || table_width < 0) return "negative size";
    if (q_heads < 1 || q_heads % c.heads) return "query heads must be a multiple of the cache's heads";
    if (batch > 65535) return "at most 65535 sequences";
    if ((int64_t)table_width * c.page_size > (1 << 30)) return "a table spans at most 2^30 tokens";
    return nullptr;
}

}  // namespace chm

extern "C" size_t chm_paged_attention_workspace_bytes(const chm_kv_cache* cache, int64_t batch, int32_t q_heads,
                                                      int32_t table_width) {
    using namespace chm;
    if (check_cache(cache, "paged_attention") != CHM_OK) return 0;
    if (const char* why = bad_sizes(*cache, batch, q_heads, table_width)) {
        refuse_attention(why);
        return 0;
    }
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
    if (const char* why = bad_sizes(*cache, batch, q->heads, table_width)) return refuse_attention(why);
    if (q->heads != out->heads) return refuse_attention("query heads of q and out must agree, a multiple of the cache's heads");
    if (batch == 0) return CHM_OK;
    if (!q->data || !out->data || !lens || (table_width > 0 && !tables)) return refuse_attention("null pointer");
    if (!spans_64gb(*cache)) return refuse_attention("keys and values span at most 64 GB each");
    AttArgs a{};
    a.c = *cache;
    const int run = 16 / type_bytes(cache->type);
    a.page16 = (uint32_t)(cache->page_stride / run);
    a.head16 = (uint32_t)(cache->head_stride / run);
    a.token16 = (uint32_t)(cache->token_stride / run);
    a.q = q->data;
    a.q_wide = aligned16(q->data) && q->batch_stride % 8 == 0 && q->head_stride % 8 == 0;
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
    return with_launch(a, [&](auto l) { return l.run(a, workspace, workspace_bytes, st); });
}
