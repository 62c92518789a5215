// Rotary positions (chm_rotary) and their frequencies.
//
// A pair (x0, x1) of a vector at position p turns by a = p * f_i:
//   y0 = s (x0 cos a - x1 sin a),  y1 = s (x0 sin a + x1 cos a);
// the gradient turns back by the same angle.  The angle is reduced to turns in
// 64 bits (p * f_i / 2 pi less its nearest integer), since 32 bits lose
// whole turns at far positions; what is left takes 32-bit sine and cosine.
//
// HBM bounds it: each vector is read and written once.  One B200: a 16,384-token
// prompt (32 + 8 heads of 128, bf16) 55 us on the device and 59 as a call for 336 MB, 5.7
// to 6.1 TB/s; the gradient of 6,141 tokens of 24 heads of 96 (64 of them turned,
// neighbours, fp16) 13 to 15 us for 57 MB: 1.7 rounds of 6,141 warps, whose first bytes
// and angles take some 4 us, and 6 of 8 lanes at work.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "vectors.cuh"

namespace chm {

struct HeadsView {
    const void* in;
    void* out;
    int64_t in_b, in_t, in_h, out_b, out_t, out_h;
};

struct RotaryArgs {
    HeadsView set[2];
    int32_t heads0, heads;  // heads of set 0, of both
    int32_t dim, rot;
    const void* positions;
    int32_t position_bytes;
    int64_t pos_b, pos_t;
    const double* freqs;
    float scale;
    float sign;            // -1: turn back
    int32_t rows, tokens;  // tokens in all, and per batch row
    int32_t parts;         // warps that share a row
    int32_t chunks, turn_chunks;  // items per vector, and those that turn
    int32_t lanes;         // lanes across a vector: a power of two
    FastDiv by_tokens, by_parts;
};

// V elements of a run, as pairs of floats.
template <typename T, int V>
struct Run {
    Pack<T, V> p;
    __device__ __forceinline__ void floats(float (&f)[V]) const {
#pragma unroll
        for (int i = 0; i < V; ++i) f[i] = to_float<T>(p.v[i]);
    }
    __device__ __forceinline__ void set(const float* f) {
        if (V > 1 && sizeof(T) == 2) {
#pragma unroll
            for (int i = 0; i < V; i += 2) two(f[i], f[(i + 1) % V], i);
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) p.v[i] = from_float<T>(f[i]);
        }
    }
    __device__ __forceinline__ void two(float a, float b, int i);
};
template <typename T, int V>
__device__ __forceinline__ void Run<T, V>::two(float a, float b, int i) {
    if constexpr (std::is_same<T, __half>::value)
        *reinterpret_cast<__half2*>(&p.v[i]) = __floats2half2_rn(a, b);
    else if constexpr (std::is_same<T, __nv_bfloat16>::value)
        *reinterpret_cast<__nv_bfloat162*>(&p.v[i]) = __floats2bfloat162_rn(a, b);
}

// Items a lane has on their way, two 16-byte loads each, with 6 blocks of 128 per SM.  A
// 16,384-token prompt of 32 + 8 heads of 128 (bf16) / the gradient of 6,141 tokens of 24 heads
// of 96 (fp16, neighbours): 57.7 / 14.6 us; 2: 57.7 / 14.7; 4 with 5 blocks: 57.0 / 16.7, 5 with
// 4: 55.7 / 17.0.
constexpr int kRotaryAhead = 3;

// A warp (or `parts` of them) has a row: a token's vectors of all heads.  Its lanes stand in
// rows of a.lanes across a vector, so that a lane keeps its place in the vector and the sine
// and cosine of its V pairs from head to head.  An item is V pairs: two runs of V elements
// that one lane loads, turns and stores (so in place is safe).  The first items are loaded
// before the row's angles are worked out, two or so per lane, into the warp's own table:
// the V pairs of an item as groups of 16 bytes, each group's items in a row.
template <typename T, int V, bool INTER>
__global__ void __launch_bounds__(128, 6) rotary_kernel(const RotaryArgs a) {
    using R = Run<T, V>;
    extern __shared__ __align__(16) float2 s_turn[];  // (cos, sin) * scale
    constexpr int kGroup = V > 1 ? 2 : 1;
    const int half = a.rot / 2, lane = threadIdx.x & 31;
    float2* const table = s_turn + (threadIdx.x >> 5) * half;
    const uint32_t warp = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);  // may pass 2^31 where parts is 1
    if (a.by_parts.div(warp) >= (uint32_t)a.rows) return;
    const int row = (int)a.by_parts.div(warp), part = (int)warp - row * a.parts;
    const int b = (int)a.by_tokens.div((uint32_t)row), t = row - b * a.tokens;
    const T* in[2];
    T* out[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        in[i] = static_cast<const T*>(a.set[i].in) + b * a.set[i].in_b + t * a.set[i].in_t;
        out[i] = static_cast<T*>(a.set[i].out) + b * a.set[i].out_b + t * a.set[i].out_t;
    }
    const int per_step = 32 / a.lanes;            // heads a warp has at a time
    const int step = per_step * a.parts;
    const int h0 = part * per_step + lane / a.lanes;
    bool ready = false;
    for (int c = lane % a.lanes; c - lane % a.lanes < a.chunks; c += a.lanes) {
        // this lane's runs of a vector
        const bool turns = c < a.turn_chunks, on = c < a.chunks;
        const int o0 = turns ? (INTER ? 2 * c * V : c * V) : a.rot + 2 * (c - a.turn_chunks) * V;
        const int o1 = turns && !INTER ? half + o0 : o0 + V;
        const bool second = o1 < a.dim;
        float2 w[V];
        for (int h = h0; h - lane / a.lanes < a.heads; h += step * kRotaryAhead) {
            R x[kRotaryAhead], y[kRotaryAhead];
            T* to[kRotaryAhead];
#pragma unroll
            for (int u = 0; u < kRotaryAhead; ++u) {
                const int hu = h + u * step;
                to[u] = nullptr;
                if (on && hu < a.heads) {
                    const bool k = hu >= a.heads0;
                    const int hh = k ? hu - a.heads0 : hu;
                    const T* from = (k ? in[1] : in[0]) + hh * (k ? a.set[1].in_h : a.set[0].in_h) + o0;
                    to[u] = (k ? out[1] : out[0]) + hh * (k ? a.set[1].out_h : a.set[0].out_h) + o0;
                    if (!turns && from == to[u]) {
                        to[u] = nullptr;  // passed on in place
                    } else {
                        x[u].p = *reinterpret_cast<const Pack<T, V>*>(from);
                        if (second) y[u].p = *reinterpret_cast<const Pack<T, V>*>(from + (o1 - o0));
                    }
                }
            }
            if (!ready) {
                const int64_t at = b * a.pos_b + t * a.pos_t;
                const double pos = a.position_bytes == 8 ? (double)static_cast<const int64_t*>(a.positions)[at]
                                                         : (double)static_cast<const int32_t*>(a.positions)[at];
                for (int i = lane; i < half; i += 32) {
                    const double turn = pos * (a.freqs[i] * 0.15915494309189533577);  // 1 / (2 pi)
                    float sine, cosine;
                    sincospif(2.0f * (float)(turn - rint(turn)), &sine, &cosine);
                    const int item = i / V, j = i % V;
                    table[(j / kGroup * a.turn_chunks + item) * kGroup + j % kGroup] =
                        make_float2(a.scale * cosine, a.sign * a.scale * sine);
                }
                __syncwarp();
                ready = true;
            }
            if (h == h0 && turns) {
#pragma unroll
                for (int j = 0; j < V; j += kGroup) {
                    const float2* p = table + (j / kGroup * a.turn_chunks + c) * kGroup;
                    if (kGroup == 2) {
                        const float4 f = *reinterpret_cast<const float4*>(p);
                        w[j] = make_float2(f.x, f.y), w[(j + 1) % V] = make_float2(f.z, f.w);
                    } else {
                        w[j] = *p;
                    }
                }
            }
#pragma unroll
            for (int u = 0; u < kRotaryAhead; ++u) {
                if (!to[u]) continue;
                if (turns) {
                    float e[2][V];
                    x[u].floats(e[0]);
                    y[u].floats(e[1]);
#pragma unroll
                    for (int j = 0; j < V; ++j) {
                        float &p = INTER ? e[2 * j / V][2 * j % V] : e[0][j];
                        float &q = INTER ? e[(2 * j + 1) / V][(2 * j + 1) % V] : e[1][j];
                        const float p0 = p;
                        p = p0 * w[j].x - q * w[j].y;
                        q = p0 * w[j].y + q * w[j].x;
                    }
                    x[u].set(e[0]);
                    y[u].set(e[1]);
                }
                *reinterpret_cast<Pack<T, V>*>(to[u]) = x[u].p;
                if (second) *reinterpret_cast<Pack<T, V>*>(to[u] + (o1 - o0)) = y[u].p;
            }
        }
    }
}

template <typename T, int V>
static void launch_rotary(const RotaryArgs& a, bool inter, cudaStream_t st) {
    const int half = a.rot / 2;
    const int warps = half <= 512 ? 4 : 1;  // each with its table in shared memory
    const int64_t all = (int64_t)a.rows * a.parts;
    const unsigned blocks = (unsigned)((all + warps - 1) / warps);
    const size_t smem = (size_t)warps * half * sizeof(float2);
    if (inter)
        rotary_kernel<T, V, true><<<blocks, warps * 32, smem, st>>>(a);
    else
        rotary_kernel<T, V, false><<<blocks, warps * 32, smem, st>>>(a);
}

// 16-byte runs fit when every vector starts on one and pairs and the rest come
// in whole runs; otherwise elements move one by one (4,096 tokens of 32 + 8 heads of
// 128 in bf16: 14 us, and 46 one by one).
template <typename T>
static void dispatch_rotary(RotaryArgs a, bool inter, cudaStream_t st) {
    constexpr int kV = 16 / sizeof(T);
    int n = a.heads > a.heads0 ? 2 : 1;
    bool wide = (a.rot / 2) % kV == 0 && a.dim % kV == 0;
    for (int i = 0; i < n; ++i) {
        const HeadsView& v = a.set[i];
        wide = wide && aligned16(v.in) && aligned16(v.out);
        for (int64_t s : {v.in_b, v.in_t, v.in_h, v.out_b, v.out_t, v.out_h}) wide = wide && s % kV == 0;
    }
    const int V = wide ? kV : 1;
    a.turn_chunks = a.rot / 2 / V;
    a.chunks = a.turn_chunks + (a.dim - a.rot + 2 * V - 1) / (2 * V);
    a.lanes = 1;
    while (a.lanes < 32 && a.lanes < a.chunks) a.lanes *= 2;
    // Few rows: several warps share one, as long as each has heads of its own.  512 / 1,024 /
    // 2,048 rows of 32 + 8 heads of 128 (bf16, device time): up to 2,048 warps 3.9 / 5.3 / 7.9 us,
    // 1,024 4.4 / 6.2 / 7.9, 4,096 5.4 / 6.1 / 8.6.
    const int steps = (a.heads + 32 / a.lanes - 1) / (32 / a.lanes);
    a.parts = 1;
    while (a.parts * 2 <= steps && (int64_t)a.rows * a.parts < 2048) a.parts *= 2;
    a.by_tokens = FastDiv((uint32_t)a.tokens);
    a.by_parts = FastDiv((uint32_t)a.parts);
    if (wide)
        launch_rotary<T, kV>(a, inter, st);
    else
        launch_rotary<T, 1>(a, inter, st);
}

static chm_status refuse(const char* why) {
    set_last_message(why);
    return CHM_ERR_INVALID;
}

}  // namespace chm

extern "C" chm_status chm_rotary_frequencies(int32_t rot_dim, double base, int32_t kind, double factor,
                                             double original_len, double slow, double fast, double* freqs) {
    if (!freqs || rot_dim < 2 || rot_dim % 2) return chm::refuse("rotary_frequencies: rot_dim must be even and freqs given");
    if (!(base > 1) || !std::isfinite(base)) return chm::refuse("rotary_frequencies: base must be above 1");
    if (kind < CHM_ROTARY_PLAIN || kind > CHM_ROTARY_PARTS) return chm::refuse("rotary_frequencies: unknown kind");
    if (kind != CHM_ROTARY_PLAIN && (!(factor >= 1) || !std::isfinite(factor)))
        return chm::refuse("rotary_frequencies: factor must be at least 1");
    if (kind == CHM_ROTARY_PARTS &&
        (!(original_len > 0) || !std::isfinite(original_len) || !(slow > 0) || !(fast > slow) || !std::isfinite(fast)))
        return chm::refuse("rotary_frequencies: parts need original_len > 0 and 0 < slow < fast");
    const double two_pi = 6.283185307179586476925;
    // one pair (rot_dim 2) has frequency 1 whatever the base
    if (kind == CHM_ROTARY_BASE && rot_dim > 2) base *= std::pow(factor, (double)rot_dim / (rot_dim - 2));
    for (int i = 0; i < rot_dim / 2; ++i) {
        double f = std::pow(base, -2.0 * i / rot_dim);
        if (kind == CHM_ROTARY_LINEAR) f /= factor;
        if (kind == CHM_ROTARY_PARTS) {
            double keep = (original_len * f / two_pi - slow) / (fast - slow);
            keep = keep < 0 ? 0 : keep > 1 ? 1 : keep;
            f = f * keep + f / factor * (1 - keep);
        }
        freqs[i] = f;
    }
    return CHM_OK;
}

extern "C" chm_status chm_rotary(const chm_heads* in, const chm_heads* out, int32_t n, int32_t type, int64_t batch,
                                 int64_t tokens, int32_t dim, int32_t rot_dim, const void* positions,
                                 int32_t position_bytes, int64_t position_batch_stride,
                                 int64_t position_token_stride, const double* freqs, float scale, int32_t flags,
                                 void* stream) {
    using namespace chm;
    if (!in || !out || n < 1 || n > 2) return refuse("rotary: one or two sets of heads");
    if (!valid_float_type(type)) return refuse("rotary: fp32, fp16 or bf16 vectors");
    if (batch < 0 || tokens < 0) return refuse("rotary: negative size");
    if (dim < 2 || dim > 4096 || rot_dim < 2 || rot_dim > dim || rot_dim % 2)
        return refuse("rotary: rot_dim must be even and at most dim, dim at most 4096");
    if (position_bytes != 4 && position_bytes != 8) return refuse("rotary: positions are int32 or int64");
    if (flags & ~(CHM_ROTARY_INTERLEAVED | CHM_ROTARY_INVERSE)) return refuse("rotary: unknown flag");
    RotaryArgs a{};
    for (int i = 0; i < n; ++i) {
        if (in[i].heads < 0 || in[i].heads != out[i].heads || in[i].heads > (1 << 14))
            return refuse("rotary: heads of in and out must agree, at most 16384");
        a.set[i] = HeadsView{in[i].data,         out[i].data,         in[i].batch_stride,  in[i].token_stride,
                             in[i].head_stride,  out[i].batch_stride, out[i].token_stride, out[i].head_stride};
        a.heads += in[i].heads;
        if (i == 0) a.heads0 = a.heads;
    }
    if (batch == 0 || tokens == 0 || a.heads == 0) return CHM_OK;
    for (int i = 0; i < n; ++i)
        if (in[i].heads && (!in[i].data || !out[i].data)) return refuse("rotary: null vectors");
    if (!positions || !freqs) return refuse("rotary: null positions or frequencies");
    if (batch > INT32_MAX / tokens) return refuse("rotary: more than 2^31 - 1 tokens");
    a.dim = dim;
    a.rot = rot_dim;
    a.positions = positions;
    a.position_bytes = position_bytes;
    a.pos_b = position_batch_stride;
    a.pos_t = position_token_stride;
    a.freqs = freqs;
    a.scale = scale;
    a.sign = flags & CHM_ROTARY_INVERSE ? -1.0f : 1.0f;
    a.rows = (int32_t)(batch * tokens);
    a.tokens = (int32_t)tokens;
    const bool inter = flags & CHM_ROTARY_INTERLEAVED;
    cudaStream_t st = (cudaStream_t)stream;
    if (type == CHM_FP32)
        dispatch_rotary<float>(a, inter, st);
    else if (type == CHM_FP16)
        dispatch_rotary<__half>(a, inter, st);
    else
        dispatch_rotary<__nv_bfloat16>(a, inter, st);
    return launch_status("rotary_kernel");
}
