// Rotary positions (chm_rotary) and their frequencies.
//
// A pair (x0, x1) of a vector at position p turns by a = p * f_i:
//   y0 = s (x0 cos a - x1 sin a),  y1 = s (x0 sin a + x1 cos a);
// the gradient turns back by the same angle.  The angle is reduced to turns in
// 64 bits (p * f_i / 2 pi less its nearest integer), since 32 bits lose
// whole turns at far positions; what is left takes 32-bit sine and cosine.
#include <cmath>

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
    float sign;  // -1: turn back
    int64_t rows;
    int64_t tokens;  // per batch row
    int32_t chunks;  // items per vector
    int32_t turn_chunks;
    FastDiv by_chunks;
};

constexpr int kRotaryThreads = 256;

// Block: one row (a token of a batch row), all heads.  An item is V pairs of a vector: two runs
// of V elements that one thread loads, turns and stores (so in place is safe).
template <typename T, int V, bool INTER>
__global__ void __launch_bounds__(kRotaryThreads) rotary_kernel(const RotaryArgs a) {
    extern __shared__ float2 s_turn[];  // (cos, sin) * scale of the row's pairs
    const int64_t row = blockIdx.x;
    const int64_t b = row / a.tokens, t = row - b * a.tokens;
    const int64_t at = b * a.pos_b + t * a.pos_t;
    const double pos = a.position_bytes == 8 ? (double)static_cast<const int64_t*>(a.positions)[at]
                                             : (double)static_cast<const int32_t*>(a.positions)[at];
    for (int i = threadIdx.x; i < a.rot / 2; i += kRotaryThreads) {
        const double turns = pos * (a.freqs[i] * 0.15915494309189533577);  // 1 / (2 pi)
        float s, c;
        sincospif(2.0f * (float)(turns - rint(turns)), &s, &c);
        s_turn[i] = make_float2(a.scale * c, a.sign * a.scale * s);
    }
    __syncthreads();
    const int half = a.rot / 2;
    const int items = a.heads * a.chunks;
    for (int it = threadIdx.x; it < items; it += kRotaryThreads) {
        const int h = (int)a.by_chunks.div((uint32_t)it);
        const int c = it - h * a.chunks;
        const bool second = h >= a.heads0;
        const HeadsView& v = a.set[second];
        const int hh = second ? h - a.heads0 : h;
        const T* in = static_cast<const T*>(v.in) + b * v.in_b + t * v.in_t + hh * v.in_h;
        T* out = static_cast<T*>(v.out) + b * v.out_b + t * v.out_t + hh * v.out_h;
        using P = Pack<T, V>;
        if (c < a.turn_chunks) {
            const int o0 = INTER ? 2 * c * V : c * V;
            const int o1 = INTER ? o0 + V : half + o0;
            P x = *reinterpret_cast<const P*>(in + o0), y = *reinterpret_cast<const P*>(in + o1);
            if (INTER) {
                // x, y: 2V neighbours, V pairs
                float e[2 * V];
#pragma unroll
                for (int j = 0; j < V; ++j) e[j] = to_float<T>(x.v[j]), e[V + j] = to_float<T>(y.v[j]);
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float2 w = s_turn[c * V + j];
                    const float p = e[2 * j], q = e[2 * j + 1];
                    e[2 * j] = p * w.x - q * w.y;
                    e[2 * j + 1] = p * w.y + q * w.x;
                }
#pragma unroll
                for (int j = 0; j < V; ++j) x.v[j] = from_float<T>(e[j]), y.v[j] = from_float<T>(e[V + j]);
            } else {
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float2 w = s_turn[c * V + j];
                    const float p = to_float<T>(x.v[j]), q = to_float<T>(y.v[j]);
                    x.v[j] = from_float<T>(p * w.x - q * w.y);
                    y.v[j] = from_float<T>(p * w.y + q * w.x);
                }
            }
            *reinterpret_cast<P*>(out + o0) = x;
            *reinterpret_cast<P*>(out + o1) = y;
        } else if (in != out) {
            const int o0 = a.rot + 2 * (c - a.turn_chunks) * V;
            *reinterpret_cast<P*>(out + o0) = *reinterpret_cast<const P*>(in + o0);
            if (o0 + V < a.dim) *reinterpret_cast<P*>(out + o0 + V) = *reinterpret_cast<const P*>(in + o0 + V);
        }
    }
}

template <typename T, int V>
static void launch_rotary(const RotaryArgs& a, bool inter, cudaStream_t st) {
    const size_t smem = (size_t)(a.rot / 2) * sizeof(float2);
    if (inter)
        rotary_kernel<T, V, true><<<(unsigned)a.rows, kRotaryThreads, smem, st>>>(a);
    else
        rotary_kernel<T, V, false><<<(unsigned)a.rows, kRotaryThreads, smem, st>>>(a);
}

// 16-byte runs fit when every vector starts on one and pairs and the rest come
// in whole runs; otherwise elements move one by one.
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
    a.by_chunks = FastDiv((uint32_t)a.chunks);
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
        if (in[i].heads < 0 || in[i].heads != out[i].heads || in[i].heads > (1 << 16))
            return refuse("rotary: heads of in and out must agree, at most 65536");
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
    a.rows = batch * tokens;
    a.tokens = tokens;
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
