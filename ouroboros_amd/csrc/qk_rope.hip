// qk_rope.hip - RMS norm of every query and key head and the rotary position of
// its first dims, in one pass (rmsnorm_head and rope_partial_neox,
// qwen35.rs:96-106,1246-1248, for a caller's rows).
//
// Of a head x of d values: x_i g_i / sqrt(mean x^2 + eps), then each pair (a, b)
// of the first n_rot becomes (a cos t - b sin t, b cos t + a sin t), t the
// token's position on the pair's axis times its frequency.
#include "common.hpp"

#include <cmath>

namespace ouro {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxHalf = 128;   // pairs of a head
constexpr int kMaxTokens = 8;   // tokens of a workgroup
constexpr int64_t kManyRows = 2048;  // from here a workgroup takes several tokens, below a part of one's heads

struct RopeArgs {
    const void *in[2];  // queries, keys
    void *out[2];
    const float *gain[2];
    const int32_t *pos, *axis;
    const float *freq;
    int64_t in_stride[2], head_stride[2], out_stride[2], out_head[2];
    int64_t rows;
    int32_t heads, q_heads;  // query and key heads together, and the queries'
    int32_t d, half, axes, adjacent;
    float eps, inv_d;
    int32_t token_shift, pad;  // tokens of a workgroup
};
// passed by value to kernels: the host and device passes must lay it out alike
static_assert(sizeof(RopeArgs) == 184, "RopeArgs: kernel argument layout");

// cos and sin of pos * freq.  In quarter turns u = pos freq 2/pi: its nearest
// integer says which of cos, sin, -cos, -sin, and of what is left, within 1/2,
// the series of x = (pi/2) rest, |x| <= pi/4, leave out less than 2^-29.  The
// product is exact but for one rounding in 64 bits and 2/pi is held in two
// parts, so that far positions keep their angle; single precision begins at x.
__device__ __forceinline__ float2 cos_sin(int pos, float freq) {
    constexpr double kHi = 0x1.45f306dc9c883p-1, kLo = -0x1.6b01ec5417056p-55;  // 2/pi = kHi + kLo
    const double angle = static_cast<double>(pos) * static_cast<double>(freq);
    const double u = angle * kHi, k = rint(u);
    const double rest = (u - k) + (fma(angle, kHi, -u) + angle * kLo);
    const float x = static_cast<float>(rest * 1.5707963267948966), y = x * x;
    const float s = x * (1.0f + y * (-1.0f / 6 + y * (1.0f / 120 + y * (-1.0f / 5040 + y * (1.0f / 362880)))));
    const float c = 1.0f + y * (-0.5f + y * (1.0f / 24 + y * (-1.0f / 720 + y * (1.0f / 40320 + y * (-1.0f / 3628800)))));
    const int q = static_cast<int>(static_cast<int64_t>(k) & 3);
    const float cc = q & 1 ? s : c, ss = q & 1 ? c : s;
    return make_float2(q == 1 || q == 2 ? -cc : cc, q >= 2 ? -ss : ss);
}

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));

// E adjacent values of a row (E sizeof(T) = 4, 8 or 16 bytes, aligned to that).
template <int E, typename T>
__device__ __forceinline__ void load(const T *p, float (&x)[E]) {
    uint32_t w[E * sizeof(T) / 4];
    if constexpr (sizeof(w) == 16) {
        const u32x4_t v = *reinterpret_cast<const u32x4_t *>(p);
        w[0] = v[0], w[1] = v[1], w[2] = v[2], w[3] = v[3];
    } else if constexpr (sizeof(w) == 8) {
        const u32x2_t v = *reinterpret_cast<const u32x2_t *>(p);
        w[0] = v[0], w[1] = v[1];
    } else {
        w[0] = *reinterpret_cast<const uint32_t *>(p);
    }
#pragma unroll
    for (int e = 0; e < E; ++e) {
        if constexpr (sizeof(T) == 4)
            x[e] = __uint_as_float(w[e]);
        else
            x[e] = __uint_as_float(e & 1 ? w[e / 2] & 0xffff0000u : w[e / 2] << 16);
    }
}
template <int E, typename T>
__device__ __forceinline__ void store(T *p, const float (&x)[E]) {
    uint32_t w[E * sizeof(T) / 4];
#pragma unroll
    for (int e = 0; e < E; ++e) {
        if constexpr (sizeof(T) == 4)
            w[e] = __float_as_uint(x[e]);
        else if (e & 1)
            w[e / 2] = f32_to_bf16_bits(x[e - 1]) | static_cast<uint32_t>(f32_to_bf16_bits(x[e])) << 16;
    }
    if constexpr (sizeof(w) == 16)
        *reinterpret_cast<u32x4_t *>(p) = u32x4_t{w[0], w[1], w[2], w[3]};
    else if constexpr (sizeof(w) == 8)
        *reinterpret_cast<u32x2_t *>(p) = u32x2_t{w[0], w[1]};
    else
        *reinterpret_cast<uint32_t *>(p) = w[0];
}

// A head is taken by G lanes, each with two pieces of E values whose pairs are
// its own, so that nothing but the sum of squares crosses lanes: for pairs
// (i, i + half) piece p of either half, for adjacent pairs pieces 2p and 2p + 1;
// past n_rot two pieces in a row.  The angles of a token are the same for all of
// its heads: they are made once, by as many threads as it has pairs, and a group
// of G lanes stays with one token and keeps its angles and gains in registers.
//
// 16385 rows of 20 heads of 128, bf16: 47 us, 3.6 TB/s where a copy has 5, bound by
// the five wavefronts a SIMD that two pieces of eight values a lane leave (95 registers;
// eight tokens a workgroup; with the angles and a division a head made anew 73).  64 fp32
// rows take 4.5 us, a part of a token's heads a workgroup: three dependent loads and the
// angles.
template <typename T, int E, int G>
__global__ __launch_bounds__(kThreads) void qk_rope_kernel(RopeArgs a) {
    __shared__ __attribute__((aligned(16))) float cs[kMaxTokens][kMaxHalf], sn[kMaxTokens][kMaxHalf];
    const int tid = threadIdx.x, p = tid % G;
    const int64_t t0 = static_cast<int64_t>(blockIdx.x) << a.token_shift;
    const int tokens = static_cast<int>(min(int64_t{1} << a.token_shift, a.rows - t0));
    const int groups = (kThreads / G) >> a.token_shift;  // of a token
    const int t = tid / G / groups, step = groups * static_cast<int>(gridDim.y);
    int h = tid / G % groups + groups * static_cast<int>(blockIdx.y);
    const int rot = a.half / E;  // pieces of a half
    int i0, i1;
    if (p < rot) {
        i0 = a.adjacent ? 2 * p * E : p * E;
        i1 = a.adjacent ? i0 + E : i0 + a.half;
    } else {
        i0 = 2 * a.half + 2 * (p - rot) * E;
        i1 = i0 + E;
    }
    const bool in0 = i0 < a.d, in1 = i1 < a.d;
    const int heads = t < tokens ? a.heads : 0;
    float x[E], y[E], u[E], v[E];
    auto fetch = [&](int head, float (&f)[E], float (&s)[E]) {
        const int key = head >= a.q_heads;
        const T *row = static_cast<const T *>(a.in[key]) + (t0 + t) * a.in_stride[key] +
                       static_cast<int64_t>(key ? head - a.q_heads : head) * a.head_stride[key];
#pragma unroll
        for (int e = 0; e < E; ++e) f[e] = s[e] = 0.f;
        if (in0) load<E>(row + i0, f);
        if (in1) load<E>(row + i1, s);
    };
    if (h < heads) fetch(h, x, y);  // on its way while the angles are made
    for (int i = tid; i < tokens * a.half; i += kThreads) {
        const int at = i / a.half, j = i % a.half;
        const int axis = a.axis ? max(0, min(a.axis[j], a.axes - 1)) : 0;
        const float2 r = cos_sin(a.pos[axis * a.rows + t0 + at], a.freq[j]);
        cs[at][j] = r.x;
        sn[at][j] = r.y;
    }
    __syncthreads();
    float c[E], s[E], g0[E], g1[E];
    if (p < rot)
#pragma unroll
        for (int e = 0; e < E; ++e) c[e] = cs[t][p * E + e], s[e] = sn[t][p * E + e];
    int have = -1;  // whose gains are held
    for (; h < heads; h += step) {
        const int key = h >= a.q_heads;
        if (h + step < heads) fetch(h + step, u, v);
        if (a.gain[key]) {
            if (have != key) {
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    g0[e] = in0 ? a.gain[key][i0 + e] : 0.f;
                    g1[e] = in1 ? a.gain[key][i1 + e] : 0.f;
                }
                have = key;
            }
            float ss = 0.f;
#pragma unroll
            for (int e = 0; e < E; ++e) ss += x[e] * x[e] + y[e] * y[e];
#pragma unroll
            for (int off = G / 2; off >= 1; off >>= 1) ss += __shfl_xor(ss, off, G);
            const float inv = rsqrtf(ss * a.inv_d + a.eps);
#pragma unroll
            for (int e = 0; e < E; ++e) x[e] = x[e] * inv * g0[e], y[e] = y[e] * inv * g1[e];
        }
        if (p < rot) {
            if (a.adjacent) {
#pragma unroll
                for (int e = 0; e < E; e += 2) {
                    const float x0 = x[e], x1 = x[e + 1], y0 = y[e], y1 = y[e + 1];
                    x[e] = x0 * c[e / 2] - x1 * s[e / 2], x[e + 1] = x1 * c[e / 2] + x0 * s[e / 2];
                    y[e] = y0 * c[(E + e) / 2] - y1 * s[(E + e) / 2], y[e + 1] = y1 * c[(E + e) / 2] + y0 * s[(E + e) / 2];
                }
            } else {
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const float x0 = x[e], y0 = y[e];
                    x[e] = x0 * c[e] - y0 * s[e];
                    y[e] = y0 * c[e] + x0 * s[e];
                }
            }
        }
        T *row = static_cast<T *>(a.out[key]) + (t0 + t) * a.out_stride[key] +
                 static_cast<int64_t>(key ? h - a.q_heads : h) * a.out_head[key];
        if (in0) store<E>(row + i0, x);
        if (in1) store<E>(row + i1, y);
#pragma unroll
        for (int e = 0; e < E; ++e) x[e] = u[e], y[e] = v[e];
    }
}

template <typename T, int E, int G>
int launch(const RopeArgs &a, hipStream_t s) {
    RopeArgs b = a;
    unsigned parts = 1;
    if (a.rows >= kManyRows) {
        // four groups a token, and less than 2^32 threads: 2^24 rows take two tokens at least
        while (b.token_shift < 3 && ((kThreads / G) >> b.token_shift > 4 || a.rows >> b.token_shift >= 1 << 24)) ++b.token_shift;
    } else {
        parts = static_cast<unsigned>((a.heads + kThreads / G - 1) / (kThreads / G));
    }
    const int64_t tokens = int64_t{1} << b.token_shift;
    hipLaunchKernelGGL((qk_rope_kernel<T, E, G>), dim3(static_cast<unsigned>((a.rows + tokens - 1) / tokens), parts), dim3(kThreads), 0, s, b);
    return check_launch("qk_rope_kernel");
}
// Pieces of 16 bytes where a half is whole pieces, else of the largest power of
// two of values that divides it.
template <typename T>
int launch(const RopeArgs &a, hipStream_t s) {
    constexpr int kFull = 16 / sizeof(T);
    const int lanes = (a.d + 2 * kFull - 1) / (2 * kFull);
    if (a.half % kFull == 0) {
        if (lanes <= 4) return launch<T, kFull, 4>(a, s);
        if (lanes <= 8) return launch<T, kFull, 8>(a, s);
        if (sizeof(T) == 2 || lanes <= 16) return launch<T, kFull, 16>(a, s);
        if constexpr (sizeof(T) == 4) return launch<T, kFull, 32>(a, s);
    }
    if constexpr (sizeof(T) == 2)
        if (a.half % 4 == 0) return launch<T, 4, 32>(a, s);
    return launch<T, 2, 64>(a, s);
}

}  // namespace
}  // namespace ouro

using namespace ouro;

extern "C" int ouro_qk_norm_rope(const void *q, size_t q_stride, size_t q_head_stride, const void *k, size_t k_stride,
                                 size_t k_head_stride, const float *q_gain, const float *k_gain, const int32_t *pos, size_t axes,
                                 const int32_t *axis, const float *freq, size_t n_rot, unsigned flags, void *q_out,
                                 size_t q_out_stride, void *k_out, size_t k_out_stride, int dtype, size_t rows, size_t n_head,
                                 size_t n_head_kv, size_t head_dim, float eps, void *stream) {
    OURO_REQUIRE_INIT();
    const char *const me = "ouro_qk_norm_rope";
    if (dtype != OURO_DT_F32 && dtype != OURO_DT_BF16) return fail(OURO_ERR_INVALID_ARG, "%s: dtype %d", me, dtype);
    if (flags & ~OURO_ROPE_ADJACENT) return fail(OURO_ERR_INVALID_ARG, "%s: flags 0x%x", me, flags);
    if (!q || !q_out || (n_head_kv && (!k || !k_out)) || (n_rot && (!pos || !freq)))
        return fail(OURO_ERR_INVALID_ARG, "%s: NULL argument", me);
    if (!std::isfinite(eps) || eps < 0) return fail(OURO_ERR_INVALID_ARG, "%s: eps is negative or not finite", me);
    if (head_dim < 8 || head_dim > 256 || head_dim % 8 || n_rot % 4 || n_rot > head_dim)
        return fail(OURO_ERR_SHAPE, "%s: head_dim %zu (a multiple of 8, 8 .. 256), n_rot %zu (of 4, up to it)", me, head_dim, n_rot);
    if (n_head < 1 || n_head > 65535 || n_head_kv > 65535 || rows > (1u << 24) || axes < 1 || axes > 65535)
        return fail(OURO_ERR_SHAPE, "%s: %zu rows of %zu and %zu heads, %zu axes", me, rows, n_head, n_head_kv, axes);
    const size_t d = head_dim, heads[2] = {n_head, n_head_kv};
    size_t in[2] = {q_stride, k_stride}, head[2] = {q_head_stride, k_head_stride}, out[2] = {q_out_stride, k_out_stride};
    const void *src[2] = {q, k};
    void *dst[2] = {q_out, k_out};
    RopeArgs a{};
    const size_t unit = dtype == OURO_DT_F32 ? 4 : 8;
    for (int i = 0; i < (n_head_kv ? 2 : 1); ++i) {
        if (!head[i]) head[i] = d;
        const size_t in_row = (heads[i] - 1) * head[i] + d;
        if (!in[i]) in[i] = heads[i] * head[i];
        const size_t out_row = dst[i] == src[i] ? in_row : heads[i] * d;
        if (!out[i]) out[i] = dst[i] == src[i] ? in[i] : heads[i] * d;
        if (head[i] < d || in[i] < in_row || out[i] < out_row)
            return fail(OURO_ERR_SHAPE, "%s: a stride shorter than its row", me);
        if (dst[i] == src[i] && out[i] != in[i])
            return fail(OURO_ERR_INVALID_ARG, "%s: an output in its input's place has its strides", me);
        if ((reinterpret_cast<uintptr_t>(src[i]) | reinterpret_cast<uintptr_t>(dst[i])) & 15 || head[i] % unit || in[i] % unit || out[i] % unit)
            return fail(OURO_ERR_ALIGN, "%s: rows and heads must start at multiples of 16 bytes", me);
        if (in[i] > (size_t{1} << 40) || out[i] > (size_t{1} << 40)) return fail(OURO_ERR_SHAPE, "%s: a stride past 2^40", me);
        a.in[i] = src[i], a.out[i] = dst[i];
        a.in_stride[i] = static_cast<int64_t>(in[i]), a.head_stride[i] = static_cast<int64_t>(head[i]);
        a.out_stride[i] = static_cast<int64_t>(out[i]), a.out_head[i] = static_cast<int64_t>(dst[i] == src[i] ? head[i] : d);
    }
    if (!rows) return OURO_OK;
    a.gain[0] = q_gain, a.gain[1] = k_gain;
    a.pos = pos, a.axis = axis, a.freq = freq;
    a.rows = static_cast<int64_t>(rows);
    a.q_heads = static_cast<int>(n_head), a.heads = static_cast<int>(n_head + n_head_kv);
    a.d = static_cast<int>(d), a.half = static_cast<int>(n_rot / 2), a.axes = static_cast<int>(axes);
    a.adjacent = flags & OURO_ROPE_ADJACENT ? 1 : 0, a.eps = eps, a.inv_d = 1.0f / static_cast<float>(d);
    return dtype == OURO_DT_F32 ? launch<float>(a, as_stream(stream)) : launch<uint16_t>(a, as_stream(stream));
}
