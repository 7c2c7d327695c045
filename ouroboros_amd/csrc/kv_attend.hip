// kv_attend.hip - attention of one new token a sequence over a caller's paged
// key-value cache.
//
// For query head h of sequence b, over its visible slots j (j < n, the page
// there, the mask byte not 0):
//   s_j = scale q.k_j,  m = max s_j,  l = sum e^(s_j - m),
//   o = (1 / l) sum e^(s_j - m) v_j  [* sigmoid(gate)],  lse = m + ln l,
// and o = 0, lse = -inf where no slot is visible.
#include "kv_cache.hpp"

#include <cmath>

namespace ouro {

int kv_view(const ouro_kv_cache *c, const char *what, KvView *out) {
    if (!c || !c->k || !c->v || !c->pages) return fail(OURO_ERR_INVALID_ARG, "%s: NULL in the cache's description", what);
    if (c->dtype != OURO_DT_F32 && c->dtype != OURO_DT_BF16)
        return fail(OURO_ERR_INVALID_ARG, "%s: cache dtype %d", what, c->dtype);
    if (c->n_pages < 1 || c->max_pages < 1 || c->n_head_kv < 1 || c->n_head_kv > 65535)
        return fail(OURO_ERR_SHAPE, "%s: %d pages, %d a sequence, %d kv heads", what, c->n_pages, c->max_pages, c->n_head_kv);
    if (c->head_dim < 8 || c->head_dim > 256 || c->head_dim % 8)
        return fail(OURO_ERR_SHAPE, "%s: head_dim %d (a multiple of 8, 8 .. 256)", what, c->head_dim);
    if (c->page_tokens < 1 || c->page_tokens > (1 << 20) || (c->page_tokens & (c->page_tokens - 1)))
        return fail(OURO_ERR_SHAPE, "%s: %d tokens a page (a power of two up to 2^20)", what, c->page_tokens);
    const int64_t unit = c->dtype == OURO_DT_F32 ? 4 : 8;  // elements in 16 bytes
    if (c->page_stride < 0 || c->token_stride < 0 || c->head_stride < 0)
        return fail(OURO_ERR_SHAPE, "%s: negative stride", what);
    if (c->page_stride % unit || c->token_stride % unit || c->head_stride % unit ||
        (reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v)) & 15)
        return fail(OURO_ERR_ALIGN, "%s: pools and their strides must be multiples of 16 bytes", what);
    int shift = 0;
    while ((1 << shift) < c->page_tokens) ++shift;
    *out = KvView{c->k, c->v, c->pages, c->page_stride, c->token_stride, c->head_stride,
                  c->n_pages, c->max_pages, shift, c->n_head_kv, c->head_dim, 0};
    return OURO_OK;
}

int kv_check_history(const ouro_kv_history *h, int n_head_kv, size_t need, const char *what) {
    if (!h->weight || !h->pos) return fail(OURO_ERR_INVALID_ARG, "%s: NULL in the history", what);
    if (h->heads != 1 && h->heads != n_head_kv)
        return fail(OURO_ERR_SHAPE, "%s: a history of %d heads (1 or the cache's %d)", what, h->heads, n_head_kv);
    if (h->slots < 0 || static_cast<size_t>(h->slots) < need)
        return fail(OURO_ERR_SHAPE, "%s: a history of %d slots (at least %zu)", what, h->slots, need);
    return OURO_OK;
}

namespace {

struct AttendArgs {
    KvView c;
    const void *q, *k_new, *v_new, *gate;
    const int32_t *pos_new, *lens;
    const uint8_t *mask;
    void *out;
    float *lse, *weight;
    int32_t *pos;
    int64_t q_stride, new_stride, mask_stride, out_stride;
    int32_t n_head, max_len, h_heads, h_slots;
    float scale;
    int32_t pad;
};
// passed by value to kernels: the host and device passes must lay it out alike
static_assert(sizeof(AttendArgs) == 216, "AttendArgs: kernel argument layout");

template <typename T>
__device__ __forceinline__ float load1(const T *p, int64_t i) {
    if constexpr (sizeof(T) == 4)
        return p[i];
    else
        return bf16_bits_to_f32(p[i]);
}
template <typename T>
__device__ __forceinline__ void store1(T *p, int64_t i, float x) {
    if constexpr (sizeof(T) == 4)
        p[i] = x;
    else
        p[i] = f32_to_bf16_bits(x);
}
__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) v += xor_shfl(v, off);
    return v;
}

__device__ __forceinline__ int slots_of(const AttendArgs &a, int64_t b) { return max(0, min(a.lens[b], a.max_len)); }

// The new token's rows into slot n - 1, its weight cleared and its position
// noted.  One workgroup a (kv head, sequence).
template <typename C, typename IO>
__global__ __launch_bounds__(256) void kv_append_kernel(AttendArgs a) {
    const int h = blockIdx.x, t = threadIdx.x;
    const int64_t b = blockIdx.y;
    const int n = slots_of(a, b);
    if (!n) return;
    const int64_t at = kv_slot(a.c, b, n - 1);
    if (at >= 0 && t < a.c.d) {
        const int64_t src = b * a.new_stride + static_cast<int64_t>(h) * a.c.d + t, dst = at + h * a.c.head_stride + t;
        store1(static_cast<C *>(a.c.k), dst, load1(static_cast<const IO *>(a.k_new), src));
        store1(static_cast<C *>(a.c.v), dst, load1(static_cast<const IO *>(a.v_new), src));
    }
    if (a.weight && h < a.h_heads && t == 0) {
        const int64_t i = (b * a.h_heads + h) * a.h_slots + n - 1;
        a.weight[i] = 0.f;
        a.pos[i] = a.pos_new[b];
    }
}

// One workgroup a (query head, sequence): wavefront w takes slots w, w + 4,
// ... with lane l on dims l, l + 64, .. and keeps its own running maximum,
// sum and output; the four are joined in LDS.
template <typename C, typename IO>
__global__ __launch_bounds__(256) void kv_attend_kernel(AttendArgs a) {
    __shared__ float os[4][256], ms[4], ls[4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int h = blockIdx.x, d = a.c.d;
    const int64_t b = blockIdx.y;
    const int kvh = h / (a.n_head / a.c.n_head_kv);
    const int n = slots_of(a, b);
    float q[4], o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 4; ++i)
        q[i] = lane + 64 * i < d
                   ? load1(static_cast<const IO *>(a.q), b * a.q_stride + static_cast<int64_t>(h) * d + lane + 64 * i)
                   : 0.f;
    float m = -INFINITY, l = 0.f;
    for (int j = wave; j < n; j += 4) {
        if (a.mask && !a.mask[b * a.mask_stride + j]) continue;
        int64_t at = kv_slot(a.c, b, j);
        if (at < 0) continue;
        at += kvh * a.c.head_stride;
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (lane + 64 * i < d) s += q[i] * load1(static_cast<const C *>(a.c.k), at + lane + 64 * i);
        s = wave_sum(s) * a.scale;
        const float mn = fmaxf(m, s);
        if (mn == -INFINITY) continue;
        const float f = expf(m - mn), p = expf(s - mn);
        m = mn;
        l = l * f + p;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (lane + 64 * i < d) o[i] = o[i] * f + p * load1(static_cast<const C *>(a.c.v), at + lane + 64 * i);
    }
    if (lane == 0) ms[wave] = m, ls[wave] = l;
#pragma unroll
    for (int i = 0; i < 4; ++i) os[wave][lane + 64 * i] = o[i];
    __syncthreads();
    const float M = fmaxf(fmaxf(ms[0], ms[1]), fmaxf(ms[2], ms[3]));
    float L = 0.f, f[4];
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        f[w] = ms[w] == -INFINITY ? 0.f : expf(ms[w] - M);
        L += f[w] * ls[w];
    }
    const int t = threadIdx.x;
    if (t < d) {
        float r = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) r += f[w] * os[w][t];
        r = L != 0.f ? r / L : 0.f;
        const int64_t i = b * a.out_stride + static_cast<int64_t>(h) * d + t;
        if (a.gate) r *= 1.0f / (1.0f + expf(-load1(static_cast<const IO *>(a.gate), b * a.q_stride + static_cast<int64_t>(h) * d + t)));
        store1(static_cast<IO *>(a.out), i, r);
    }
    if (t == 0) a.lse[b * a.n_head + h] = M + logf(L);
}

// Adds each slot's attention weight to the history: one wavefront a slot, over
// the query heads of its history head, by the heads' log-sum-exp.
template <typename C, typename IO>
__global__ __launch_bounds__(256) void kv_weight_kernel(AttendArgs a) {
    const int lane = threadIdx.x & 63, d = a.c.d;
    const int j = blockIdx.x * 4 + (threadIdx.x >> 6), hs = blockIdx.y;
    const int64_t b = blockIdx.z;
    if (j >= slots_of(a, b)) return;
    if (a.mask && !a.mask[b * a.mask_stride + j]) return;
    const int64_t row = kv_slot(a.c, b, j);
    if (row < 0) return;
    const int G = a.n_head / a.h_heads, per = a.n_head / a.c.n_head_kv;
    float w = 0.f;
    for (int h = hs * G; h < hs * G + G; ++h) {
        const int64_t at = row + (h / per) * a.c.head_stride;
        float s = 0.f;
        for (int i = lane; i < d; i += 64)
            s += load1(static_cast<const IO *>(a.q), b * a.q_stride + static_cast<int64_t>(h) * d + i) *
                 load1(static_cast<const C *>(a.c.k), at + i);
        s = wave_sum(s) * a.scale;
        if (s != -INFINITY) w += expf(s - a.lse[b * a.n_head + h]);
    }
    if (lane == 0) a.weight[(b * a.h_heads + hs) * a.h_slots + j] += w;
}

template <typename C, typename IO>
int launch_attend(const AttendArgs &a, unsigned seqs, hipStream_t s) {
    int st;
    if (a.k_new) {
        hipLaunchKernelGGL((kv_append_kernel<C, IO>), dim3(a.c.n_head_kv, seqs), dim3(256), 0, s, a);
        if ((st = check_launch("kv_append_kernel"))) return st;
    }
    hipLaunchKernelGGL((kv_attend_kernel<C, IO>), dim3(a.n_head, seqs), dim3(256), 0, s, a);
    if ((st = check_launch("kv_attend_kernel"))) return st;
    if (a.weight && a.max_len) {
        hipLaunchKernelGGL((kv_weight_kernel<C, IO>), dim3((a.max_len + 3) / 4, a.h_heads, seqs), dim3(256), 0, s, a);
        if ((st = check_launch("kv_weight_kernel"))) return st;
    }
    return OURO_OK;
}

size_t attend_ws_bytes(size_t seqs, size_t n_head) { return (seqs * n_head * sizeof(float) + 255) & ~size_t{255}; }

}  // namespace
}  // namespace ouro

using namespace ouro;

extern "C" {

size_t ouro_kv_attend_workspace_bytes(size_t seqs, size_t n_head, size_t head_dim, size_t max_len, int with_history) {
    (void)head_dim;
    (void)max_len;
    (void)with_history;
    return attend_ws_bytes(seqs, n_head);
}

int ouro_kv_attend(const ouro_kv_cache *cache, const ouro_kv_history *history, const void *q, size_t q_stride,
                   const void *k_new, const void *v_new, size_t new_stride, const int32_t *pos_new,
                   const int32_t *lens, const uint8_t *mask, size_t mask_stride, const void *gate, void *out,
                   size_t out_stride, float *lse, int dtype, size_t seqs, size_t n_head, size_t max_len, float scale,
                   void *ws, void *stream) {
    OURO_REQUIRE_INIT();
    const char *const me = "ouro_kv_attend";
    AttendArgs a{};
    int st = kv_view(cache, me, &a.c);
    if (st) return st;
    if (!q || !lens || !out) return fail(OURO_ERR_INVALID_ARG, "%s: NULL argument", me);
    if (!k_new != !v_new) return fail(OURO_ERR_INVALID_ARG, "%s: a new key without its value, or the reverse", me);
    if (dtype != OURO_DT_F32 && dtype != OURO_DT_BF16) return fail(OURO_ERR_INVALID_ARG, "%s: dtype %d", me, dtype);
    if (!std::isfinite(scale)) return fail(OURO_ERR_INVALID_ARG, "%s: scale is not finite", me);
    const size_t hkv = cache->n_head_kv, d = cache->head_dim;
    if (seqs > 65535 || n_head < 1 || n_head > 65535 || n_head % hkv)
        return fail(OURO_ERR_SHAPE, "%s: %zu sequences (up to 65535), %zu heads over %zu kv heads", me, seqs, n_head, hkv);
    if (max_len > static_cast<size_t>(cache->max_pages) * cache->page_tokens || max_len > (1u << 30))
        return fail(OURO_ERR_SHAPE, "%s: %zu slots of %d pages of %d tokens", me, max_len, cache->max_pages, cache->page_tokens);
    if (!q_stride) q_stride = n_head * d;
    if (!out_stride) out_stride = n_head * d;
    if (!new_stride) new_stride = hkv * d;
    if (!mask_stride) mask_stride = max_len;
    if (q_stride < n_head * d || out_stride < n_head * d || new_stride < hkv * d || mask_stride < max_len)
        return fail(OURO_ERR_SHAPE, "%s: a stride shorter than its row", me);
    const size_t unit = dtype == OURO_DT_F32 ? 4 : 8;
    const uintptr_t bits = reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(k_new) |
                           reinterpret_cast<uintptr_t>(v_new) | reinterpret_cast<uintptr_t>(gate);
    if (bits & 15 || q_stride % unit || out_stride % unit || new_stride % unit)
        return fail(OURO_ERR_ALIGN, "%s: rows must start at multiples of 16 bytes", me);
    if (history) {
        if ((st = kv_check_history(history, cache->n_head_kv, max_len, me))) return st;
        if (k_new && !pos_new) return fail(OURO_ERR_INVALID_ARG, "%s: a new key without its position in the history", me);
        a.weight = history->weight;
        a.pos = history->pos;
        a.h_heads = history->heads;
        a.h_slots = history->slots;
    }
    if (!seqs) return OURO_OK;
    if (!lse) {
        if (!ws && !(ws = workspace(attend_ws_bytes(seqs, n_head), stream))) return OURO_ERR_HIP;
        lse = static_cast<float *>(ws);
    }
    a.q = q, a.k_new = k_new, a.v_new = v_new, a.gate = gate, a.pos_new = pos_new, a.lens = lens, a.mask = mask, a.out = out, a.lse = lse;
    a.q_stride = q_stride, a.new_stride = new_stride, a.mask_stride = mask_stride, a.out_stride = out_stride;
    a.n_head = static_cast<int>(n_head), a.max_len = static_cast<int>(max_len), a.scale = scale;
    const bool bc = cache->dtype == OURO_DT_BF16, bi = dtype == OURO_DT_BF16;
    const unsigned B = static_cast<unsigned>(seqs);
    hipStream_t s = as_stream(stream);
    if (bc) return bi ? launch_attend<uint16_t, uint16_t>(a, B, s) : launch_attend<uint16_t, float>(a, B, s);
    return bi ? launch_attend<float, uint16_t>(a, B, s) : launch_attend<float, float>(a, B, s);
}

}  // extern "C"
