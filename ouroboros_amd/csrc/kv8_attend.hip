// kv8_attend.hip - attention of each sequence's newest rows over a paged cache
// of 8-bit codes with a scale for each block of slots and kv head.
//
// For query head h of the row in slot r, over its visible slots j:
//   s_j = scale q.k_j,  m = max s_j,  l = sum e^(s_j - m),
//   o = (1 / l) sum e^(s_j - m) v_j  [* sigmoid(gate)],  lse = m + ln l,
// and o = 0, lse = -inf where no slot is visible.
#include "kv_cache.hpp"

#include <cmath>

namespace ouro {
namespace {

struct Attend8Args {
    Kv8View c;
    NewRows r;
    const void *q, *gate;
    const uint8_t *mask;
    void *out;
    float *lse;
    int64_t q_stride, mask_stride, out_stride;
    int32_t n_head, window, sinks;
    float scale;
};

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

// One wavefront a row and head, 64 slots at a time, a lane each.
template <typename IO>
__global__ __launch_bounds__(64) void kv8_attend_kernel(Attend8Args a) {
    const SeqRows s = seq_rows(a.r, blockIdx.z);
    const int i = blockIdx.x, h = blockIdx.y, lane = threadIdx.x;
    if (i >= s.count) return;
    const int64_t b = blockIdx.z, row = s.first + i;
    const int d = a.c.d, at = s.n - s.count + i, kvh = h / (a.n_head / a.c.n_head_kv);
    const IO *q = static_cast<const IO *>(a.q) + row * a.q_stride + static_cast<int64_t>(h) * d;
    float o[4] = {0.f, 0.f, 0.f, 0.f}, m = -INFINITY, l = 0.f;
    for (int j0 = 0; j0 <= at; j0 += 64) {
        const int j = j0 + lane;
        bool seen = j <= at && (!a.window || at - j < a.window || j < a.sinks);
        int32_t page = -1;
        if (seen) {
            page = a.c.pages[b * a.c.max_pages + (j >> a.c.page_shift)];
            seen = page >= 0 && page < a.c.n_pages && (!a.mask || a.mask[b * a.mask_stride + j] != 0);
        }
        const int t = j & ((1 << a.c.page_shift) - 1);
        float sc = -INFINITY;
        if (seen) {
            const int8_t *k = a.c.k + kv8_row(a.c, page, t) + kvh * a.c.head_stride;
            float x = 0.f;
            for (int e = 0; e < d; ++e) x += load1(q, e) * static_cast<float>(k[e]);
            sc = x * a.c.k_scale[kv8_scale(a.c, page, t, kvh)] * a.scale;
        }
        const uint64_t any = __ballot(seen);
        float top = sc;
        for (int off = 32; off >= 1; off >>= 1) top = fmaxf(top, xor_shfl(top, off));
        const float mn = fmaxf(m, top), ref = mn == -INFINITY ? 0.f : mn, corr = expf(m - ref);
        m = mn;
        const float p = seen ? expf(sc - ref) : 0.f;
        float sum = p;
        for (int off = 32; off >= 1; off >>= 1) sum += xor_shfl(sum, off);
        l = l * corr + sum;
        for (int e = 0; e < 4; ++e) o[e] *= corr;
        for (int u = 0; u < 64; ++u) {
            if (!((any >> u) & 1)) continue;
            const int pg = __shfl(page, u, 64), tu = (j0 + u) & ((1 << a.c.page_shift) - 1);
            const float w = __shfl(p, u, 64) * a.c.v_scale[kv8_scale(a.c, pg, tu, kvh)];
            const int8_t *v = a.c.v + kv8_row(a.c, pg, tu) + kvh * a.c.head_stride;
            for (int e = 0; e < 4; ++e)
                if (lane + 64 * e < d) o[e] += w * static_cast<float>(v[lane + 64 * e]);
        }
    }
    for (int e = 0; e < 4; ++e) {
        const int dim = lane + 64 * e;
        if (dim >= d) break;
        float x = l == 0.f ? 0.f : o[e] / l;
        if (a.gate) x *= 1.0f / (1.0f + expf(-load1(static_cast<const IO *>(a.gate), row * a.q_stride + static_cast<int64_t>(h) * d + dim)));
        store1(static_cast<IO *>(a.out), row * a.out_stride + static_cast<int64_t>(h) * d + dim, x);
    }
    if (lane == 0 && a.lse) a.lse[row * a.n_head + h] = l == 0.f ? -INFINITY : m + logf(l);
}

}  // namespace
}  // namespace ouro

using namespace ouro;

extern "C" {

size_t ouro_kv8_attend_workspace_bytes(size_t, size_t, size_t, size_t, size_t, size_t, size_t) { return 0; }

int ouro_kv8_attend(const ouro_kv8_cache *cache, const void *q, size_t q_stride, const int32_t *lens, const int32_t *cu,
                    const uint8_t *mask, size_t mask_stride, const void *gate, void *out, size_t out_stride, float *lse, int dtype,
                    size_t seqs, size_t rows, size_t max_new, size_t n_head, size_t max_len, size_t window, size_t sinks,
                    float scale, void *ws, void *stream) {
    OURO_REQUIRE_INIT();
    const char *const me = "ouro_kv8_attend";
    Attend8Args a{};
    int st = kv8_view(cache, me, &a.c);
    if (st) return st;
    if (max_len > static_cast<size_t>(cache->max_pages) * static_cast<size_t>(cache->page_tokens) || max_len > (1u << 30))
        return fail(OURO_ERR_SHAPE, "%s: %zu slots of %d pages of %d tokens", me, max_len, cache->max_pages, cache->page_tokens);
    if ((st = new_rows(lens, cu, seqs, rows, max_new, max_len, me, &a.r))) return st;
    if (!q || !out) return fail(OURO_ERR_INVALID_ARG, "%s: NULL argument", me);
    if (dtype != OURO_DT_F32 && dtype != OURO_DT_BF16) return fail(OURO_ERR_INVALID_ARG, "%s: dtype %d", me, dtype);
    if (!std::isfinite(scale)) return fail(OURO_ERR_INVALID_ARG, "%s: scale is not finite", me);
    const size_t hkv = static_cast<size_t>(cache->n_head_kv), d = static_cast<size_t>(cache->head_dim);
    if (n_head < 1 || n_head > 65535 || n_head % hkv)
        return fail(OURO_ERR_SHAPE, "%s: %zu heads over %zu kv heads", me, n_head, hkv);
    if (!q_stride) q_stride = n_head * d;
    if (!out_stride) out_stride = n_head * d;
    if (!mask_stride) mask_stride = max_len;
    if (q_stride < n_head * d || out_stride < n_head * d || mask_stride < max_len)
        return fail(OURO_ERR_SHAPE, "%s: a stride shorter than its row", me);
    const size_t unit = dtype == OURO_DT_F32 ? 4 : 8;
    if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(gate)) & 15 ||
        q_stride % unit || out_stride % unit)
        return fail(OURO_ERR_ALIGN, "%s: rows must start at multiples of 16 bytes", me);
    if (!seqs || !(max_new = static_cast<size_t>(a.r.max_new))) return OURO_OK;
    auto most = [](size_t x) { return static_cast<int32_t>(x < (1u << 30) ? x : 1u << 30); };
    a.q = q, a.gate = gate, a.mask = mask, a.out = out, a.lse = lse;
    a.q_stride = static_cast<int64_t>(q_stride), a.out_stride = static_cast<int64_t>(out_stride);
    a.mask_stride = static_cast<int64_t>(mask_stride);
    a.n_head = static_cast<int>(n_head), a.window = most(window), a.sinks = most(sinks), a.scale = scale;
    (void)ws;
    const dim3 grid(static_cast<unsigned>(max_new), static_cast<unsigned>(n_head), static_cast<unsigned>(seqs));
    if (dtype == OURO_DT_F32)
        hipLaunchKernelGGL(kv8_attend_kernel<float>, grid, dim3(64), 0, as_stream(stream), a);
    else
        hipLaunchKernelGGL(kv8_attend_kernel<uint16_t>, grid, dim3(64), 0, as_stream(stream), a);
    return check_launch("kv8_attend_kernel");
}

}  // extern "C"
