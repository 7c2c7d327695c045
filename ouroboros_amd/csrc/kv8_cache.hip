// kv8_cache.hip - a paged key-value cache of int8 codes with a float scale for
// each block of slots and kv head: new rows quantised as they are written, and
// rows read back.
//
// A block's scale is the smallest power of two s with max |x| <= 127 s over its
// rows, code = rint(x / s).  A power of two, not max |x| / 127, because rows come
// a few at a time: what the scale must grow by is then a shift of the codes, so
// that all the roundings that a row can suffer add up to less than one step, the
// scale does not depend on the pieces in which the rows came, code * s is exact
// in bf16 and fp32, and x / s is exact, so that the codes are the same wherever
// they are computed.  It costs up to one of the eight bits.
#include "kv_cache.hpp"

namespace ouro {

int kv8_view(const ouro_kv8_cache *c, const char *what, Kv8View *out) {
    if (!c || !c->k || !c->v || !c->k_scale || !c->v_scale || !c->pages)
        return fail(OURO_ERR_INVALID_ARG, "%s: NULL in the cache's description", what);
    if (c->n_pages < 1 || c->max_pages < 1 || c->n_head_kv < 1 || c->n_head_kv > 32767)
        return fail(OURO_ERR_SHAPE, "%s: %d pages, %d a sequence, %d kv heads", what, c->n_pages, c->max_pages, c->n_head_kv);
    if (c->head_dim < 16 || c->head_dim > 256 || c->head_dim % 16)
        return fail(OURO_ERR_SHAPE, "%s: head_dim %d (a multiple of 16, 16 .. 256)", what, c->head_dim);
    auto power = [](int x) { return (x & (x - 1)) == 0; };
    if (c->page_tokens < 16 || c->page_tokens > (1 << 20) || !power(c->page_tokens))
        return fail(OURO_ERR_SHAPE, "%s: %d tokens a page (a power of two, 16 .. 2^20)", what, c->page_tokens);
    if (c->block_tokens < 16 || c->block_tokens > 256 || c->block_tokens > c->page_tokens || !power(c->block_tokens))
        return fail(OURO_ERR_SHAPE, "%s: %d tokens a block (a power of two, 16 .. 256, at most a page)", what, c->block_tokens);
    if (c->page_stride < 0 || c->token_stride < 0 || c->head_stride < 0 || c->token_stride > (1 << 24))
        return fail(OURO_ERR_SHAPE, "%s: a negative stride, or tokens over 2^24 bytes apart", what);
    if (c->page_stride % 16 || c->token_stride % 16 || c->head_stride % 16 ||
        (reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v)) & 15)
        return fail(OURO_ERR_ALIGN, "%s: pools and their strides must be multiples of 16 bytes", what);
    if ((reinterpret_cast<uintptr_t>(c->k_scale) | reinterpret_cast<uintptr_t>(c->v_scale)) & 3)
        return fail(OURO_ERR_ALIGN, "%s: scales must be floats at multiples of 4 bytes", what);
    auto shift = [](int x) {
        int s = 0;
        while ((1 << s) < x) ++s;
        return s;
    };
    *out = Kv8View{c->k, c->v, c->k_scale, c->v_scale, c->pages, c->page_stride, c->token_stride, c->head_stride,
                   c->n_pages, c->max_pages, shift(c->page_tokens), shift(c->block_tokens), c->n_head_kv, c->head_dim};
    return OURO_OK;
}

int new_rows(const int32_t *lens, const int32_t *cu, size_t seqs, size_t rows, size_t max_new, size_t max_len, const char *what,
             NewRows *out) {
    if (!lens) return fail(OURO_ERR_INVALID_ARG, "%s: lens is NULL", what);
    if (seqs > 65535 || rows > (1u << 23))
        return fail(OURO_ERR_SHAPE, "%s: %zu sequences (up to 65535), %zu rows (up to 2^23)", what, seqs, rows);
    if (!cu && (max_new > rows || rows != seqs * max_new))
        return fail(OURO_ERR_SHAPE, "%s: %zu rows of %zu sequences of %zu", what, rows, seqs, max_new);
    if (max_new > rows) max_new = rows;
    *out = NewRows{lens, cu, static_cast<int32_t>(rows), static_cast<int32_t>(max_new), static_cast<int32_t>(max_len)};
    return OURO_OK;
}

namespace {

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));

// Slots that the page table can name: lengths are held to it.
size_t table_slots(const ouro_kv8_cache *c) {
    const size_t n = static_cast<size_t>(c->max_pages) * static_cast<size_t>(c->page_tokens);
    return n < (1u << 30) ? n : 1u << 30;
}

struct WriteArgs {
    Kv8View c;
    NewRows r;
    const void *src[2];
    int64_t stride;
    uint32_t row_magic;  // floor(i / (d / 8)) = i row_magic >> 18, i < 8192
    int32_t pad;
};
static_assert(sizeof(WriteArgs) == 152, "WriteArgs: kernel argument layout");

// Eight adjacent values of a row.
template <typename T>
__device__ __forceinline__ void load8(const T *p, float (&x)[8]) {
    if constexpr (sizeof(T) == 4) {
        const f32x4_t a = *reinterpret_cast<const f32x4_t *>(p), b = *reinterpret_cast<const f32x4_t *>(p + 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = a[e], x[4 + e] = b[e];
    } else {
        const u32x4_t v = *reinterpret_cast<const u32x4_t *>(p);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = __uint_as_float(e & 1 ? v[e / 2] & 0xffff0000u : v[e / 2] << 16);
    }
}
// The smallest power of two s with m <= 127 s: m = f 2^e with 1 <= f < 2 takes
// e - 6 where f <= 127/64 and e - 5 above, held to normal numbers; 0 for 0.
__device__ __forceinline__ float scale_for(float m) {
    if (m == 0.f) return 0.f;
    const uint32_t u = __float_as_uint(m);
    const int e = static_cast<int>(u >> 23) - ((u & 0x7fffffu) <= 0x7e0000u ? 6 : 5);
    return __uint_as_float(static_cast<uint32_t>(max(e, 1)) << 23);
}
// rint(x r) as an int8's bits, NaN as 0.
__device__ __forceinline__ uint32_t code_of(float x, float r) {
    const float t = rintf(x * r);
    const int i = t != t ? 0 : static_cast<int>(fminf(fmaxf(t, -127.f), 127.f));
    return static_cast<uint32_t>(i) & 0xffu;
}

// One workgroup of U threads takes a block of slots that gets rows, of one kv
// head and of keys or values: its new rows into registers, NC pieces of eight
// values a thread, their largest magnitude, the scale, the codes.  Only where the
// block holds older rows and its scale grew are they read and written.
//
// 32 prompts of up to 2048 rows, bf16, blocks of 16: 32 us, 3.9 TB/s where a copy has
// 5 (a wavefront a block; four blocks a workgroup 33).  64 single rows 4.5 us on the
// GPU: lengths, page, old scale and rows are loads that wait for each other.
template <typename T, int U, int NC>
__global__ __launch_bounds__(U) void kv8_write_kernel(WriteArgs a) {
    __shared__ float top[U / 64];
    const int tid = threadIdx.x, which = blockIdx.y & 1, head = blockIdx.y >> 1;
    const SeqRows s = seq_rows(a.r, blockIdx.z);
    const int start = s.n - s.count;  // below 0 where rows have no slot
    const int bt = 1 << a.c.block_shift;
    const int block = (max(start, 0) >> a.c.block_shift) + static_cast<int>(blockIdx.x);
    const int j0 = block << a.c.block_shift, lo = max(max(start, 0), j0), hi = min(s.n, j0 + bt);
    if (lo >= hi) return;  // whole workgroup
    const int32_t page = a.c.pages[static_cast<int64_t>(blockIdx.z) * a.c.max_pages + (j0 >> a.c.page_shift)];
    if (page < 0 || page >= a.c.n_pages) return;
    const int t0 = j0 & ((1 << a.c.page_shift) - 1);  // the block's first token in its page
    float *const scale = (which ? a.c.v_scale : a.c.k_scale) + kv8_scale(a.c, page, t0, head);
    int8_t *const codes = (which ? a.c.v : a.c.k) + kv8_row(a.c, page, t0) + head * a.c.head_stride;
    const float before = lo > j0 ? *scale : 0.f;
    const int d = a.c.d, pieces = (hi - lo) * (d / 8);
    const T *const src = static_cast<const T *>(a.src[which]) + static_cast<int64_t>(head) * d;
    auto row_of = [&](int i) { return static_cast<int>(static_cast<uint32_t>(i) * a.row_magic >> 18); };
    float x[NC][8];
    float m = 0.f;
#pragma unroll
    for (int k = 0; k < NC; ++k) {
        const int i = k * U + tid, row = row_of(i);
        if (i < pieces) load8(src + (s.first + (lo - start) + row) * a.stride + 8 * (i - row * (d / 8)), x[k]);
    }
#pragma unroll
    for (int k = 0; k < NC; ++k)
        if (k * U + tid < pieces)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float v = fabsf(x[k][e]);
                m = fmaxf(m, v < INFINITY ? v : 0.f);
            }
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) m = fmaxf(m, xor_shfl(m, off));
    if constexpr (U > 64) {
        if ((tid & 63) == 0) top[tid >> 6] = m;
        __syncthreads();  // every thread has read the old scale too
#pragma unroll
        for (int w = 0; w < U / 64; ++w) m = fmaxf(m, top[w]);
    }
    const float now = fmaxf(before, scale_for(m));
    const float inv = now > 0.f ? 1.0f / now : 0.f;
#pragma unroll
    for (int k = 0; k < NC; ++k) {
        const int i = k * U + tid, row = row_of(i);
        if (i < pieces) {
            uint32_t w[2];
#pragma unroll
            for (int e = 0; e < 2; ++e)
                w[e] = code_of(x[k][4 * e], inv) | code_of(x[k][4 * e + 1], inv) << 8 | code_of(x[k][4 * e + 2], inv) << 16 |
                       code_of(x[k][4 * e + 3], inv) << 24;
            *reinterpret_cast<u32x2_t *>(codes + (lo - j0 + row) * a.c.token_stride + 8 * (i - row * (d / 8))) = u32x2_t{w[0], w[1]};
        }
    }
    if (now != before || lo == j0) {
        if (tid == 0) *scale = now;
        const float ratio = now > 0.f ? before / now : 0.f;
        for (int i = tid; i < (lo - j0) * (d / 8); i += U) {  // none where the block begins here
            const int row = row_of(i);
            u32x2_t *const p = reinterpret_cast<u32x2_t *>(codes + row * a.c.token_stride + 8 * (i - row * (d / 8)));
            u32x2_t w = *p;
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                uint32_t u = 0;
#pragma unroll
                for (int e = 0; e < 4; ++e) u |= code_of(static_cast<float>(static_cast<int8_t>(w[q] >> (8 * e))), ratio) << (8 * e);
                w[q] = u;
            }
            *p = w;
        }
    }
}

template <typename T, int U, int NC>
int launch_write(const WriteArgs &a, unsigned blocks, unsigned seqs, hipStream_t s) {
    hipLaunchKernelGGL((kv8_write_kernel<T, U, NC>), dim3(blocks, 2 * a.c.n_head_kv, seqs), dim3(U), 0, s, a);
    return check_launch("kv8_write_kernel");
}
// Threads and pieces of a workgroup by the values that a block can get in a call.
template <typename T>
int launch_write(const WriteArgs &a, unsigned blocks, unsigned seqs, hipStream_t s) {
    const int bt = 1 << a.c.block_shift, rows = a.r.max_new < bt ? a.r.max_new : bt;
    const int values = rows * a.c.d;
    if (values <= 64 * 32) return launch_write<T, 64, 4>(a, blocks, seqs, s);
    if (values <= 256 * 32) return launch_write<T, 256, 4>(a, blocks, seqs, s);
    if (values <= 1024 * 32) return launch_write<T, 1024, 4>(a, blocks, seqs, s);
    return launch_write<T, 1024, 8>(a, blocks, seqs, s);
}

struct ReadArgs {
    Kv8View c;
    NewRows r;
    void *dst[2];
    int64_t stride;
};
static_assert(sizeof(ReadArgs) == 144, "ReadArgs: kernel argument layout");

// A thread makes 16 bytes of the output, four or eight codes of a row and head, of
// kReadRows rows, whose loads are on their way together: 48 contexts of up to 2048
// rows to bf16 38 us, 4.4 TB/s where a copy has 5 (one row at a time 52).
constexpr int kReadRows = 4;
template <typename T>
__global__ __launch_bounds__(256) void kv8_read_kernel(ReadArgs a, int per_row) {
    constexpr int E = 16 / sizeof(T);
    const SeqRows s = seq_rows(a.r, blockIdx.z);
    const int which = blockIdx.y;
    if (!a.dst[which]) return;
    const int d = a.c.d, pieces = d / E * a.c.n_head_kv;  // of a row
    const int at_once = 256 / per_row, row0 = static_cast<int>(blockIdx.x) * at_once * kReadRows + static_cast<int>(threadIdx.x) / per_row;
    if (static_cast<int>(threadIdx.x) >= at_once * per_row) return;
    int32_t page[kReadRows];
    int t[kReadRows];
#pragma unroll
    for (int k = 0; k < kReadRows; ++k) {
        const int row = row0 + k * at_once, slot = s.n - s.count + row;
        page[k] = -1;
        if (row < s.count && slot >= 0) page[k] = a.c.pages[static_cast<int64_t>(blockIdx.z) * a.c.max_pages + (slot >> a.c.page_shift)];
        t[k] = slot & ((1 << a.c.page_shift) - 1);
    }
    for (int i = static_cast<int>(threadIdx.x) % per_row; i < pieces; i += per_row) {
        const int head = i / (d / E), dim = i % (d / E) * E;
        const int8_t *const pool = (which ? a.c.v : a.c.k) + head * a.c.head_stride + dim;
        uint32_t w[kReadRows][E / 4];
        float f[kReadRows];
#pragma unroll
        for (int k = 0; k < kReadRows; ++k) {
            f[k] = 0.f;
            w[k][0] = w[k][E / 4 - 1] = 0;
            if (page[k] < 0 || page[k] >= a.c.n_pages) continue;
            const int8_t *p = pool + kv8_row(a.c, page[k], t[k]);
            f[k] = (which ? a.c.v_scale : a.c.k_scale)[kv8_scale(a.c, page[k], t[k], head)];
            if constexpr (E == 4) {
                w[k][0] = *reinterpret_cast<const uint32_t *>(p);
            } else {
                const u32x2_t v = *reinterpret_cast<const u32x2_t *>(p);
                w[k][0] = v[0], w[k][1] = v[1];
            }
        }
#pragma unroll
        for (int k = 0; k < kReadRows; ++k) {
            const int row = row0 + k * at_once;
            if (row >= s.count) break;
            float x[E];
#pragma unroll
            for (int e = 0; e < E; ++e) x[e] = static_cast<float>(static_cast<int8_t>(w[k][e / 4] >> (8 * (e & 3)))) * f[k];
            T *out = static_cast<T *>(a.dst[which]) + (s.first + row) * a.stride + static_cast<int64_t>(head) * d + dim;
            if constexpr (E == 4) {
                *reinterpret_cast<f32x4_t *>(out) = f32x4_t{x[0], x[1], x[2], x[3]};
            } else {
                u32x4_t v;
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = f32_to_bf16_bits(x[2 * e]) | static_cast<uint32_t>(f32_to_bf16_bits(x[2 * e + 1])) << 16;
                *reinterpret_cast<u32x4_t *>(out) = v;
            }
        }
    }
}

// Rows' stride: whole rows of n_head_kv heads, 16-byte multiples.
int row_stride(const char *me, const ouro_kv8_cache *c, int dtype, size_t *stride, const void *a, const void *b) {
    if (dtype != OURO_DT_F32 && dtype != OURO_DT_BF16) return fail(OURO_ERR_INVALID_ARG, "%s: dtype %d", me, dtype);
    const size_t row = static_cast<size_t>(c->n_head_kv) * c->head_dim, unit = dtype == OURO_DT_F32 ? 4 : 8;
    if (!*stride) *stride = row;
    if (*stride < row || *stride > (size_t{1} << 32)) return fail(OURO_ERR_SHAPE, "%s: a stride shorter than its row, or past 2^32", me);
    if ((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b)) & 15 || *stride % unit)
        return fail(OURO_ERR_ALIGN, "%s: rows must start at multiples of 16 bytes", me);
    return OURO_OK;
}

}  // namespace
}  // namespace ouro

using namespace ouro;

extern "C" {

int ouro_kv8_write(const ouro_kv8_cache *cache, const void *k_new, const void *v_new, size_t new_stride, int dtype,
                   const int32_t *lens, const int32_t *cu, size_t seqs, size_t rows, size_t max_new, void *stream) {
    OURO_REQUIRE_INIT();
    const char *const me = "ouro_kv8_write";
    WriteArgs a{};
    int st = kv8_view(cache, me, &a.c);
    if (st) return st;
    if ((st = new_rows(lens, cu, seqs, rows, max_new, table_slots(cache), me, &a.r))) return st;
    if (!k_new || !v_new) return fail(OURO_ERR_INVALID_ARG, "%s: NULL argument", me);
    if ((st = row_stride(me, cache, dtype, &new_stride, k_new, v_new))) return st;
    if (!seqs || !(max_new = static_cast<size_t>(a.r.max_new))) return OURO_OK;
    a.src[0] = k_new, a.src[1] = v_new;
    a.stride = static_cast<int64_t>(new_stride);
    const uint32_t per = static_cast<uint32_t>(cache->head_dim) / 8;
    a.row_magic = ((1u << 18) + per - 1) / per;
    // blocks that max_new rows in a row can touch
    const size_t bt = static_cast<size_t>(cache->block_tokens);
    const unsigned blocks = static_cast<unsigned>((max_new + bt - 2) / bt + 1);
    return dtype == OURO_DT_F32 ? launch_write<float>(a, blocks, static_cast<unsigned>(seqs), as_stream(stream))
                                : launch_write<uint16_t>(a, blocks, static_cast<unsigned>(seqs), as_stream(stream));
}

int ouro_kv8_read(const ouro_kv8_cache *cache, const int32_t *lens, const int32_t *cu, size_t seqs, size_t rows, size_t max_new,
                  void *k_out, void *v_out, size_t out_stride, int dtype, void *stream) {
    OURO_REQUIRE_INIT();
    const char *const me = "ouro_kv8_read";
    ReadArgs a{};
    int st = kv8_view(cache, me, &a.c);
    if (st) return st;
    if ((st = new_rows(lens, cu, seqs, rows, max_new, table_slots(cache), me, &a.r))) return st;
    if ((st = row_stride(me, cache, dtype, &out_stride, k_out, v_out))) return st;
    if (!seqs || !(max_new = static_cast<size_t>(a.r.max_new)) || (!k_out && !v_out)) return OURO_OK;
    a.dst[0] = k_out, a.dst[1] = v_out;
    a.stride = static_cast<int64_t>(out_stride);
    const int pieces = cache->head_dim / (dtype == OURO_DT_F32 ? 4 : 8) * cache->n_head_kv;
    const int per_row = pieces < 256 ? pieces : 256;
    const size_t at_once = static_cast<size_t>(256 / per_row * kReadRows);
    const dim3 grid(static_cast<unsigned>((max_new + at_once - 1) / at_once), 2, static_cast<unsigned>(seqs));
    hipStream_t s = as_stream(stream);
    if (dtype == OURO_DT_F32)
        hipLaunchKernelGGL(kv8_read_kernel<float>, grid, dim3(256), 0, s, a, per_row);
    else
        hipLaunchKernelGGL(kv8_read_kernel<uint16_t>, grid, dim3(256), 0, s, a, per_row);
    return check_launch("kv8_read_kernel");
}

}  // extern "C"
