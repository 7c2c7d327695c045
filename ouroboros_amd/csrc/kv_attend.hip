// kv_attend.hip - attention of one new token a sequence over a caller's paged
// key-value cache.
//
// For query head h of sequence b, over its visible slots j (j < n, the page
// there, the mask byte not 0):
//   s_j = scale q.k_j,  m = max s_j,  l = sum e^(s_j - m),
//   o = (1 / l) sum e^(s_j - m) v_j  [* sigmoid(gate)],  lse = m + ln l,
// and o = 0, lse = -inf where no slot is visible.
//
// A running maximum passes over a NaN score, whose p = e^(s - m) makes the sum
// NaN: the sum alone says whether anything was there (0: no score above -inf).
#include "kv_cache.hpp"

#include <atomic>
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
    if (c->page_stride < 0 || c->token_stride < 0 || c->head_stride < 0 || c->token_stride > (1 << 24))
        return fail(OURO_ERR_SHAPE, "%s: a negative stride, or tokens over 2^24 elements apart", what);
    if (c->page_stride % unit || c->token_stride % unit || c->head_stride % unit ||
        (reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v)) & 15)
        return fail(OURO_ERR_ALIGN, "%s: pools and their strides must be multiples of 16 bytes", what);
    int shift = 0;
    while ((1 << shift) < c->page_tokens) ++shift;
    *out = KvView{c->k, c->v, c->pages, c->page_stride, c->token_stride, c->head_stride,
                  c->n_pages, c->max_pages, shift, c->n_head_kv, c->head_dim, c->dtype == OURO_DT_F32 ? 4 : 2};
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

typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef float f32x2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef short bf16x4_t __attribute__((ext_vector_type(4)));  // the builtin's type of four bf16
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef short i16x2_t __attribute__((ext_vector_type(2)));
typedef unsigned short u16x2_t __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));

constexpr int kSplit = 256;  // slots of a workgroup
constexpr int kQ = 16;       // query heads of a workgroup: the columns of its products
// Caches of more bytes are read with non-temporal loads: half of the last-level
// cache, which holds a smaller one from one call to the next where nothing else
// comes between.  (64 sequences of up to 1025 keys, 134 MB: 37.4 -> 34.2 us; 24
// of up to 8191 of half the width, 100 MB, called again and again: 24.9 -> 30.3)
// Between these two the line is not measured closely: 63 sequences of 1025 keys,
// just below it, take 39.7 us over three caches in turn, 64 above it 37.0.
constexpr int64_t kKeptBytes = 128 << 20;
constexpr int kJoin = 8;     // query heads that the wavefronts' outputs are joined for at a time

struct AttendArgs {
    KvView c;
    const void *q, *k_new, *v_new, *gate;
    const int32_t *pos_new, *lens;
    const uint8_t *mask;
    void *out;
    float *lse, *weight;
    int32_t *pos;
    float *part;   // [seqs][n_head][n_split][d]: the splits' outputs, not normalised
    float2 *ml;    // [seqs][n_head][n_split]: their maxima (of scores times log2 e) and sums
    float *score;  // [seqs][n_head][s_stride]: scores times log2 e, where there is a history
    int64_t q_stride, new_stride, mask_stride, out_stride, s_stride;
    int32_t n_head, max_len, h_heads, h_slots, n_split, q_tiles;
    float scale;
    int32_t w_slots;  // slots of a workgroup that adds weights: 512 or 256
};
// passed by value to kernels: the host and device passes must lay it out alike
static_assert(sizeof(AttendArgs) == 256, "AttendArgs: kernel argument layout");

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
// Eight (N = 8) or four adjacent values of a row, from 16-byte aligned rows.
template <int N, typename T>
__device__ __forceinline__ void load_row(const T *p, float (&x)[N]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const f32x4_t v = *reinterpret_cast<const f32x4_t *>(p + i);
#pragma unroll
            for (int e = 0; e < 4; ++e) x[i + e] = v[e];
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const u32x2_t v = *reinterpret_cast<const u32x2_t *>(p + i);
            x[i] = __uint_as_float(v[0] << 16), x[i + 1] = __uint_as_float(v[0] & 0xffff0000u);
            x[i + 2] = __uint_as_float(v[1] << 16), x[i + 3] = __uint_as_float(v[1] & 0xffff0000u);
        }
    }
}
// Two floats as bf16, rounded to nearest even, in one dword.
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2_t{a, b}, bf16x2_t));
}
// Two bf16 with infinities and NaN as the largest finite value of their sign:
// by their bits, positive ones order as signed numbers and negative ones as
// unsigned.
__device__ __forceinline__ uint32_t finite_bf16(uint32_t w) {
    const i16x2_t pos = __builtin_elementwise_min(__builtin_bit_cast(i16x2_t, w), i16x2_t(0x7f7f));
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_min(__builtin_bit_cast(u16x2_t, pos), u16x2_t(0xff7f)));
}
// x as a sum of N bf16 operands, each the rounding of what the ones before
// leave (the differences are exact): 8 bits of the significand apiece, so three
// hold a float whole.
template <int N, int M>
__device__ __forceinline__ void split(const float (&x)[M], uint32_t (&w)[N][M / 2]) {
    float r[M];
#pragma unroll
    for (int i = 0; i < M; ++i) r[i] = x[i];
#pragma unroll
    for (int k = 0; k < N; ++k)
#pragma unroll
        for (int i = 0; i < M / 2; ++i) {
            w[k][i] = pack_bf16(r[2 * i], r[2 * i + 1]);
            if (k + 1 < N) {
                r[2 * i] -= __uint_as_float(w[k][i] << 16);
                r[2 * i + 1] -= __uint_as_float(w[k][i] & 0xffff0000u);
            }
        }
}
// A query's: each operand cut off instead of rounded, so that the first is
// infinite only where x is, and a finite x is finite whole; a NaN stays one.
template <int N>
__device__ __forceinline__ void split_query(const float (&x)[8], bf16x8_t (&s)[N]) {
    uint32_t w[N][4];
    float r[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = __builtin_canonicalizef(x[i]);  // a NaN with a top bit of its significand set
#pragma unroll
    for (int k = 0; k < N; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            w[k][i] = __builtin_amdgcn_perm(__float_as_uint(r[2 * i + 1]), __float_as_uint(r[2 * i]), 0x07060302u);
            if (k + 1 < N) {
                r[2 * i] -= __uint_as_float(__float_as_uint(r[2 * i]) & 0xffff0000u);
                r[2 * i + 1] -= __uint_as_float(__float_as_uint(r[2 * i + 1]) & 0xffff0000u);
            }
        }
#pragma unroll
    for (int k = 0; k < N; ++k) s[k] = __builtin_bit_cast(bf16x8_t, u32x4_t{w[k][0], w[k][1], w[k][2], w[k][3]});
}
template <int N>
__device__ __forceinline__ void split4(const float (&x)[4], bf16x4_t (&s)[N]) {
    uint32_t w[N][2];
    split<N>(x, w);
#pragma unroll
    for (int k = 0; k < N; ++k) s[k] = __builtin_bit_cast(bf16x4_t, u32x2_t{w[k][0], w[k][1]});
}
// Maximum and sum over the four lanes l, l + 16, l + 32, l + 48.
__device__ __forceinline__ float quad_max(float v) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float quad_sum(float v) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

__device__ __forceinline__ int slots_of(const AttendArgs &a, int64_t b) { return max(0, min(a.lens[b], a.max_len)); }
__device__ __forceinline__ float sigmoid(float x) { return 1.0f / (1.0f + expf(-x)); }

// A load of the cache: Once = non-temporal, for caches that no cache of the
// chip holds until the next call.
template <bool Once, typename T>
__device__ __forceinline__ T load_cache(const T *p) {
    if constexpr (Once) return __builtin_nontemporal_load(p);
    return *p;
}

// x, as a value that is made where this stands: what is computed from it stays
// in the loop instead of being kept in registers throughout it.  The asm holds no
// instruction, so that no wait state is owed around it.
__device__ __forceinline__ int in_loop(int x) {
    asm volatile("" : "+v"(x));
    return x;
}

// A head's joined output (normalised), through the gate to its place.
template <typename IO>
__device__ __forceinline__ void store_out(const AttendArgs &a, int64_t b, int h, int dim, float o) {
    const int64_t i = static_cast<int64_t>(h) * a.c.d + dim;
    if (a.gate) o *= sigmoid(load1(static_cast<const IO *>(a.gate), b * a.q_stride + i));
    store1(static_cast<IO *>(a.out), b * a.out_stride + i, o);
}
__device__ __forceinline__ void store_lse(const AttendArgs &a, int64_t b, int h, float m, float l) {
    if (a.lse) a.lse[b * a.n_head + h] = (m + log2f(l)) * 0.6931471805599453f;  // -inf where l = 0
}

// One workgroup a split of kSplit slots, (kv head, tile of 16 query heads) and
// sequence, its four wavefronts on alternate tiles of 16 slots, each with its
// own running maximum, sum and output.
//
// Both products run on the matrix cores with the slots as rows of the first
// and as the inner axis of the second, the query heads as columns:
//   S^T[slot][head] = K Q^T, O^T[dim][head] += V^T P^T.
// A lane of S^T holds one head (lane % 16) and slots 4 (lane / 16) + 0 .. 3 of
// the tile, and that is the order in which V's rows are loaded, so the scores
// become the second product's operand without leaving their registers.  K's
// rows are read whole, 16 bytes a lane, and turned into operands through LDS.
// A bf16 row of V is loaded with eight (DP = 64: four) adjacent dims a lane,
// and pairs of rows are merged by byte permutes into operands of one dim and
// four slots; fp32 operands hold one slot and need none.
// fp32 queries and the weights against a bf16 cache are split into three bf16
// operands (exact), so that a bf16 output is rounded once, when it is stored;
// everything else is fp32.
//
// Bound by memory where the splits fill the chip: 64 sequences of 16384 keys
// (4 kv heads of 128, bf16) at 5.8 TB/s, 64 of up to 2176 in fp32 in 52.7 us
// (5.1); a kernel that only reads 4 GiB reaches 7.  Below that by what a
// workgroup does before its first products and after its last (pages, queries,
// the four outputs joined): 64 sequences of up to 1025 keys take 26.9 us, of
// which some 21 remain without reading K or V, one sequence of 16384 11.0, one of
// 300 8.0.  Splits of 256 slots because one
// sequence must fill the chip; several splits a workgroup were no faster.  The
// loads of the next tile stand before a tile's products and need no count of
// what is in flight: there is always a tile's worth.
template <typename C, typename IO, int DP, bool Paged, bool Once>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(sizeof(C) == 2 ? (DP <= 64 ? 5 : DP <= 128 ? 4 : 2) : (DP <= 64 ? 5 : DP <= 128 ? 3 : 2)))) void kv_attend_split_kernel(AttendArgs a) {
    constexpr bool kHalf = sizeof(C) == 2;
    constexpr int TS = 16;                                // slots of a tile
    constexpr int STEP = 4 * TS;                          // slots of a step of the four wavefronts
    constexpr int KC = kHalf ? 8 : 4;                     // dims of a lane's 16 bytes of K
    constexpr int NJ = DP / (4 * KC);                     // steps over the dims
    constexpr int NQ = kHalf && sizeof(IO) == 4 ? 3 : 1;  // operands of a query
    constexpr int NP = 3;                                 // and of a weight (bf16 cache); two, for bf16 rows, saved 0.15 us of 23.75
    constexpr int CH = kHalf && DP > 64 ? 8 : 4;          // adjacent dims of V a lane
    constexpr int NB = DP / (16 * CH);
    constexpr int NR = TS / 4;                            // slots of a lane
    constexpr size_t kQBytes = kHalf ? NQ * DP * 32 : DP * 64;
    constexpr int CPR = DP / KC;                          // chunks of 16 bytes of a row
    constexpr int RK = 64 / CPR;                          // rows of a load of K
    constexpr size_t kKRow = 16 * CPR + 16;               // bytes of a row of K in LDS: 16 rows start in different banks
    constexpr size_t kKBytes = 16 * kKRow;
    extern __shared__ __attribute__((aligned(16))) unsigned char lds[];  // queries | the wavefronts' rows of K, later their outputs
    __shared__ float sm[4][kQ], sl[4][kQ];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = lane & 15, g = lane >> 4;
    const int64_t b = blockIdx.z;
    const int kvh = static_cast<int>(blockIdx.y) / a.q_tiles, qt = static_cast<int>(blockIdx.y) % a.q_tiles;
    const int G = a.n_head / a.c.n_head_kv, d = a.c.d;
    const int h0 = kvh * G + qt * kQ, nq = min(kQ, G - qt * kQ);  // heads h0 .. h0 + nq - 1
    // Workgroups go round the eight XCDs, so with an even number of splits some
    // XCDs would have the low ones of every sequence and others the high ones,
    // which few sequences reach: each kv head of each sequence starts at another
    // split.  (64 sequences of 16 .. 8000 slots, 32 splits: 93.6 us, 116 without;
    // one sequence, which has work for all, 13.9 without and 14.8 with it)
    const uint32_t turn = gridDim.x & 1 || gridDim.z == 1 ? blockIdx.x : (blockIdx.x + blockIdx.y + gridDim.y * blockIdx.z) % gridDim.x;
    const int split_at = static_cast<int>(turn), j0 = split_at * kSplit;
    // Lane l of wavefront w stands for slot 16 (w + 4 (l / 16)) + l % 16 of a
    // split: the wavefront's own tiles, so that their pages and visible slots
    // stay in its registers.  They are read without waiting for the length.
    const int mine = 16 * (wave + 4 * g) + r;
    int32_t page = 0;  // held to 0 .. n_pages - 1: a hole's rows are read (of a page that is there), never used
    bool seen = false;
    if (j0 + mine < a.max_len) {
        const int32_t id = a.c.pages[b * a.c.max_pages + ((j0 + mine) >> a.c.page_shift)];
        const bool there = id >= 0 && id < a.c.n_pages;
        if (there) page = id;
        seen = there && (!a.mask || a.mask[b * a.mask_stride + j0 + mine] != 0);
    }
    const int n = slots_of(a, b);
    if (j0 >= n && j0 > 0) return;  // whole workgroup; an empty sequence's first split writes its zeros
    const int end = min(n, j0 + kSplit);  // the split's slots are j0 .. end - 1
    typedef uint32_t vch_t __attribute__((ext_vector_type(CH * sizeof(C) / 4)));
    u32x4_t kf[NJ];  // K: chunk kc of rows RK i + kr
    vch_t vf[NR][NB];
    const C *const kp = static_cast<const C *>(a.c.k) + kvh * a.c.head_stride;
    const C *const vp = static_cast<const C *>(a.c.v) + kvh * a.c.head_stride;
    // Element offset of a slot's row.  16 slots from a multiple of 16 stay in
    // their page, so that every row that is read is a row of the pool, visible
    // or not; scores and V's values of those that are not are replaced below.
    auto row_of = [&](int pg, int slot) {
        return static_cast<int64_t>(pg) * a.c.page_stride +
               static_cast<int64_t>(slot & ((1 << a.c.page_shift) - 1)) * a.c.token_stride;
    };
    // a lane's places in 16 rows, in bytes (the host checks that they fit);
    // chunks past d are read from the row's last chunk
    constexpr int kSize = sizeof(C);
    const uint32_t row_bytes = static_cast<uint32_t>(a.c.token_stride) * kSize;
    const int kr = lane / CPR, kc = lane % CPR;
    // Rows of the tile of 16 slots from `slot`, the wavefront's k-th of its
    // split; where there is none, one line over and over, so that the loads in
    // flight can be counted without knowing.
    auto load_k = [&](int slot, int k, bool there) {
        if constexpr (Paged) {
            const int64_t row = there ? row_of(__builtin_amdgcn_readlane(page, 16 * k), slot) : 0;
            const char *base = reinterpret_cast<const char *>(kp + row);
            const uint32_t step = there ? row_bytes : 0u;
            const uint32_t off = static_cast<uint32_t>(in_loop(kr)) * step + min(KC * kc, d - KC) * kSize;
#pragma unroll
            for (int i = 0; i < NJ; ++i)
                kf[i] = load_cache<Once>(reinterpret_cast<const u32x4_t *>(base + static_cast<uint64_t>(RK * i) * step + off));
        } else {
#pragma unroll
            for (int i = 0; i < NJ; ++i) {
                const int s = RK * i + kr;
                const int64_t row = there ? row_of(__shfl(page, 16 * k + s, 64), slot + s) : 0;
                kf[i] = load_cache<Once>(reinterpret_cast<const u32x4_t *>(kp + row + min(KC * kc, d - KC)));
            }
        }
    };
    auto load_v = [&](int slot, int k, bool there) {
        if constexpr (Paged) {
            const int64_t row = there ? row_of(__builtin_amdgcn_readlane(page, 16 * k), slot) : 0;
            const char *base = reinterpret_cast<const char *>(vp + row);
            const uint32_t step = there ? row_bytes : 0u;
            const uint32_t off = 4 * static_cast<uint32_t>(in_loop(g)) * step;
#pragma unroll
            for (int i = 0; i < NR; ++i)
#pragma unroll
                for (int nb = 0; nb < NB; ++nb)
                    vf[i][nb] = load_cache<Once>(reinterpret_cast<const vch_t *>(
                        base + static_cast<uint64_t>(i) * step + (off + min(16 * CH * nb + CH * r, d - CH) * kSize)));
        } else {
#pragma unroll
            for (int i = 0; i < NR; ++i) {
                const int64_t row = there ? row_of(__shfl(page, 16 * k + 4 * g + i, 64), slot + 4 * g + i) : 0;
#pragma unroll
                for (int nb = 0; nb < NB; ++nb)
                    vf[i][nb] = load_cache<Once>(reinterpret_cast<const vch_t *>(vp + row + min(16 * CH * nb + CH * r, d - CH)));
            }
        }
    };
    const uint64_t bits = __ballot(seen && j0 + mine < n);  // visible slots: 16 of each of the wavefront's tiles
    load_k(j0 + TS * wave, 0, j0 + TS * wave < end);
    load_v(j0 + TS * wave, 0, j0 + TS * wave < end);
    const int fresh = a.k_new && n <= end ? n - 1 : -1;  // the new token's slot, if it is in the split
    if (fresh >= 0 && qt == 0) {
        // its rows into the cache; this launch takes them from k_new and v_new
        const int64_t to = kv_slot(a.c, b, n - 1);
        if (tid < d && to >= 0) {
            const int64_t src = b * a.new_stride + static_cast<int64_t>(kvh) * d + tid, dst = to + kvh * a.c.head_stride + tid;
            store1(static_cast<C *>(a.c.k), dst, load1(static_cast<const IO *>(a.k_new), src));
            store1(static_cast<C *>(a.c.v), dst, load1(static_cast<const IO *>(a.v_new), src));
        }
        if (a.weight && kvh < a.h_heads && tid == 0) {
            const int64_t i = (b * a.h_heads + kvh) * a.h_slots + n - 1;
            a.weight[i] = 0.f;
            a.pos[i] = a.pos_new[b];
        }
    }
    // the queries as second operands: head r, dims 4 KC j + KC g .. of step j
    for (int i = tid; i < NJ * 64; i += 256) {
        const int jr = i & 15, dim = (i >> 6) * (4 * KC) + ((i >> 4) & 3) * KC;
        float x[KC];
#pragma unroll
        for (int e = 0; e < KC; ++e) x[e] = 0.f;
        if (jr < nq && dim < d) load_row<KC>(static_cast<const IO *>(a.q) + b * a.q_stride + static_cast<int64_t>(h0 + jr) * d + dim, x);
        if constexpr (kHalf) {
            bf16x8_t s[NQ];
            split_query<NQ>(x, s);
#pragma unroll
            for (int k = 0; k < NQ; ++k) reinterpret_cast<bf16x8_t *>(lds)[k * NJ * 64 + i] = s[k];
        } else {
            reinterpret_cast<f32x4_t *>(lds)[i] = f32x4_t{x[0], x[1], x[2], x[3]};
        }
    }
    __syncthreads();

    f32x4_t o[NB][CH];  // o[nb][e][i]: dim 16 CH nb + CH (4 g + i) + e of head r
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int e = 0; e < CH; ++e) o[nb][e] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.f;
    const float sl2 = a.scale * 1.4426950408889634f;
    // the new token's rows, as the cache stores them, over what was loaded of its slot
    auto fresh_rows = [&](int slot) {
#pragma unroll
        for (int i = 0; i < NJ; ++i)
            if (slot + RK * i + kr == fresh) {
                float x[KC];
                load_row<KC>(static_cast<const IO *>(a.k_new) + b * a.new_stride + static_cast<int64_t>(kvh) * d + min(KC * in_loop(kc), d - KC), x);
#pragma unroll
                for (int w = 0; w < 4; ++w)
                    if constexpr (kHalf)
                        kf[i][w] = pack_bf16(x[2 * w], x[2 * w + 1]);
                    else
                        kf[i][w] = __float_as_uint(x[w]);
            }
#pragma unroll
        for (int i = 0; i < NR; ++i)
            if (slot + 4 * g + i == fresh) {
                const IO *row = static_cast<const IO *>(a.v_new) + b * a.new_stride + static_cast<int64_t>(kvh) * d;
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) {
                    float x[CH];
                    load_row<CH>(row + min(16 * CH * nb + CH * in_loop(r), d - CH), x);
#pragma unroll
                    for (int w = 0; w < static_cast<int>(CH * sizeof(C) / 4); ++w)
                        if constexpr (kHalf)
                            vf[i][nb][w] = pack_bf16(x[2 * w], x[2 * w + 1]);
                        else
                            vf[i][nb][w] = __float_as_uint(x[w]);
                }
            }
    };
    // K's rows to LDS, from where they are read as operands; dims past d of a
    // row count as 0, whatever stands there.
    unsigned char *const kw = lds + kQBytes + wave * kKBytes;
    auto stage_k = [&] {
#pragma unroll
        for (int i = 0; i < NJ; ++i) {
            u32x4_t x = kf[i];
            if (KC * kc >= d) x = u32x4_t{0, 0, 0, 0};
            *reinterpret_cast<u32x4_t *>(kw + (RK * i + kr) * kKRow + 16 * kc) = x;
        }
    };
    // The tile of 16 slots from `slot`, of which `now` are visible, into the
    // running maximum, sum and output of head r; maximum and scores in base 2.
    auto products = [&](int slot, uint32_t now) {
        // sc[e]: score of slot 4 g + e against head r, by as many chains as a query has operands
        f32x4_t part[NQ];
#pragma unroll
        for (int k = 0; k < NQ; ++k) part[k] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            const u32x4_t kx = *reinterpret_cast<const u32x4_t *>(kw + r * kKRow + 64 * j + 16 * g);
            if constexpr (kHalf) {
#pragma unroll
                for (int k = 0; k < NQ; ++k)
                    part[k] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, kx),
                                                                      reinterpret_cast<const bf16x8_t *>(lds)[(k * NJ + j) * 64 + lane], part[k], 0, 0, 0);
            } else {
                const f32x4_t q = reinterpret_cast<const f32x4_t *>(lds)[j * 64 + lane];
#pragma unroll
                for (int e = 0; e < 4; ++e) part[0] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(kx[e]), q[e], part[0], 0, 0, 0);
            }
        }
        f32x4_t sc = part[NQ - 1];  // the smallest first
#pragma unroll
        for (int k = NQ - 2; k >= 0; --k) sc += part[k];
        // Where a key or a query is infinite or NaN the first operands alone say
        // what the score is: they have the queries' signs and zeros, and the
        // others, of either sign or 0, would make an infinity NaN.
        if constexpr (NQ > 1) {
#pragma unroll
            for (int i = 0; i < NR; ++i) sc[i] = fabsf(part[0][i]) < INFINITY ? sc[i] : part[0][i];
        }
        sc *= sl2;
        if (now != 0xffffu) {
#pragma unroll
            for (int i = 0; i < NR; ++i)
                if (!((now >> (4 * g + i)) & 1)) {
                    sc[i] = -INFINITY;
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb) vf[i][nb] = vch_t(0);
                }
        }
        if (a.score && r < nq)
            *reinterpret_cast<f32x4_t *>(a.score + (b * a.n_head + h0 + in_loop(r)) * a.s_stride + slot + 4 * g) = sc;
        const float mn = fmaxf(m, quad_max(fmaxf(fmaxf(sc[0], sc[1]), fmaxf(sc[2], sc[3]))));
        const float mref = mn == -INFINITY ? 0.f : mn;  // no finite score yet: avoid inf - inf
        const float corr = __builtin_amdgcn_exp2f(m - mref);
        m = mn;
        float ps = 0.f, p[NR];
#pragma unroll
        for (int i = 0; i < NR; ++i) {
            p[i] = __builtin_amdgcn_exp2f(sc[i] - mref);
            ps += p[i];
        }
        l = l * corr + quad_sum(ps);
        if (!__all(corr == 1.0f)) {
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                for (int e = 0; e < CH; ++e) o[nb][e] *= corr;
        }
        if constexpr (kHalf) {
            bf16x4_t pf[NP];
            split4<NP>(p, pf);
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                for (int e0 = 0; e0 < CH; e0 += 4) {  // four dims' chains at a time
                    u32x2_t w[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e)
#pragma unroll
                        for (int i = 0; i < 2; ++i)
                            w[e][i] = __builtin_amdgcn_perm(vf[2 * i + 1][nb][(e0 + e) >> 1], vf[2 * i][nb][(e0 + e) >> 1],
                                                            e & 1 ? 0x07060302u : 0x05040100u);
#pragma unroll
                    for (int k = 0; k < NP; ++k) {
                        // a value that is not finite counts by its weight's first
                        // operand: the others, 0 or negative, would make an infinity NaN
                        if (k == 1)
#pragma unroll
                            for (int e = 0; e < 4; ++e) w[e] = u32x2_t{finite_bf16(w[e][0]), finite_bf16(w[e][1])};
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            o[nb][e0 + e] = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(bf16x4_t, w[e]), pf[k], o[nb][e0 + e], 0, 0, 0);
                    }
                }
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        o[nb][e] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(vf[i][nb][e]), p[i], o[nb][e], 0, 0, 0);
        }
    };
    constexpr int OS = DP + 4;  // floats of an output row: padded, so that the heads' rows start in different banks
    float *const ob = reinterpret_cast<float *>(lds + kQBytes);
    const bool whole = n <= kSplit;  // the sequence's only split
    for (int k = 0; k < 4; ++k) {
        const int slot = j0 + TS * wave + STEP * k;
        if (fresh >= slot && fresh < slot + TS) fresh_rows(slot);
        stage_k();
        const bool next = k < 3 && slot + STEP < end;
        load_k(slot + STEP, k + 1, next);
        if (slot < end) products(slot, static_cast<uint32_t>(bits >> (16 * k)) & 0xffffu);
        load_v(slot + STEP, k + 1, next);
    }
    // the four wavefronts' outputs joined, kJoin heads at a time
    if (g == 0) sm[wave][r] = m, sl[wave][r] = l;
    for (int q0 = 0; q0 < nq; q0 += kJoin) {
        __syncthreads();  // K's rows, or the heads before, have been read
        if (r >= q0 && r < min(nq, q0 + kJoin)) {
            float *row = ob + (wave * kJoin + r - q0) * OS + 4 * g;
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                for (int e = 0; e < CH; ++e) *reinterpret_cast<f32x4_t *>(row + 16 * (CH * nb + e)) = o[nb][e];
        }
        __syncthreads();
        const int dim = tid % DP;
        const int place = dim / (16 * CH) * (16 * CH) + dim % CH * 16 + dim % (16 * CH) / CH;  // of dim in a row of ob
        for (int q = q0 + tid / DP; q < min(nq, q0 + kJoin); q += 256 / DP) {
            const float M = fmaxf(fmaxf(sm[0][q], sm[1][q]), fmaxf(sm[2][q], sm[3][q]));
            float L = 0.f, x = 0.f;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const float f = __builtin_amdgcn_exp2f(sm[w][q] - (M == -INFINITY ? 0.f : M));
                L += f * sl[w][q];
                x += f * ob[(w * kJoin + q - q0) * OS + place];
            }
            if (dim >= d) continue;
            const int64_t rec = (b * a.n_head + h0 + q) * a.n_split + split_at;
            if (dim == 0 && a.ml) a.ml[rec] = make_float2(M, L);
            if (whole) {
                store_out<IO>(a, b, h0 + q, dim, L == 0.f ? 0.f : x / L);
                if (dim == 0) store_lse(a, b, h0 + q, M, L);
            } else {
                a.part[rec * d + dim] = x;
            }
        }
    }
}

// Maximum and sum of a head over its splits, by N lanes of a wavefront, to each
// of them.
template <int N>
__device__ __forceinline__ float2 join_ml(const float2 *ml, int ns) {
    float M = -INFINITY, L = 0.f;
    for (int s = threadIdx.x % N; s < ns; s += N) {
        const float2 x = ml[s];
        const float mn = fmaxf(M, x.x), ref = mn == -INFINITY ? 0.f : mn;
        L = L * __builtin_amdgcn_exp2f(M - ref) + x.y * __builtin_amdgcn_exp2f(x.x - ref);
        M = mn;
    }
#pragma unroll
    for (int off = N / 2; off >= 1; off >>= 1) {
        const float m2 = xor_shfl(M, off), l2 = xor_shfl(L, off), mn = fmaxf(M, m2);
        const float ref = mn == -INFINITY ? 0.f : mn;
        L = L * __builtin_amdgcn_exp2f(M - ref) + l2 * __builtin_amdgcn_exp2f(m2 - ref);
        M = mn;
    }
    return make_float2(M, L);
}

// The splits of (head, sequence) joined: a thread takes four dims of every
// (1024 / DP)-th split.  Latency: 2.5 to 4 us a launch for 2 to 64 splits.
template <typename IO, int DP>
__device__ __forceinline__ void join_splits(const AttendArgs &a, int64_t b, int h, int ns, f32x4_t *red) {
    const int tid = threadIdx.x, d = a.c.d;
    constexpr int DL = DP / 4, NG = 256 / DL;
    const int64_t rec = (b * a.n_head + h) * a.n_split;
    const int dim = 4 * (tid % DL), s0 = tid / DL;
    // the first kAhead splits' outputs are on their way while the maxima are joined
    constexpr int kAhead = 4;
    f32x4_t first[kAhead];
    float fm[kAhead];
    const bool in = dim < d;
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
        const int s = min(s0 + i * NG, ns - 1);
        fm[i] = a.ml[rec + s].x;
        first[i] = *reinterpret_cast<const f32x4_t *>(a.part + (rec + s) * d + (in ? dim : 0));
    }
    const float2 t = join_ml<64>(a.ml + rec, ns);
    const float ref = t.x == -INFINITY ? 0.f : t.x;
    f32x4_t x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
        if (s0 + i * NG < ns) x += __builtin_amdgcn_exp2f(fm[i] - ref) * first[i];
    if (in)
        for (int s = s0 + kAhead * NG; s < ns; s += NG)
            x += __builtin_amdgcn_exp2f(a.ml[rec + s].x - ref) * *reinterpret_cast<const f32x4_t *>(a.part + (rec + s) * d + dim);
    red[tid] = x;
    __syncthreads();
    if (tid >= DP) return;
    float o = 0.f;
#pragma unroll
    for (int s = 0; s < NG; ++s) o += red[s * DL + tid / 4][tid % 4];
    if (tid < d) store_out<IO>(a, b, h, tid, t.y == 0.f ? 0.f : o / t.y);
    if (tid == 0) store_lse(a, b, h, t.x, t.y);
}

// Each slot's attention weight, summed over the query heads of its history
// head, onto the history: by the scores that the splits left and the heads'
// joined maxima and sums.  NW slots a thread.
constexpr int kWHeads = 64;
template <int NW>
__device__ __forceinline__ void add_weights(const AttendArgs &a, int64_t b, int hs, int j0, int n, float2 *ml) {
    const int tid = threadIdx.x;
    const int ns = (n + kSplit - 1) / kSplit, G = a.n_head / a.h_heads;
    float *const out = a.weight + (b * a.h_heads + hs) * a.h_slots;
    float w[NW], sum[NW];
#pragma unroll
    for (int i = 0; i < NW; ++i) {
        const int j = j0 + 256 * i + tid;
        w[i] = j < n ? out[j] : 0.f;
        sum[i] = 0.f;
    }
    for (int g0 = 0; g0 < G; g0 += kWHeads) {
        const int ng = min(kWHeads, G - g0);
        const int64_t h0 = b * a.n_head + static_cast<int64_t>(hs) * G + g0;
        // the first heads' scores are on their way while the maxima are joined
        constexpr int kAhead = 4;
        float first[kAhead][NW];
#pragma unroll
        for (int k = 0; k < kAhead; ++k)
            if (k < ng)
#pragma unroll
                for (int i = 0; i < NW; ++i) first[k][i] = a.score[(h0 + k) * a.s_stride + min(j0 + 256 * i + tid, n - 1)];
        __syncthreads();
        for (int i = tid >> 4; i < ng; i += 16) {
            const float2 t = join_ml<16>(a.ml + (h0 + i) * a.n_split, ns);
            if (tid % 16 == 0) ml[i] = make_float2(t.x == -INFINITY ? 0.f : t.x, 1.0f / t.y);  // no -inf - -inf
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < NW; ++i) {
            const int j = j0 + 256 * i + tid;
            // a slot that is not visible has a score of -inf, and takes nothing
            // even of a head whose sum is NaN (or 0: nothing visible)
            auto add = [&](float s, float2 h) { sum[i] += __builtin_amdgcn_exp2f(s - h.x) * (s == -INFINITY ? 0.f : h.y); };
#pragma unroll
            for (int k = 0; k < kAhead; ++k)
                if (k < ng) add(first[k][i], ml[k]);
            if (j < n)
#pragma unroll 8
                for (int k = kAhead; k < ng; ++k) add(a.score[(h0 + k) * a.s_stride + j], ml[k]);
        }
    }
#pragma unroll
    for (int i = 0; i < NW; ++i) {
        const int j = j0 + 256 * i + tid;
        if (j < n) out[j] = w[i] + sum[i];
    }
}

// What the splits left brought together: workgroups 0 .. joins - 1 of a
// sequence take a head's output each, the others w_slots slots of a history
// head: 512, so that few workgroups repeat the heads' maxima, or 256 where a
// slot's weight takes the scores of many heads (24 sequences of up to 8191
// slots: 32 heads 27.0 us with 512 and 25.5 with 256, 64 of up to 1025 with 4
// heads 32.5 and 33.1; between them, where the line is drawn, nothing is measured).
template <typename IO, int DP>
__global__ __launch_bounds__(256) void kv_attend_join_kernel(AttendArgs a, int joins) {
    __shared__ f32x4_t red[256];
    const int64_t b = blockIdx.y;
    // turned by the sequence, as the splits are: 24.0 us instead of 24.6 for the 24
    const int x = static_cast<int>((blockIdx.x + blockIdx.y) % gridDim.x), n = slots_of(a, b);
    if (x < joins) {
        if (n > kSplit) join_splits<IO, DP>(a, b, x, (n + kSplit - 1) / kSplit, red);  // else its only split wrote it
    } else {
        const int hs = (x - joins) % a.h_heads, j0 = (x - joins) / a.h_heads * a.w_slots;
        if (j0 >= n) return;
        if (a.w_slots == 256)
            add_weights<1>(a, b, hs, j0, n, reinterpret_cast<float2 *>(red));
        else
            add_weights<2>(a, b, hs, j0, n, reinterpret_cast<float2 *>(red));
    }
}

template <typename C, typename IO, int DP>
int launch_attend(const AttendArgs &a, unsigned seqs, hipStream_t s) {
    constexpr bool kHalf = sizeof(C) == 2;
    constexpr size_t q_bytes = kHalf ? (sizeof(IO) == 4 ? 3 : 1) * DP * 32 : DP * 64;
    constexpr size_t o_bytes = 4 * kJoin * (DP + 4) * sizeof(float), k_bytes = 4 * 16 * (DP * sizeof(C) + 16);
    constexpr size_t lds = q_bytes + (o_bytes > k_bytes ? o_bytes : k_bytes);
    const dim3 grid(a.n_split, a.c.n_head_kv * a.q_tiles, seqs);
    const int64_t bytes = static_cast<int64_t>(seqs) * a.max_len * a.c.n_head_kv * a.c.d * 2 * sizeof(C);
    const int which = (a.c.page_shift >= 4 ? 2 : 0) + (bytes > kKeptBytes);
    using Kernel = void (*)(AttendArgs);
    static const Kernel kernels[4] = {kv_attend_split_kernel<C, IO, DP, false, false>, kv_attend_split_kernel<C, IO, DP, false, true>,
                                      kv_attend_split_kernel<C, IO, DP, true, false>, kv_attend_split_kernel<C, IO, DP, true, true>};
    if (lds + 1024 > 65536) {  // one opt-in per kernel and device for more than 64 KiB of LDS (idempotent)
        static std::atomic<uint64_t> done[4];
        const int dev = current_device();
        const uint64_t bit = dev >= 0 && dev < 64 ? uint64_t{1} << dev : 0;
        if (!(done[which].load(std::memory_order_acquire) & bit)) {
            const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(kernels[which]),
                                                     hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(lds));
            if (e != hipSuccess) return fail(OURO_ERR_HIP, "ouro_kv_attend: LDS opt-in: %s", hipGetErrorString(e));
            done[which].fetch_or(bit, std::memory_order_release);
        }
    }
    hipLaunchKernelGGL(kernels[which], grid, dim3(256), lds, s, a);
    int st = check_launch("kv_attend_split_kernel");
    if (st) return st;
    const int joins = a.n_split > 1 ? a.n_head : 0;
    const int64_t weights = a.weight ? static_cast<int64_t>((a.max_len + a.w_slots - 1) / a.w_slots) * a.h_heads : 0;
    if (joins + weights > 0) {
        hipLaunchKernelGGL((kv_attend_join_kernel<IO, DP>), dim3(static_cast<unsigned>(joins + weights), seqs), dim3(256), 0, s, a, joins);
        st = check_launch("kv_attend_join_kernel");
    }
    return st;
}
template <typename C, typename IO>
int launch_attend(const AttendArgs &a, unsigned seqs, hipStream_t s) {
    if (a.c.d <= 64) return launch_attend<C, IO, 64>(a, seqs, s);
    if (a.c.d <= 128) return launch_attend<C, IO, 128>(a, seqs, s);
    return launch_attend<C, IO, 256>(a, seqs, s);
}

// The workspace: the splits' maxima and sums, their outputs, the scores.
struct AttendWs {
    size_t ml, part, score, bytes;
    int n_split;
    int64_t s_stride;
};
AttendWs attend_ws(size_t seqs, size_t n_head, size_t d, size_t max_len, bool history) {
    AttendWs w{};
    const size_t rows = seqs * n_head, ns = max_len ? (max_len + kSplit - 1) / kSplit : 1;
    auto up = [](size_t x) { return (x + 255) & ~size_t{255}; };
    w.n_split = static_cast<int>(ns);
    w.s_stride = static_cast<int64_t>((max_len + 31) / 32 * 32);  // whole tiles are stored
    w.part = ns > 1 || history ? up(rows * ns * sizeof(float2)) : 0;
    w.score = w.part + (ns > 1 ? up(rows * ns * d * sizeof(float)) : 0);
    w.bytes = w.score + (history ? up(rows * w.s_stride * sizeof(float)) : 0);
    return w;
}

}  // namespace
}  // namespace ouro

using namespace ouro;

extern "C" {

size_t ouro_kv_attend_workspace_bytes(size_t seqs, size_t n_head, size_t head_dim, size_t max_len, int with_history) {
    return attend_ws(seqs, n_head, head_dim, max_len, with_history != 0).bytes;
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
        a.w_slots = n_head / history->heads > 8 ? 256 : 512;
    }
    if (!seqs) return OURO_OK;
    if (!max_len) a.weight = nullptr;  // no slots to weigh
    const AttendWs w = attend_ws(seqs, n_head, d, max_len, history != nullptr);
    if (w.bytes) {
        if (!ws && !(ws = workspace(w.bytes, stream))) return OURO_ERR_HIP;
        unsigned char *p = static_cast<unsigned char *>(ws);
        a.ml = reinterpret_cast<float2 *>(p);
        if (w.n_split > 1) a.part = reinterpret_cast<float *>(p + w.part);
        if (history) a.score = reinterpret_cast<float *>(p + w.score);
    }
    a.s_stride = w.s_stride;
    a.n_split = w.n_split;
    a.q_tiles = static_cast<int>((n_head / hkv + kQ - 1) / kQ);
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
