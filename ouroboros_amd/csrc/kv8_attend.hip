// kv8_attend.hip - attention of each sequence's newest rows over a paged cache
// of 8-bit codes with a scale for each block of slots and kv head.
//
// For query head h of the row in slot r, over its visible slots j:
//   s_j = scale q.k_j,  m = max s_j,  l = sum e^(s_j - m),
//   o = (1 / l) sum e^(s_j - m) v_j  [* sigmoid(gate)],  lse = m + ln l,
// and o = 0, lse = -inf where no slot is visible.  Scores are fp32: one of +inf makes o
// and lse NaN, one of -inf weighs nothing.
#include "kv_cache.hpp"

#include <atomic>
#include <cmath>
#include <type_traits>

namespace ouro {
namespace {

typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef float f32x2_t __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef int i32x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));

constexpr int kTurn = 256;  // slots that a workgroup's four wavefronts take in turn: 2 tiles of 32 each

struct Attend8Args {
    Kv8View c;
    NewRows r;
    const void *q, *gate;
    const uint8_t *mask;
    void *out;
    float *lse;
    float *part;  // [records][n_head][n_split][d]: the splits' outputs, averages by their own sums
    float2 *ml;   // [records][n_head][n_split]: their maxima (of scores times log2 e) and sums
    int64_t q_stride, mask_stride, out_stride;
    int32_t n_head, window, sinks;  // window 2^30: every slot
    float scale;
    int32_t n_split, turns;  // turns of a split
    int32_t by_seq;          // records: max_new of each sequence, or else one of each packed row
};
static_assert(sizeof(Attend8Args) == 232, "Attend8Args: kernel argument layout");

// What a packed row of sequence b is off from its record.
__device__ __forceinline__ int64_t record_shift(const Attend8Args &a, int64_t b, const SeqRows &s) {
    return a.by_seq ? b * a.r.max_new - s.first : 0;
}

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
// Sixteen adjacent values of a row.
template <typename T>
__device__ __forceinline__ void load16(const T *p, float (&x)[16]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const f32x4_t v = reinterpret_cast<const f32x4_t *>(p)[i];
#pragma unroll
            for (int e = 0; e < 4; ++e) x[4 * i + e] = v[e];
        }
    } else {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const u32x4_t v = reinterpret_cast<const u32x4_t *>(p)[i];
#pragma unroll
            for (int e = 0; e < 8; ++e) x[8 * i + e] = __uint_as_float(e & 1 ? v[e / 2] & 0xffff0000u : v[e / 2] << 16);
        }
    }
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
__device__ __forceinline__ float lane_float(float v, int lane) {
    return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), lane));
}
// Two codes of a byte pair each (code + 128 in the low bytes) as fp16 times 2^-9:
// (c + 128) 2^-24 2^15 - 128 2^-9 = c 2^-9, exact.
__device__ __forceinline__ uint32_t codes_f16(uint32_t two) {
    const f16x2_t c = __builtin_elementwise_fma(__builtin_bit_cast(f16x2_t, two), f16x2_t{32768.f16, 32768.f16}, f16x2_t{-0.25f16, -0.25f16});
    return __builtin_bit_cast(uint32_t, c);
}

// N adjacent dwords of a row of codes, at a multiple of 4 bytes for N = 3 (12 dims a
// lane), of 4 N else.  A vector of three is no type to read them by: it has the size
// and the alignment of four, so that the last lane of a pool's last row could read 4
// bytes past its end.
template <int N>
struct Dwords {
    uint32_t w[N];
};
template <int N>
__device__ __forceinline__ auto load_dwords(const int8_t *p) {
    typedef uint32_t vec_t __attribute__((ext_vector_type(N)));
    if constexpr (N == 3) {
        static_assert(sizeof(Dwords<3>) == 12 && alignof(Dwords<3>) == 4, "Dwords: what is read of a row");
        const Dwords<3> d = *reinterpret_cast<const Dwords<3> *>(p);
        return vec_t{d.w[0], d.w[1], d.w[2]};
    } else {
        static_assert(sizeof(vec_t) == 4 * N, "Dwords: what is read of a row");
        return *reinterpret_cast<const vec_t *>(p);
    }
}
// x, as a value that is made where this stands: what is read by it stays in the
// loop.  The asm holds no instruction, so that no wait state is owed around it.
__device__ __forceinline__ int in_loop(int x) {
    asm volatile("" : "+v"(x));
    return x;
}

// A row's weights against V, e^(s - m) times the scale of the slot's block, are held in
// fp16 against a bound of the largest so far, z its log2: it is no more than the largest
// scale of what the row itself sees, and at most kHead above the largest such weight, so
// that neither a block that another row sees nor one of a large scale and little weight
// takes their bits.  They are taken times 2^unit, to kFull at most.
constexpr float kNoWeight = -112.f, kHead = 8.f, kFull = 32768.f;
constexpr float kLow = 130.f;  // kFull / 2^kHead, and a little
__device__ __forceinline__ int unit_of(float z) { return 15 - static_cast<int>(ceilf(z)); }
__device__ __forceinline__ int unit_of_scale(float unit_scale) { return __builtin_amdgcn_frexp_expf(unit_scale) - 1; }
// A scale times 2^unit where that is past fp32, which it can be only of slots whose
// weights are below kFull / 2^127: what those are short of then is less than they are,
// and a weight of 0 stays one.
__device__ __forceinline__ float no_infinity(float f) { return f > 3.4028234663852886e38f ? 3.4028234663852886e38f : f; }

// A tile of 32 slots of the row that a lane has: slots 4 g + i and 16 + 4 g + i of it are
// s[0][i] and s[1][i].  Those that the row does not see score -inf from here on: of the
// tile's slots `now`, it sees them up to `last`, but for what lies between `sinks` and the
// window (all of them counted from the lane's first, j + 4 g).
__device__ __forceinline__ void hide_unseen(f32x4_t (&s)[2], uint32_t now, int last, int window, int sinks) {
    // the lowest n of 32 bits
    auto below = [](int n) { return n >= 32 ? 0xffffffffu : (1u << max(n, 0)) - 1u; };
    const uint32_t seen = now & below(last + 1) & (~below(last - window + 1) | below(sinks));
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t keep = static_cast<uint32_t>(__builtin_amdgcn_sbfe(static_cast<int>(seen), 16 * u + i, 1));  // all ones or none
            s[u][i] = __uint_as_float((keep & __float_as_uint(s[u][i])) | (~keep & 0xff800000u));
        }
}

// What a wavefront keeps of its N tiles of 16 rows, a lane of row r of each.
template <int N, int CH>
struct Rows {
    f32x4_t o[N][CH];             // o[t][e][i]: dim CH (4 g + i) + e, times unit, of codes times 2^-9
    float m[N], l[N];             // the row's maximum and sum so far
    float z[N], unit[N];          // the bound of its weights, log2, and 2^unit_of(z)
    float held_to[N];             // and what the largest is at least, log2
    __device__ __forceinline__ Rows() {
#pragma unroll
        for (int t = 0; t < N; ++t) {
            m[t] = held_to[t] = -INFINITY, l[t] = 0.f, z[t] = kNoWeight, unit[t] = ldexpf(1.0f, unit_of(kNoWeight));
#pragma unroll
            for (int e = 0; e < CH; ++e) o[t][e] = f32x4_t{0.f, 0.f, 0.f, 0.f};
        }
    }
    // Takes in the scores s of a tile of 32 slots, whose scales of V are vs: f is what its
    // weights are taken by.  The references move only where some row has a larger score or
    // weight, all of a row's four lanes alike.
    __device__ __forceinline__ void take(const f32x4_t (&s)[N][2], const float (&vs)[2], float (&f)[N][2]) {
#pragma unroll
        for (int t = 0; t < N; ++t) {
            float top[2];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                top[u] = fmaxf(fmaxf(s[t][u][0], s[t][u][1]), fmaxf(s[t][u][2], s[t][u][3]));
                f[t][u] = vs[u] * unit[t];
            }
            const bool wider = !(__builtin_elementwise_maximum(f[t][0], f[t][1]) <= kFull);  // or NaN
            if (__any(wider || fmaxf(top[0], top[1]) > m[t])) move(t, top, vs, wider, f[t]);
        }
    }
    // A tile's weights of rows t as two operands, h + w.
    __device__ __forceinline__ void weigh(int t, const f32x4_t (&s)[2], const float (&f)[2], u32x4_t &h, u32x4_t &w) {
        const float ref = m[t] == -INFINITY ? 0.f : m[t];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            float p[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                p[i] = __builtin_amdgcn_exp2f(s[u][i] - ref);
                l[t] += p[i];
                p[i] *= f[u];
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const f16x2_t a = __builtin_convertvector(f32x2_t{p[2 * i], p[2 * i + 1]}, f16x2_t);
                // what a leaves, by an fma that takes it as it is: one instruction, not two
                const f16x2_t b = __builtin_convertvector(
                    f32x2_t{__builtin_fmaf(static_cast<float>(a[0]), -1.f, p[2 * i]), __builtin_fmaf(static_cast<float>(a[1]), -1.f, p[2 * i + 1])}, f16x2_t);
                h[2 * u + i] = __builtin_bit_cast(uint32_t, a);
                w[2 * u + i] = __builtin_bit_cast(uint32_t, b);
            }
        }
    }
    // Moves the references of rows t, whose largest scores in the tile are top.  A row's
    // bound rises to a larger scale that it sees, which takes one times unit above kFull,
    // and falls where a new maximum has left it more than kHead above that slot's weight,
    // which takes one below kLow.  It goes by what the row itself sees, whatever the rows
    // beside it do.
    __device__ __forceinline__ void move(int t, const float (&top)[2], const float (&vs)[2], bool wider, float (&f)[2]) {
        const float mn = fmaxf(m[t], quad_max(fmaxf(top[0], top[1]))), to = mn == -INFINITY ? 0.f : mn;  // no inf - inf
        const float back = __builtin_amdgcn_exp2f(m[t] - to);
        float by = back;
        held_to[t] += m[t] - to;
        if (__any(wider || (fminf(f[0], f[1]) < kLow && mn > m[t]))) {  // seldom
            const float lv[2] = {__builtin_amdgcn_logf(vs[0]), __builtin_amdgcn_logf(vs[1])};
            const float most = quad_max(fmaxf(top[0] - to + lv[0], top[1] - to + lv[1]));
            const float scale = quad_max(fmaxf(top[0] > -INFINITY ? lv[0] : -INFINITY, top[1] > -INFINITY ? lv[1] : -INFINITY));
            if (scale > ceilf(z[t]) + 0.01f || (mn > m[t] && z[t] > most + kHead)) {
                held_to[t] = fmaxf(held_to[t], most);
                z[t] = fmaxf(fmaxf(fmaxf(z[t] + (m[t] - to), most), fminf(fmaxf(z[t], scale), held_to[t] + kHead)), kNoWeight);
            }
            by = ldexpf(back, unit_of(z[t]) - unit_of_scale(unit[t]));
            unit[t] = ldexpf(1.0f, unit_of(z[t]));
#pragma unroll
            for (int u = 0; u < 2; ++u) f[u] = top[u] > -INFINITY ? no_infinity(vs[u] * unit[t]) : 0.f;  // whatever the scale of what is not seen
        }
        m[t] = mn;
        l[t] *= back;
#pragma unroll
        for (int e = 0; e < CH; ++e) o[t][e] *= by;
    }
};

// A head's joined output (normalised; its sum l) through the gate to its place: 0 where
// nothing was visible, whatever the gate is.
template <typename IO>
__device__ __forceinline__ void store_out(const Attend8Args &a, int64_t row, int h, int dim, float o, float l) {
    const int64_t i = static_cast<int64_t>(h) * a.c.d + dim;
    if (a.gate && l != 0.f) o *= 1.0f / (1.0f + expf(-load1(static_cast<const IO *>(a.gate), row * a.q_stride + i)));
    store1(static_cast<IO *>(a.out), row * a.out_stride + i, o);
}
__device__ __forceinline__ void store_lse(const Attend8Args &a, int64_t row, int h, float m, float l) {
    if (a.lse) a.lse[row * a.n_head + h] = (m + log2f(l)) * 0.6931471805599453f;  // -inf where l = 0
}
// Whether a row in slot `at` can see any of slots j0 .. j1 - 1.
__device__ __forceinline__ bool sees(const Attend8Args &a, int at, int j0, int j1) {
    return j0 <= at && (at + 1 - a.window < j1 || j0 < a.sinks);
}

// Of the slots j0 .. j1 - 1 of a split, seen by some of the rows in slots at_min ..
// at_max: the last that is walked through, and the first, a multiple of `step` away.
__device__ __forceinline__ int seen_end(const Attend8Args &a, int at_min, int at_max, int j1) {
    return min(at_min + 1 - a.window >= j1 ? min(j1, a.sinks) : j1, at_max + 1);
}
__device__ __forceinline__ int seen_begin(const Attend8Args &a, int at_min, int j0, int step) {
    return j0 < a.sinks ? j0 : j0 + max(at_min + 1 - a.window - j0, 0) / step * step;
}

// As many as fit 40 KiB.
constexpr int joined_rows(int dp) { return dp <= 128 ? 16 : 8; }

// One workgroup takes 16 NT rows (token by token, each token's query heads of one
// kv head) of a sequence and kv head against a split of its slots, its four
// wavefronts on alternate tiles of 32 slots, each with its own running maxima,
// sums and outputs.
//
// Both products run on the matrix cores with the slots as rows of the first and
// as the inner axis of the second, the query rows as columns:
//   S^T[slot][row] = K Q^T,  O^T[dim][row] += V^T P^T.
// K's codes are the first product's operand as they lie in the cache: the query is
// held in three signed digits of base 256 against a power of two of its row (2 U of
// the row's largest magnitude, U = 2^-24), and the digits' products with the codes
// are exact sums in 32-bit integers.  A lane then has one row and slots
// 4 (lane / 16) + 0 .. 3 of two tiles of 16, and that is the order in which V's rows
// are loaded, so the weights become the second operand without leaving their
// registers.  V's codes become fp16 by a byte permute, which puts the offset code
// of two slots into the low bytes of two fp16 as multiples of 2^-24, and one fused
// multiply-add, which takes the offset off: exact.  A weight times its slot's scale of
// V is held in two fp16 (2^-22 of it, or 2^-31 of the row's largest: 2^-25 at a power of
// two that takes 2^kHead times the largest to 2^14 .. 2^15); sums, maxima and outputs are
// fp32.
//
// Bound by memory where the splits fill the chip (128 sequences of 8192 slots, 4 kv
// heads of 128: 226 us, 4.8 TB/s), below that by what a workgroup does before its
// first products and after its last: one sequence of 300 slots takes 9 us.  Four
// wavefronts a SIMD instead of three (128 dims, 16 rows) take 18.4 us for 64 sequences
// of 1024 slots and 227 for 128 of 8192 instead of 18.2 and 226.
template <typename IO, int DP, int NT>
__global__ __launch_bounds__(256) void kv8_attend_kernel(Attend8Args a) {
    constexpr int NJ = DP / 64;                   // steps of the first product over the dims
    constexpr int CH = DP / 16;                   // adjacent dims of V a lane
    constexpr int VW = CH / 4;                    // and their dwords
    constexpr int LPR = NJ == 1 ? 4 : NJ == 2 ? 8 : 16;  // lanes that make a row's digits
    constexpr int OS = DP + 4;                    // floats of an output row in LDS: rows start in different banks
    constexpr int kJoin = joined_rows(DP);        // rows that the wavefronts' outputs are joined for at a time
    constexpr int kRows = 16 * NT;
    extern __shared__ __attribute__((aligned(16))) unsigned char lds[];  // digits [3][NT][NJ][64 lanes] of 16 bytes; later the outputs
    __shared__ float row_scale[kRows];
    __shared__ float sm[4][kRows], sl[4][kRows];
    __shared__ int su[4][kRows];                  // what brings a wavefront's outputs to the codes' size
    __shared__ int2 place[kRows];                 // packed row and head of each
    typedef uint32_t vch_t __attribute__((ext_vector_type(VW)));
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = lane & 15, g = lane >> 4;
    const int kvh = static_cast<int>(blockIdx.x) % a.c.n_head_kv;
    const int64_t b = static_cast<int64_t>(blockIdx.x) / a.c.n_head_kv;
    const int G = a.n_head / a.c.n_head_kv, d = a.c.d;
    const int split = blockIdx.z, split_first = split * a.turns * kTurn;
    // Lane l of wavefront w stands for slot 32 (w + 4 (l / 32)) + l % 32 of a turn:
    // the wavefront's own tiles, whose pages, scales and visible slots stay in its
    // registers.  A turn's page ids and mask are read without waiting for the length.
    const int mine = 32 * (wave + 4 * (lane >> 5)) + (lane & 31);
    const int32_t *const pages = a.c.pages + b * a.c.max_pages;
    int32_t id = -1;   // of the turn that is looked at next
    uint32_t kept = 1;  // and its mask byte
    auto fetch = [&](int j) {
        id = -1;
        if (j >= a.r.max_len) return;
        id = pages[j >> a.c.page_shift];
        if (a.mask) kept = a.mask[b * a.mask_stride + j];
    };
    fetch(split_first + mine);
    const SeqRows s = seq_rows(a.r, b);
    const int R = s.count * G, row0 = static_cast<int>(blockIdx.y) * kRows;
    if (row0 >= R) return;  // whole workgroup
    const int before = s.n - s.count;  // slots ahead of the new rows
    const int at_min = before + row0 / G, at_max = before + (min(row0 + kRows, R) - 1) / G;
    const int split_end = min(split_first + a.turns * kTurn, s.n);
    const bool whole = s.n <= a.turns * kTurn;  // the sequence's only split
    if (whole ? split > 0 : !sees(a, at_max, split_first, split_end) && !sees(a, at_min, split_first, split_end)) return;
    // the slots taken are first_slot .. end - 1, of those that are seen; turns behind every row's window are left out
    const int end = seen_end(a, at_min, at_max, split_end), first_slot = seen_begin(a, at_min, split_first, kTurn);
    if (first_slot != split_first) fetch(first_slot + mine);

    // The rows' queries are on their way while the cache is looked at: 16 dims a lane,
    // LPR lanes a row.
    constexpr int NI = (kRows * LPR + 255) / 256;
    float x[NI][16];
#pragma unroll
    for (int k = 0; k < NI; ++k) {
        const int i = 256 * k + tid, rho = row0 + i / LPR, ch = i % LPR;
#pragma unroll
        for (int e = 0; e < 16; ++e) x[k][e] = 0.f;
        if (i < kRows * LPR && rho < R && 16 * ch < d)
            load16(static_cast<const IO *>(a.q) + (s.first + rho / G) * a.q_stride + static_cast<int64_t>(kvh * G + rho % G) * d + 16 * ch, x[k]);
    }
    int32_t page = 0;   // held to 0 .. n_pages - 1: a hole's rows are read (of a page that is there), never used
    float k_raw = 0.f, v_raw = 0.f;
    uint64_t bits = 0;  // the turn's slots that some row sees
    auto look = [&](int j) {  // at slot j, which was fetched
        const bool there = id >= 0 && id < a.c.n_pages;
        page = there ? id : 0;
        bits = __ballot(there && kept != 0 && j < end && (j > at_min - a.window || j < a.sinks));
        // a tile of 16 slots lies in one block, whose scales all of its lanes read
        k_raw = v_raw = 0.f;
        if (static_cast<uint32_t>(bits >> (lane & 48)) & 0xffffu) {
            const int64_t i = kv8_scale(a.c, page, j & ((1 << a.c.page_shift) - 1), kvh);
            k_raw = a.c.k_scale[i];
            v_raw = a.c.v_scale[i];
        }
    };
    const int8_t *const kp = a.c.k + kvh * a.c.head_stride, *const vp = a.c.v + kvh * a.c.head_stride;
    const uint32_t row_bytes = static_cast<uint32_t>(a.c.token_stride);
    u32x4_t kf[2][NJ];  // K: slot r, dims 16 (4 j + g) .. + 15 of either tile
    vch_t vf[2][4];     // V: slot 4 g + i, dims CH r .. + CH - 1
    // 16 slots from a multiple of 16 stay in their page and block, so that every row
    // that is read is a row of the pool.  Where a tile has nothing that is seen one
    // line is read over and over, so that the loads in flight can be counted.
    auto row_of = [&](int j, int k, int u) {
        return static_cast<int64_t>(__builtin_amdgcn_readlane(page, 32 * k + 16 * u)) * a.c.page_stride +
               static_cast<int64_t>((j + 16 * u) & ((1 << a.c.page_shift) - 1)) * a.c.token_stride;
    };
    auto load_k = [&](int j, int k, bool there) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int8_t *base = kp + (there ? row_of(j, k, u) : 0);
            const uint32_t off = static_cast<uint32_t>(in_loop(r)) * (there ? row_bytes : 0u);
#pragma unroll
            for (int i = 0; i < NJ; ++i)
                kf[u][i] = *reinterpret_cast<const u32x4_t *>(base + (off + static_cast<uint32_t>(min(16 * (4 * i + g), d - 16))));
        }
    };
    auto load_v = [&](int j, int k, bool there) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int8_t *base = vp + (there ? row_of(j, k, u) : 0);
            const uint32_t step = there ? row_bytes : 0u, off = 4 * static_cast<uint32_t>(in_loop(g)) * step;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                vf[u][i] = load_dwords<VW>(base + static_cast<uint64_t>(i) * step + (off + static_cast<uint32_t>(min(CH * r, d - CH))));
        }
    };
    auto tile_bits = [&](int k) { return static_cast<uint32_t>(bits >> (32 * k)); };
    look(first_slot + mine);
    {
        const int j = first_slot + 32 * wave;
        load_k(j, 0, tile_bits(0) != 0);
        load_v(j, 0, tile_bits(0) != 0);
    }

    if (tid < kRows && row0 + tid < R) place[tid] = make_int2(s.first + (row0 + tid) / G, kvh * G + (row0 + tid) % G);
    // The rows' digits.  A negative scale goes into their sign, so that a row's
    // largest score is that of its largest sum.
    const bool negative = a.scale < 0.f;
#pragma unroll
    for (int k = 0; k < NI; ++k) {
        const int i = 256 * k + tid, row = i / LPR, ch = i % LPR;
        if (i >= kRows * LPR) break;
        uint32_t top = 0;  // magnitudes order as their bits do, NaN above infinity
#pragma unroll
        for (int e = 0; e < 16; ++e) top = max(top, __float_as_uint(x[k][e]) & 0x7fffffffu);
#pragma unroll
        for (int off = LPR / 2; off >= 1; off >>= 1) top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), off, LPR)));
        // the smallest power of two with max <= 127 65536 2^e (a row below 2^-94 takes 2^-117)
        const int ex = max(static_cast<int>(top >> 23) - ((top & 0x7fffffu) <= 0x7e0000u ? 6 : 5), 26) - 127 - 16;
        if (ch == 0) row_scale[row] = top >= 0x7f800000u ? NAN : ldexpf(fabsf(a.scale) * 1.4426950408889634f, ex);
        if (ch < 4 * NJ) {
            u32x4_t dg[3];
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                uint32_t p0 = 0, p1 = 0, p2 = 0;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    int v = static_cast<int>(rintf(ldexpf(x[k][4 * w + e], -ex)));
                    if (negative) v = -v;
                    const int c0 = static_cast<int8_t>(v), v1 = (v - c0) >> 8, c1 = static_cast<int8_t>(v1), c2 = (v1 - c1) >> 8;
                    p0 |= (static_cast<uint32_t>(c0) & 0xffu) << (8 * e);
                    p1 |= (static_cast<uint32_t>(c1) & 0xffu) << (8 * e);
                    p2 |= (static_cast<uint32_t>(c2) & 0xffu) << (8 * e);
                }
                dg[0][w] = p0, dg[1][w] = p1, dg[2][w] = p2;
            }
            const int to = ((row >> 4) * NJ + (ch >> 2)) * 64 + 16 * (ch & 3) + (row & 15);
#pragma unroll
            for (int n = 0; n < 3; ++n) reinterpret_cast<u32x4_t *>(lds)[n * NT * NJ * 64 + to] = dg[n];
        }
    }
    __syncthreads();

    Rows<NT, CH> rows;
    float qs[NT];
    int at[NT];  // the row's own slot; -1 past the last row
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int rho = row0 + 16 * t + r;
        at[t] = rho < R ? before + place[16 * t + r].x - s.first : -1;
        qs[t] = row_scale[16 * t + r];
    }
    const int turns = (end - first_slot + kTurn - 1) / kTurn;
    for (int turn = 0; turn < turns; ++turn) {
        const int t0 = first_slot + turn * kTurn;
        const float k_sc = k_raw >= 0.f && k_raw < INFINITY ? k_raw : NAN, v_sc = v_raw >= 0.f && v_raw < INFINITY ? v_raw : NAN;
        fetch(turn + 1 < turns ? t0 + kTurn + mine : a.r.max_len);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int j = t0 + 32 * (wave + 4 * k);
            const uint32_t now = tile_bits(k);
            const float ks[2] = {lane_float(k_sc, 32 * k), lane_float(k_sc, 32 * k + 16)};
            const float vs[2] = {lane_float(v_sc, 32 * k), lane_float(v_sc, 32 * k + 16)};
            const bool all = now == 0xffffffffu && j + 31 <= at_min && (j > at_max - a.window || j + 31 < a.sinks);
            // The tile's scores, rounded as the maxima are: fused with the subtraction the largest
            // one's distance is what the rounding left, whose e^ passes an fp16 from 2^24 on.
            f32x4_t sum[NT][2];
            if (now) {
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        i32x4_t hi = {0, 0, 0, 0}, lo = {0, 0, 0, 0};
                        const u32x4_t *dg = reinterpret_cast<const u32x4_t *>(lds) + t * NJ * 64 + (NT > 1 ? in_loop(lane) : lane);
#pragma unroll
                        for (int i = 0; i < NJ; ++i)
                            hi = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4_t, kf[u][i]),
                                                                       __builtin_bit_cast(i32x4_t, dg[2 * NT * NJ * 64 + i * 64]), hi, 0, 0, 0);
#pragma unroll
                        for (int i = 0; i < NJ; ++i)
                            lo = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4_t, kf[u][i]),
                                                                       __builtin_bit_cast(i32x4_t, dg[i * 64]), lo, 0, 0, 0);
                        hi = hi << 8;  // below 2^31: 256 dims of 127 128
#pragma unroll
                        for (int i = 0; i < NJ; ++i)
                            hi = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4_t, kf[u][i]),
                                                                       __builtin_bit_cast(i32x4_t, dg[NT * NJ * 64 + i * 64]), hi, 0, 0, 0);
                        const float kq = qs[t] * ks[u];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
#pragma clang fp contract(off)
                            sum[t][u][i] = __builtin_fmaf(static_cast<float>(hi[i]), 256.f, static_cast<float>(lo[i])) * kq;
                        }
                    }
            }
            // K's registers are free: the next tile's rows
            if (k == 0) {
                load_k(j + 128, 1, tile_bits(1) != 0);
            } else {
                look(t0 + kTurn + mine);  // past the last turn nothing is seen
                load_k(j + 128, 0, tile_bits(0) != 0);
            }
            if (now) {
                u32x4_t ph[NT], pl[NT];  // the weights' two operands
                if (!all)
#pragma unroll
                    for (int t = 0; t < NT; ++t) hide_unseen(sum[t], now >> (4 * g), in_loop(at[t] - j - 4 * g), a.window, a.sinks - j - 4 * g);  // a branch of its own
                float f[NT][2];
                rows.take(sum, vs, f);
#pragma unroll
                for (int t = 0; t < NT; ++t) rows.weigh(t, sum[t], f[t], ph[t], pl[t]);
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int i = 0; i < 4; ++i) vf[u][i] ^= vch_t(0x80808080u);  // code + 128
#pragma unroll
                for (int e = 0; e < CH; ++e) {
                    u32x4_t w;
#pragma unroll
                    for (int u = 0; u < 2; ++u)
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            w[2 * u + i] = codes_f16(__builtin_amdgcn_perm(vf[u][2 * i + 1][e / 4], vf[u][2 * i][e / 4],
                                                                           0x0c040c00u + 0x00010001u * static_cast<uint32_t>(e % 4)));
                        }
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        rows.o[t][e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, w), __builtin_bit_cast(f16x8_t, ph[t]), rows.o[t][e], 0, 0, 0);
                        rows.o[t][e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, w), __builtin_bit_cast(f16x8_t, pl[t]), rows.o[t][e], 0, 0, 0);
                    }
                }
            }
            load_v(j + 128, 1 - k, tile_bits(1 - k) != 0);
        }
    }

    // The four wavefronts' outputs joined, kJoin rows at a time: first what each
    // wavefront's are to be taken by, a row a thread, then four dims a thread.
    const int64_t shift = record_shift(a, b, s);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const float sum = quad_sum(rows.l[t]);
        if (g == 0) sm[wave][16 * t + r] = rows.m[t], sl[wave][16 * t + r] = sum, su[wave][16 * t + r] = 9 - unit_of_scale(rows.unit[t]);
    }
    __syncthreads();  // and the digits have been read
    if (tid < kRows && row0 + tid < R) {
        const float M = fmaxf(fmaxf(sm[0][tid], sm[1][tid]), fmaxf(sm[2][tid], sm[3][tid])), ref = M == -INFINITY ? 0.f : M;
        float L = 0.f, f[4];
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            f[w] = __builtin_amdgcn_exp2f(sm[w][tid] - ref);
            L += f[w] * sl[w][tid];
        }
        const int64_t row = place[tid].x;
        const int h = place[tid].y;
        const float norm = L == 0.f ? 0.f : 1.0f / L;
#pragma unroll
        for (int w = 0; w < 4; ++w) sm[w][tid] = f[w] * norm;
        sl[0][tid] = L;
        if (whole)
            store_lse(a, row, h, M, L);
        else
            a.ml[((row + shift) * a.n_head + h) * a.n_split + split] = make_float2(M, L);
    }
    float *const ob = reinterpret_cast<float *>(lds);
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int k = 0; k < 16 / kJoin; ++k) {
            const int q0 = 16 * t + kJoin * k;
            if (row0 + q0 >= R) continue;  // whole workgroup
            if (q0) __syncthreads();  // the rows before have been read
            if (r / kJoin == k) {
                float *row = ob + (wave * kJoin + r % kJoin) * OS + 4 * g;
#pragma unroll
                for (int e = 0; e < CH; ++e) *reinterpret_cast<f32x4_t *>(row + 16 * e) = rows.o[t][e];
            }
            __syncthreads();
            for (int i = tid; i < kJoin * DP / 4; i += 256) {
                const int q = q0 + i / (DP / 4), dim = i % (DP / 4) * 4;
                if (dim >= d || row0 + q >= R) continue;
                f32x4_t x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    const float f = sm[w][q];
                    const float *from = ob + (w * kJoin + q - q0) * OS;
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[e] += ldexpf(f * from[(dim + e) % CH * 16 + (dim + e) / CH], su[w][q]);
                }
                const int64_t row = place[q].x;
                const int h = place[q].y;
                if (whole)
#pragma unroll
                    for (int e = 0; e < 4; ++e) store_out<IO>(a, row, h, dim + e, x[e], sl[0][q]);
                else
                    *reinterpret_cast<f32x4_t *>(a.part + (((row + shift) * a.n_head + h) * a.n_split + split) * d + dim) = x;
            }
        }
}

// The same for many rows of a sequence and kv head: 128 of them a workgroup, two tiles
// of 16 a wavefront, which takes them through all slots of the split, so that nothing is
// joined but splits.  64 slots at a time of K and V are turned to fp16 operands
// once for all of them and go through LDS, a buffer being filled while the other
// is read; wavefronts 0 and 1 make V's operands, 2 and 3 K's.  A query is one fp16
// operand against a power of two of its row (bf16 fits it whole) or, in fp32, two
// (2^-22 of a value), and the scores are summed in fp32: the codes' exact products
// of three digits cost a third more matrix instructions and four conversions a
// score.
//
// Bound by issue: two pieces of 1024 bf16 rows over up to 16384 slots take 487 us (250
// GFLOP, 0.51 PFLOP/s), of which a SIMD is busy for 1.00 million cycles (some 2.1 GHz
// under this load). Matrix instructions take 0.36 of them, the others 0.49 (130 for each
// 16 rows and 32 slots, some 45 of them the staging), and the two wavefronts that the LDS
// leaves a SIMD overlap little of that.  One tile's weights stand beside the other's
// products (after both 549); one tile a wavefront takes 667 us for fp32 rows, two 542.
constexpr int kRowTiles = 2, kGroupRows = 64 * kRowTiles;
template <typename IO, int DP>
__global__ __launch_bounds__(256, 2) void kv8_rows_kernel(Attend8Args a) {
    constexpr int RT = kRowTiles;
    constexpr int NC = DP / 32;                // steps of the first product over the dims
    constexpr int CH = DP / 16, VW = CH / 4;   // adjacent dims of V a lane, and their dwords
    constexpr int NQ = sizeof(IO) == 4 ? 2 : 1;
    constexpr int kStage = 64;
    constexpr int kK = 4 * NC * 64, kV = 2 * CH * 64;  // operands of 16 bytes a buffer
    extern __shared__ __attribute__((aligned(16))) unsigned char lds[];  // two buffers of K's [4][NC][64] and V's [2][CH][64]
    typedef uint32_t vch_t __attribute__((ext_vector_type(VW)));
    u32x4_t *const buf = reinterpret_cast<u32x4_t *>(lds);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = lane & 15, g = lane >> 4;
    const int kvh = static_cast<int>(blockIdx.x) % a.c.n_head_kv;
    const int64_t b = static_cast<int64_t>(blockIdx.x) / a.c.n_head_kv;
    const int G = a.n_head / a.c.n_head_kv, d = a.c.d;
    const SeqRows s = seq_rows(a.r, b);
    const int R = s.count * G, group0 = static_cast<int>(blockIdx.y) * kGroupRows;
    if (group0 >= R) return;  // whole workgroup
    const int before = s.n - s.count;  // slots ahead of the new rows
    const int slots = a.turns * kTurn, split = blockIdx.z, split_first = split * slots, split_end = min(split_first + slots, s.n);
    const int at_min = before + group0 / G, at_max = before + (min(group0 + kGroupRows, R) - 1) / G;
    const bool whole = s.n <= slots;  // the sequence's only split
    if (whole ? split > 0 : !sees(a, at_max, split_first, split_end) && !sees(a, at_min, split_first, split_end)) return;
    const int end = seen_end(a, at_min, at_max, split_end), first = seen_begin(a, at_min, split_first, kStage);
    const int stages = end > first ? (end - first + kStage - 1) / kStage : 0;
    const int row0 = group0 + 16 * RT * wave;  // the wavefront's
    const int mine_min = before + min(row0, R - 1) / G, mine_max = before + (min(row0 + 16 * RT, R) - 1) / G;

    // Lane l stands for slot l of a stage; every wavefront looks at all of them.
    const int32_t *const pages = a.c.pages + b * a.c.max_pages;
    int32_t id = -1;
    uint32_t kept = 1;
    auto fetch = [&](int stage) {
        const int j = first + kStage * stage + lane;
        id = -1;
        if (stage >= stages || j >= a.r.max_len) return;
        id = pages[j >> a.c.page_shift];
        if (a.mask) kept = a.mask[b * a.mask_stride + j];
    };
    int32_t page = 0;
    float k_raw = 0.f, v_raw = 0.f;
    uint64_t bits = 0;
    auto look = [&](int stage) {
        const int j = first + kStage * stage + lane;
        const bool there = id >= 0 && id < a.c.n_pages;
        page = there ? id : 0;  // a hole's rows are read (of a page that is there), never used
        bits = __ballot(there && kept != 0 && j < end && (j > at_min - a.window || j < a.sinks));
        k_raw = v_raw = 0.f;
        if (static_cast<uint32_t>(bits >> (lane & 48)) & 0xffffu) {
            const int64_t i = kv8_scale(a.c, page, j & ((1 << a.c.page_shift) - 1), kvh);
            k_raw = a.c.k_scale[i];
            v_raw = a.c.v_scale[i];
        }
    };
    // The wavefront's part of a stage: 32 slots, from 32 (wave % 2).  16 slots from a
    // multiple of 16 stay in their page; where none of 16 is seen, one line is read.
    const int8_t *const kp = a.c.k + kvh * a.c.head_stride, *const vp = a.c.v + kvh * a.c.head_stride;
    u32x4_t raw[2 * (DP / 64) > 4 * VW / 2 ? 2 * (DP / 64) : 4 * VW / 2];  // 2 DP / 64 pieces of K, or 8 of VW dwords of V
    constexpr int NJ = DP / 64;
    const int part = 32 * (wave & 1);
    auto load = [&](int stage) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const bool there = static_cast<uint32_t>(bits >> (part + 16 * u)) & 0xffffu;
            const int j = first + kStage * stage + part + 16 * u;
            const int64_t row = there ? static_cast<int64_t>(__builtin_amdgcn_readlane(page, part + 16 * u)) * a.c.page_stride +
                                            static_cast<int64_t>(j & ((1 << a.c.page_shift) - 1)) * a.c.token_stride
                                      : 0;
            const uint32_t step = there ? static_cast<uint32_t>(a.c.token_stride) : 0u;
            if (wave >= 2) {
                const int8_t *const base = kp + row;
                const uint32_t off = static_cast<uint32_t>(r) * step;
#pragma unroll
                for (int i = 0; i < NJ; ++i)
                    raw[u * NJ + i] = *reinterpret_cast<const u32x4_t *>(base + (off + static_cast<uint32_t>(min(16 * (4 * i + g), d - 16))));
            } else {
                const int8_t *const base = vp + row;
                const uint32_t off = 4 * static_cast<uint32_t>(g) * step + static_cast<uint32_t>(min(CH * r, d - CH));
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const vch_t v = load_dwords<VW>(base + static_cast<uint64_t>(i) * step + off);
#pragma unroll
                    for (int w = 0; w < VW; ++w) raw[(VW * (4 * u + i) + w) / 4][(VW * (4 * u + i) + w) % 4] = v[w];
                }
            }
        }
    };
    auto stage_out = [&](int into) {
        u32x4_t *const to = buf + into * (kK + kV);
#pragma unroll
        for (int i = 0; i < static_cast<int>(sizeof(raw) / 16); ++i) raw[i] ^= u32x4_t(0x80808080u);  // code + 128
        if (wave >= 2) {
            // 16 dims of a slot: eight each of operands 2 j and 2 j + 1
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int i = 0; i < NJ; ++i)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        u32x4_t w;
#pragma unroll
                        for (int x = 0; x < 4; ++x) {
                            const uint32_t four = raw[u * NJ + i][2 * h + x / 2];
                            w[x] = codes_f16(__builtin_amdgcn_perm(four, four, x & 1 ? 0x0c030c02u : 0x0c010c00u));
                        }
                        to[((part / 16 + u) * NC + 2 * i + h) * 64 + lane] = w;
                    }
        } else {
            // eight slots of CH dims: an operand of each dim
#pragma unroll
            for (int e = 0; e < CH; ++e) {
                u32x4_t w;
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const int n0 = VW * (2 * x) + e / 4, n1 = VW * (2 * x + 1) + e / 4;
                    w[x] = codes_f16(__builtin_amdgcn_perm(raw[n1 / 4][n1 % 4], raw[n0 / 4][n0 % 4], 0x0c040c00u + 0x00010001u * static_cast<uint32_t>(e % 4)));
                }
                to[kK + (part / 32 * CH + e) * 64 + lane] = w;
            }
        }
    };

    fetch(0);
    // The wavefront's queries as operands: dims 64 j + 16 g + 8 h .. + 7 of row r in
    // operand 2 j + h, against a power of two at or above the row's largest half.
    u32x4_t qf[RT][NQ][NC];
    float qs[RT];
    int at[RT];
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        const int rho = row0 + 16 * t + r;
        at[t] = rho < R ? before + rho / G : -1;
        float x[NJ][16];
        uint32_t top = 0;  // magnitudes order as their bits do, NaN above infinity
#pragma unroll
        for (int i = 0; i < NJ; ++i) {
            const int dim = 64 * i + 16 * g;
#pragma unroll
            for (int e = 0; e < 16; ++e) x[i][e] = 0.f;
            if (rho < R && dim < d) load16(static_cast<const IO *>(a.q) + (s.first + rho / G) * a.q_stride + static_cast<int64_t>(kvh * G + rho % G) * d + dim, x[i]);
#pragma unroll
            for (int e = 0; e < 16; ++e) top = max(top, __float_as_uint(x[i][e]) & 0x7fffffffu);
        }
        top = max(top, static_cast<uint32_t>(xor_shfl(static_cast<int>(top), 16)));
        top = max(top, static_cast<uint32_t>(xor_shfl(static_cast<int>(top), 32)));
        const int ex = max(static_cast<int>(top >> 23), 27) - 127 - 14;  // max < 2^15 2^ex (a row below 2^-100 takes 2^-114)
        // the codes are multiples of 2^-9; a negative scale goes into the operands' sign
        qs[t] = top >= 0x7f800000u ? NAN : ldexpf(fabsf(a.scale) * 1.4426950408889634f * 512.f, ex);
#pragma unroll
        for (int i = 0; i < NJ; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    const float x0 = ldexpf(a.scale < 0.f ? -x[i][8 * h + 2 * w] : x[i][8 * h + 2 * w], -ex);
                    const float x1 = ldexpf(a.scale < 0.f ? -x[i][8 * h + 2 * w + 1] : x[i][8 * h + 2 * w + 1], -ex);
                    const f16x2_t hi = __builtin_convertvector(f32x2_t{x0, x1}, f16x2_t);
                    qf[t][0][2 * i + h][w] = __builtin_bit_cast(uint32_t, hi);
                    if constexpr (NQ == 2)
                        qf[t][1][2 * i + h][w] = __builtin_bit_cast(
                            uint32_t, __builtin_convertvector(f32x2_t{x0 - static_cast<float>(hi[0]), x1 - static_cast<float>(hi[1])}, f16x2_t));
                }
    }
    Rows<RT, CH> rows;
    look(0);
    load(0);
    fetch(1);
    stage_out(0);
    uint64_t seen = bits;
    float k_sc = k_raw, v_sc = v_raw;
    __syncthreads();
    for (int stage = 0; stage < stages; ++stage) {
        k_sc = k_sc >= 0.f && k_sc < INFINITY ? k_sc : NAN, v_sc = v_sc >= 0.f && v_sc < INFINITY ? v_sc : NAN;
        look(stage + 1);  // past the last nothing is seen
        load(stage + 1);
        fetch(stage + 2);
        const u32x4_t *const from = buf + (stage & 1) * (kK + kV);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int j = first + kStage * stage + 32 * half;
            uint32_t now = static_cast<uint32_t>(seen >> (32 * half));
            if (j > mine_max || (j + 31 <= mine_min - a.window && j >= a.sinks) || row0 >= R) now = 0;
            const bool all = now == 0xffffffffu && j + 31 <= mine_min && (j > mine_max - a.window || j + 31 < a.sinks);
            const float ks[2] = {lane_float(k_sc, 32 * half), lane_float(k_sc, 32 * half + 16)};
            const float vs[2] = {lane_float(v_sc, 32 * half), lane_float(v_sc, 32 * half + 16)};
            if (now) {
                f32x4_t sum[RT][2];
#pragma unroll
                for (int t = 0; t < RT; ++t) sum[t][0] = sum[t][1] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int n = NQ - 1; n >= 0; --n)  // the smaller operand first
#pragma unroll
                    for (int c = 0; c < NC; ++c) {
                        u32x4_t k[2];
#pragma unroll
                        for (int u = 0; u < 2; ++u) k[u] = from[((2 * half + u) * NC + c) * 64 + lane];
#pragma unroll
                        for (int u = 0; u < 2; ++u)
#pragma unroll
                            for (int t = 0; t < RT; ++t)
                                sum[t][u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, k[u]), __builtin_bit_cast(f16x8_t, qf[t][n][c]), sum[t][u], 0, 0, 0);
                    }
#pragma unroll
                for (int t = 0; t < RT; ++t)
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        const float kq = qs[t] * ks[u];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
#pragma clang fp contract(off)
                            sum[t][u][i] *= kq;
                        }
                    }
                if (!all)
#pragma unroll
                    for (int t = 0; t < RT; ++t) hide_unseen(sum[t], now >> (4 * g), in_loop(at[t] - j - 4 * g), a.window, a.sinks - j - 4 * g);  // a branch of its own
                float f[RT][2];
                rows.take(sum, vs, f);
                u32x4_t w[CH];
#pragma unroll
                for (int e = 0; e < CH; ++e) w[e] = from[kK + (half * CH + e) * 64 + lane];
                // one tile's weights beside the other's products
#pragma unroll
                for (int t = 0; t < RT; ++t) {
                    u32x4_t p[2];
                    rows.weigh(t, sum[t], f[t], p[0], p[1]);
#pragma unroll
                    for (int n = 0; n < 2; ++n)
#pragma unroll
                        for (int e = 0; e < CH; ++e)
                            rows.o[t][e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, w[e]), __builtin_bit_cast(f16x8_t, p[n]), rows.o[t][e], 0, 0, 0);
                }
            }
        }
        if (stage + 1 < stages) stage_out((stage + 1) & 1);  // last read a stage ago, before the barrier
        seen = bits;
        k_sc = k_raw, v_sc = v_raw;
        __syncthreads();
    }
    const int64_t shift = record_shift(a, b, s);
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        const float L = quad_sum(rows.l[t]);
        const int rho = row0 + 16 * t + r;
        if (rho >= R) continue;
        const int64_t row = s.first + rho / G;
        const int h = kvh * G + rho % G;
        const int64_t rec = ((row + shift) * a.n_head + h) * a.n_split + split;
        const float norm = L == 0.f ? 0.f : 1.0f / L;
        const int to = 9 - unit_of_scale(rows.unit[t]);
        if (g == 0) {
            if (whole)
                store_lse(a, row, h, rows.m[t], L);
            else
                a.ml[rec] = make_float2(rows.m[t], L);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int dim = CH * (4 * g + i);
            if (dim >= d) continue;
#pragma unroll
            for (int e = 0; e < CH; e += 4) {
                f32x4_t x;
#pragma unroll
                for (int k = 0; k < 4; ++k) x[k] = ldexpf(rows.o[t][e + k][i] * norm, to);
                if (whole) {
#pragma unroll
                    for (int k = 0; k < 4; ++k) store_out<IO>(a, row, h, dim + e + k, x[k], L);
                } else {
                    *reinterpret_cast<f32x4_t *>(a.part + rec * d + dim + e) = x;
                }
            }
        }
    }
}

__device__ __forceinline__ float reciprocal(float l) { return l == 0.f ? 0.f : __builtin_amdgcn_rcpf(l); }
// The splits of a row and head joined by NG groups of DP / 4 lanes, each with
// every NG-th split and four dims a lane, kAhead splits on their way at a time;
// 256 / (NG DP / 4) heads a workgroup.  What is joined stays an average at every step (its
// rounding 3 U, of at most 64 + NG steps), so that values up to fp32's last do not pass it.
constexpr int kAhead = 4;
template <typename IO, int DP, int NG>
__global__ __launch_bounds__(256) void kv8_join_kernel(Attend8Args a) {
    constexpr int DL = DP / 4, PER = 256 / (NG * DL);
    __shared__ f32x4_t red[256];
    __shared__ float2 rml[256];
    const int tid = threadIdx.x, who = tid / (NG * DL), grp = tid / DL % NG, dim = 4 * (tid % DL);
    const int64_t b = blockIdx.z;
    const SeqRows s = seq_rows(a.r, b);
    const int64_t item = static_cast<int64_t>(blockIdx.x) * PER + who;  // row of the sequence, head
    const int i = static_cast<int>(item / a.n_head), h = static_cast<int>(item % a.n_head);
    const int slots = a.turns * kTurn;
    if (s.n <= slots) return;  // its only split wrote it
    if (static_cast<int64_t>(blockIdx.x) * PER >= static_cast<int64_t>(s.count) * a.n_head) return;  // whole workgroup
    // threads past the last whole head (of 192 dims 16 or 64) have no work but the barrier
    const bool live = who < PER && i < s.count;
    const int at = s.n - s.count + i, d = a.c.d;
    const int64_t row = s.first + i, rec = ((row + record_shift(a, b, s)) * a.n_head + h) * a.n_split;
    f32x4_t x = {0.f, 0.f, 0.f, 0.f};
    float M = -INFINITY, L = 0.f;
    if (live)
        for (int s0 = grp; s0 * slots <= at; s0 += kAhead * NG) {
            float2 ml[kAhead];
            f32x4_t part[kAhead];
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                const int sp = s0 + k * NG;
                ml[k] = make_float2(-INFINITY, 0.f);
                part[k] = f32x4_t{0.f, 0.f, 0.f, 0.f};
                if (sp * slots <= at && sees(a, at, sp * slots, min((sp + 1) * slots, s.n))) {
                    ml[k] = a.ml[rec + sp];
                    if (dim < d) part[k] = *reinterpret_cast<const f32x4_t *>(a.part + (rec + sp) * d + dim);
                }
            }
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                const float mn = fmaxf(M, ml[k].x), ref = mn == -INFINITY ? 0.f : mn;
                const float f = L * __builtin_amdgcn_exp2f(M - ref), w = ml[k].y * __builtin_amdgcn_exp2f(ml[k].x - ref);
                L = f + w, M = mn;
                const float inv = reciprocal(L);
                x = f * inv * x + w * inv * part[k];
            }
        }
    if constexpr (NG > 1) {
        red[tid] = x;
        rml[tid] = make_float2(M, L);
        __syncthreads();
        if (grp) return;
#pragma unroll
        for (int k = 1; k < NG; ++k) {
            const float2 ml = rml[tid + k * DL];
            const float mn = fmaxf(M, ml.x), ref = mn == -INFINITY ? 0.f : mn;
            const float f = L * __builtin_amdgcn_exp2f(M - ref), w = ml.y * __builtin_amdgcn_exp2f(ml.x - ref);
            L = f + w, M = mn;
            const float inv = reciprocal(L);
            x = f * inv * x + w * inv * red[tid + k * DL];
        }
    }
    if (!live || dim >= d) return;
#pragma unroll
    for (int e = 0; e < 4; ++e) store_out<IO>(a, row, h, dim + e, x[e], L);
    if (dim == 0) store_lse(a, row, h, M, L);
}

// The join after a kernel of the splits.
template <typename IO, int DP>
int launch_join(const Attend8Args &a, size_t seqs, hipStream_t s);

template <typename IO, int DP>
int launch_rows(const Attend8Args &a, size_t seqs, hipStream_t s) {
    constexpr size_t lds = 2 * (4 * (DP / 32) + 2 * (DP / 16)) * 1024;
    static_assert(lds <= 65536, "more LDS than a launch gets unasked");
    const int64_t rows = static_cast<int64_t>(a.r.max_new) * (a.n_head / a.c.n_head_kv);
    const dim3 grid(static_cast<unsigned>(seqs * static_cast<size_t>(a.c.n_head_kv)), static_cast<unsigned>((rows + kGroupRows - 1) / kGroupRows),
                    static_cast<unsigned>(a.n_split));
    hipLaunchKernelGGL((kv8_rows_kernel<IO, DP>), grid, dim3(256), lds, s, a);
    const int st = check_launch("kv8_rows_kernel");
    return st ? st : launch_join<IO, DP>(a, seqs, s);
}

template <typename IO, int DP, int NT>
int launch_attend(const Attend8Args &a, size_t seqs, hipStream_t s) {
    constexpr size_t digits = 3 * NT * (DP / 64) * 1024, outputs = 4 * joined_rows(DP) * (DP + 4) * sizeof(float);
    constexpr size_t lds = digits > outputs ? digits : outputs;
    static_assert(lds + 4096 <= 65536, "more LDS than a launch gets unasked");
    const int64_t rows = static_cast<int64_t>(a.r.max_new) * (a.n_head / a.c.n_head_kv);
    const dim3 grid(static_cast<unsigned>(seqs * static_cast<size_t>(a.c.n_head_kv)), static_cast<unsigned>((rows + 16 * NT - 1) / (16 * NT)),
                    static_cast<unsigned>(a.n_split));
    hipLaunchKernelGGL((kv8_attend_kernel<IO, DP, NT>), grid, dim3(256), lds, s, a);
    const int st = check_launch("kv8_attend_kernel");
    return st ? st : launch_join<IO, DP>(a, seqs, s);
}

template <typename IO, int DP>
int launch_join(const Attend8Args &a, size_t seqs, hipStream_t s) {
    if (a.n_split == 1) return OURO_OK;
    const int64_t heads = static_cast<int64_t>(a.r.max_new) * a.n_head;
    // groups that can have work: a group takes kAhead splits at a time
    constexpr int DL = DP / 4, kMost = 256 / DL, kSome = kMost < 4 ? kMost : 4;
    auto go = [&](auto groups) {
        constexpr int NG = decltype(groups)::value, PER = 256 / (NG * DL);
        hipLaunchKernelGGL((kv8_join_kernel<IO, DP, NG>), dim3(static_cast<unsigned>((heads + PER - 1) / PER), 1, static_cast<unsigned>(seqs)),
                           dim3(256), 0, s, a);
    };
    if (a.n_split <= kAhead)
        go(std::integral_constant<int, 1>{});
    else if (a.n_split <= 4 * kAhead)
        go(std::integral_constant<int, kSome>{});
    else
        go(std::integral_constant<int, kMost>{});
    return check_launch("kv8_join_kernel");
}

// The dims of a lane of V must divide the head: 192 only for its multiples of 12.
int padded(size_t d) { return d <= 64 ? 64 : d <= 128 ? 128 : d <= 192 && d % 12 == 0 ? 192 : 256; }

// How a call goes, by the most rows that a sequence has of a kv head (new tokens
// times query heads of it): never by how many sequences there are, so that a
// sequence's bits do not depend on the batch it is in.
struct Way {
    int tiles;   // of 16 rows of a workgroup, or 0: kv8_rows_kernel
    int turns;   // of 256 slots of a split
    int splits;  // no more for any shorter max_len
};
constexpr int kFewRows = 16, kSomeRows = 256, kMostSplits = 1024;
// how often the grid of kv8_rows_kernel is split
constexpr int kManyGroups = 512, kLeastSplits = 4;
Way way_of(int64_t rows, int n_head_kv, int dp, size_t max_len) {
    Way w;
    const int64_t all = static_cast<int64_t>((max_len + kTurn - 1) / kTurn);
    if (rows <= kFewRows) {
        // two turns: 64 sequences of 1024 slots 18.2 us (one turn 21.2, four 15.7), one of
        // 16384 13.9 (12.7, 17.9); wider heads four: 32 of 4096 and 256 dims 47.0 us (two 48.5)
        w = {1, dp <= 128 ? 2 : 4, 0};
    } else if (rows <= kSomeRows || dp > 128) {
        // 64 sequences of 2048 slots and 20 rows 35.0 us (one tile at best 44.9), 48 of 4096
        // and 96 rows 77 (kv8_rows_kernel 89; of 64 dims 53 and 54), 4 of 4096 and 256 rows
        // 38 (48); wider heads eight turns: 32 of 4096, 24 rows of 256 dims 62 (four 73)
        w = {2, dp <= 128 ? 4 : 8, 0};
    } else {
        // splits until some 512 workgroups of a sequence's have work, and four at least, of
        // four to sixteen turns: one sequence of 16384 slots and 1024 rows 92 us with four
        // turns (eight 122), two of 4096 rows 499 with sixteen (eight 518, thirty-two 474),
        // one prompt of 4096 tokens, 16384 rows, 194 with four (eight 206, sixteen 231)
        const int64_t groups = (rows + kGroupRows - 1) / kGroupRows * n_head_kv;
        const int64_t splits = groups * kLeastSplits < kManyGroups ? kManyGroups / groups : kLeastSplits;
        const int64_t turns = (all + splits - 1) / splits, least = (all + 15) / 16, most = (all + 3) / 4;
        w = {0, static_cast<int>(turns < 4 ? 4 : turns > 16 ? 16 : turns), 0};
        // turns go up in whole ones, and the splits of a longer max_len can be fewer
        const int64_t bound = splits > least ? splits : least;
        w.splits = static_cast<int>(bound < most ? bound : most);
    }
    if (w.tiles) w.splits = static_cast<int>((all + w.turns - 1) / w.turns);
    if (w.splits > kMostSplits) w.splits = kMostSplits;
    while ((all + w.turns - 1) / w.turns > kMostSplits) w.turns *= 2;
    return w;
}
struct Attend8Ws {
    Way way;
    int n_split;
    bool by_seq;
    size_t part, bytes;
};
// Records are of the packed rows or of max_new rows of each sequence, whichever are fewer.
size_t records_bytes(size_t rows, size_t seqs, size_t max_new, size_t n_head, size_t d, int splits, size_t *part) {
    if (splits < 2) return 0;
    const size_t recs = (seqs * max_new < rows ? seqs * max_new : rows) * n_head * static_cast<size_t>(splits);
    *part = (recs * sizeof(float2) + 255) & ~size_t{255};
    return *part + recs * d * sizeof(float);
}
// A sequence's rows of a kv head, of the caller's max_new, whatever rows there are: a
// sequence alone goes the way that it goes with others.
int64_t rows_of_one(size_t max_new, size_t n_head, size_t n_head_kv) {
    return static_cast<int64_t>((max_new < (1u << 24) ? max_new : 1u << 24) * (n_head / n_head_kv));
}
Attend8Ws attend_ws(size_t seqs, size_t rows, size_t max_new, size_t n_head, size_t n_head_kv, size_t d, size_t max_len) {
    Attend8Ws w{};
    w.way = way_of(rows_of_one(max_new, n_head, n_head_kv), static_cast<int>(n_head_kv), padded(d), max_len);
    const size_t slots = static_cast<size_t>(w.way.turns) * kTurn;
    w.n_split = max_len ? static_cast<int>((max_len + slots - 1) / slots) : 1;
    if (max_new > rows) max_new = rows;
    w.by_seq = seqs * max_new < rows;
    w.bytes = records_bytes(rows, seqs, max_new, n_head, d, w.n_split, &w.part);
    return w;
}

// The most that a call of no more rows, new ones of a sequence or slots can take: fewer rows of a sequence can go a way of more splits.  Records grow
// with max_new while the way's splits are the same, so what counts is the largest
// max_new of each: of few rows, of some, of each number of groups that is split anew.
size_t attend_most(size_t seqs, size_t rows, size_t max_new, size_t n_head, size_t n_head_kv, size_t d, size_t max_len) {
    if (!n_head_kv || n_head < n_head_kv || seqs > 65535 || rows > (1u << 23)) return 0;
    const size_t G = n_head / n_head_kv;
    size_t most = 0;
    auto see = [&](size_t of_one) {  // rows of a kv head
        const size_t t = of_one / G < max_new ? of_one / G : max_new;
        size_t part;
        const Way w = way_of(rows_of_one(t, n_head, n_head_kv), static_cast<int>(n_head_kv), padded(d), max_len);
        const size_t b = records_bytes(rows, seqs, t < rows ? t : rows, n_head, d, w.splits, &part);
        if (b > most) most = b;
    };
    see(kFewRows);
    see(kSomeRows);
    for (size_t g = 1; g * n_head_kv * kLeastSplits < kManyGroups + n_head_kv * kLeastSplits; ++g) see(g * kGroupRows);
    see(max_new < (1u << 24) ? max_new * G : static_cast<size_t>(1u << 24) * G);
    return most;
}

template <typename IO>
int launch_attend(const Attend8Args &a, size_t seqs, int tiles, hipStream_t s) {
    const int dp = padded(static_cast<size_t>(a.c.d));
    if (tiles == 0) return dp == 64 ? launch_rows<IO, 64>(a, seqs, s) : launch_rows<IO, 128>(a, seqs, s);
    if (dp == 64) return tiles == 1 ? launch_attend<IO, 64, 1>(a, seqs, s) : launch_attend<IO, 64, 2>(a, seqs, s);
    if (dp == 128) return tiles == 1 ? launch_attend<IO, 128, 1>(a, seqs, s) : launch_attend<IO, 128, 2>(a, seqs, s);
    if (dp == 192) return tiles == 1 ? launch_attend<IO, 192, 1>(a, seqs, s) : launch_attend<IO, 192, 2>(a, seqs, s);
    return tiles == 1 ? launch_attend<IO, 256, 1>(a, seqs, s) : launch_attend<IO, 256, 2>(a, seqs, s);
}

}  // namespace
}  // namespace ouro

using namespace ouro;

extern "C" {

size_t ouro_kv8_attend_workspace_bytes(size_t seqs, size_t rows, size_t max_new, size_t n_head, size_t n_head_kv, size_t head_dim,
                                       size_t max_len) {
    return attend_most(seqs, rows, max_new, n_head, n_head_kv, head_dim, max_len);
}

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
    if (q_stride > (size_t{1} << 40) || out_stride > (size_t{1} << 40) || mask_stride > (size_t{1} << 40))
        return fail(OURO_ERR_SHAPE, "%s: a stride past 2^40", me);
    const size_t unit = dtype == OURO_DT_F32 ? 4 : 8;
    if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(gate)) & 15 ||
        q_stride % unit || out_stride % unit)
        return fail(OURO_ERR_ALIGN, "%s: rows must start at multiples of 16 bytes", me);
    if (!seqs || !a.r.max_new) return OURO_OK;
    auto most = [](size_t x) { return static_cast<int32_t>(x < (1u << 30) ? x : 1u << 30); };
    a.q = q, a.gate = gate, a.mask = mask, a.out = out, a.lse = lse;
    a.q_stride = static_cast<int64_t>(q_stride), a.out_stride = static_cast<int64_t>(out_stride);
    a.mask_stride = static_cast<int64_t>(mask_stride);
    a.n_head = static_cast<int>(n_head), a.window = window ? most(window) : 1 << 30, a.sinks = most(sinks), a.scale = scale;
    const Attend8Ws w = attend_ws(seqs, rows, max_new, n_head, hkv, d, max_len);
    a.n_split = w.n_split, a.turns = w.way.turns, a.by_seq = w.by_seq;
    const size_t most_new = static_cast<size_t>(a.r.max_new);
    if (seqs * hkv >= (1u << 24) || most_new * (n_head / hkv) > (1u << 20) || most_new * n_head >= (1u << 24))
        return fail(OURO_ERR_SHAPE, "%s: %zu rows of one sequence of %zu heads, %zu sequences", me, most_new, n_head, seqs);
    if (w.bytes) {
        if (!ws && !(ws = workspace(w.bytes, stream))) return OURO_ERR_HIP;
        a.ml = static_cast<float2 *>(ws);
        a.part = reinterpret_cast<float *>(static_cast<unsigned char *>(ws) + w.part);
    }
    return dtype == OURO_DT_F32 ? launch_attend<float>(a, seqs, w.way.tiles, as_stream(stream)) : launch_attend<uint16_t>(a, seqs, w.way.tiles, as_stream(stream));
}

}  // extern "C"
