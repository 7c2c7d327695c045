// verify.hip - drafted tokens judged by the target's logits, and the token that
// follows those that are kept.
//
// Row i of a sequence gives p_i = softmax(x / T), its draft row q_i; a drafted
// token t is kept while u q_i(t) < p_i(t); the next token is drawn from
// r = max(p_i - q_i, 0) of the first row that refuses, else from the last row's
// p, as the lowest t whose cumulative sum exceeds u' sum r.
//
// Which token is drawn hangs on sums over the whole vocabulary: at 248320 tokens
// a sum that is off by 1e-9 gives another token once in some thousand draws.  So
// exponentials, sums and comparisons are made in 64 bits, where it is once in 1e9
// or rarer; the logits are read in their own type and their differences are exact.
#include "logits.hpp"

#include "kv_cache.hpp"

#include <cmath>

namespace ouro {
namespace {

constexpr int kThreads = 256;
constexpr int kLogits = 32;  // logits of a thread
constexpr int kPartLogits = kThreads * kLogits;
constexpr double kLog2e = 1.4426950408889634;

// Sum of e^((x - m) / T) and the argmax (key) of a part of a row.
struct Part {
    double sum;
    float m;
    uint32_t at;
};
static_assert(sizeof(Part) == 16, "Part: workspace layout");

struct VerifyArgs {
    NewRows r;
    const void *x[2];  // logits, draft
    int64_t stride[2];
    const int32_t *tokens, *lens;
    const float *temperature, *u_accept, *u_next;
    int32_t *accepted, *next, *lens_out;
    Part *part;        // [2][rows][parts]
    double *left;      // [seqs][parts]: sums of max(p - q, 0)
    int32_t n, parts;
};
static_assert(sizeof(VerifyArgs) == 152, "VerifyArgs: kernel argument layout");

// 2^y for y <= 0: y = k + f, |f| <= 1/2, 2^f by its Taylor series, whose first
// term left out is (f ln 2)^12 / 12! <= 7e-15.  Below 2^-1000 it is 0, so that a
// product of what is not 0 never is.
__device__ __forceinline__ double exp2_64(double y) {
    if (!(y > -1000.0)) return 0.0;
    const double k = rint(y), z = (y - k) * 0.6931471805599453;
    double s = 1.0 / 39916800;
    s = fma(s, z, 1.0 / 3628800);
    s = fma(s, z, 1.0 / 362880);
    s = fma(s, z, 1.0 / 40320);
    s = fma(s, z, 1.0 / 5040);
    s = fma(s, z, 1.0 / 720);
    s = fma(s, z, 1.0 / 120);
    s = fma(s, z, 1.0 / 24);
    s = fma(s, z, 1.0 / 6);
    s = fma(s, z, 0.5);
    s = fma(s, z, 1.0);
    s = fma(s, z, 1.0);
    return __builtin_amdgcn_ldexp(s, static_cast<int>(k));
}
// e^((x - m) / T), c = log2 e / T, x <= m: 1 where x = m, infinite or not.
__device__ __forceinline__ double weight(float x, float m, double c) {
    return x == m ? 1.0 : exp2_64((static_cast<double>(x) - static_cast<double>(m)) * c);
}
__device__ __forceinline__ double shfl_xor64(double v, int mask) {
    const uint64_t u = __double_as_longlong(v);
    const uint32_t lo = __shfl_xor(static_cast<uint32_t>(u), mask, 64), hi = __shfl_xor(static_cast<uint32_t>(u >> 32), mask, 64);
    return __longlong_as_double(static_cast<long long>(static_cast<uint64_t>(hi) << 32 | lo));
}
__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) v += shfl_xor64(v, off);
    return v;
}
__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) v = fmaxf(v, xor_shfl(v, off));
    return v;
}
// Draws by likeliest token where the temperature is not above 0.
__device__ __forceinline__ float heat(const VerifyArgs &a, int64_t b) { return a.temperature ? a.temperature[b] : 1.f; }

template <typename T>
__device__ __forceinline__ LogitRow<T> row_at(const VerifyArgs &a, int which, int64_t row) {
    return LogitRow<T>(static_cast<const T *>(a.x[which]) + row * a.stride[which], a.n);
}

// A part of a row: its maximum, the lowest index of it, the sum against it.
template <typename T>
__device__ __forceinline__ void part_of(const VerifyArgs &a, int which, int64_t row, double c, Part *out) {
    constexpr int VL = LogitRow<T>::VL, kVec = kLogits / VL;
    __shared__ float top[kThreads / 64];
    __shared__ double sums[kThreads / 64];
    __shared__ uint32_t first[kThreads / 64];
    const int tid = threadIdx.x, wave = tid >> 6;
    const LogitRow<T> x = row_at<T>(a, which, row);
    const int q0 = static_cast<int>(blockIdx.x) * (kPartLogits / VL) + tid;
    u32x4_t v[kVec];
#pragma unroll
    for (int k = 0; k < kVec; ++k) v[k] = x.load(q0 + k * kThreads);
    float m = -INFINITY;
#pragma unroll
    for (int k = 0; k < kVec; ++k)
#pragma unroll
        for (int e = 0; e < VL; ++e) m = fmaxf(m, x.raw(v[k], e));  // passes over a NaN
    m = wave_max(m);
    if ((tid & 63) == 0) top[wave] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kThreads / 64; ++w) m = fmaxf(m, top[w]);
    double sum = 0.0;
    uint32_t at = 0xffffffffu;
    if (m > -INFINITY) {
#pragma unroll
        for (int k = 0; k < kVec; ++k)
#pragma unroll
            for (int e = 0; e < VL; ++e) {
                const float f = x.at(v[k], e);
                if (c > 0.0) sum += weight(f, m, c);
                if (f == m) at = min(at, static_cast<uint32_t>(x.first(q0 + k * kThreads) + e));
            }
    }
    sum = wave_sum(sum);
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) at = min(at, static_cast<uint32_t>(xor_shfl(static_cast<int>(at), off)));
    if ((tid & 63) == 0) sums[wave] = sum, first[wave] = at;
    __syncthreads();
    if (tid == 0) {
        for (int w = 1; w < kThreads / 64; ++w) sum += sums[w], at = min(at, first[w]);
        *out = Part{sum, m, at};
    }
}

template <typename T, typename D>
__global__ __launch_bounds__(kThreads) void verify_part_kernel(VerifyArgs a) {
    const int which = static_cast<int>(blockIdx.y) / a.r.max_new, i = static_cast<int>(blockIdx.y) % a.r.max_new;
    const SeqRows s = seq_rows(a.r, blockIdx.z);
    if (i >= s.count - which) return;  // the last row has no token to judge
    const float t = heat(a, blockIdx.z);
    const bool draws = t > 0.f;
    if (which && !draws) return;
    const int64_t row = s.first + i;
    Part *out = a.part + (static_cast<int64_t>(which) * a.r.rows + row) * a.parts + blockIdx.x;
    if (which)
        part_of<D>(a, 1, row, kLog2e, out);
    else
        part_of<T>(a, 0, row, draws ? kLog2e / static_cast<double>(t) : 0.0, out);
}

// A row's maximum, sum and argmax by one wavefront, to each of its lanes.
struct Sums {
    double z;
    float m;
    uint32_t at;
};
__device__ __forceinline__ Sums join_parts(const VerifyArgs &a, int which, int64_t row, double c) {
    const Part *p = a.part + (static_cast<int64_t>(which) * a.r.rows + row) * a.parts;
    const int lane = threadIdx.x & 63;
    Sums s{0.0, -INFINITY, 0xffffffffu};
    for (int i = lane; i < a.parts; i += 64) s.m = fmaxf(s.m, p[i].m);
    s.m = wave_max(s.m);
    for (int i = lane; i < a.parts; i += 64) {
        const Part x = p[i];
        if (x.m == -INFINITY) continue;
        s.z += x.sum * weight(x.m, s.m, c);
        if (x.m == s.m) s.at = min(s.at, x.at);
    }
    s.z = wave_sum(s.z);
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) s.at = min(s.at, static_cast<uint32_t>(xor_shfl(static_cast<int>(s.at), off)));
    return s;
}

// What a sequence came to: its deciding row (relative), whether that refused a
// token, its sums of p and q, the token refused (-1: none in the vocabulary).
struct Verdict {
    Sums p, q;
    int32_t row, refused, token, pad;
};

// The rows of a sequence judged, a wavefront each, up to the first that refuses.
template <typename T, typename D>
__device__ __forceinline__ Verdict decide(const VerifyArgs &a, const SeqRows &s, float t, Verdict *lds) {
    const int wave = threadIdx.x >> 6;
    const bool draws = t > 0.f;
    const double c = draws ? kLog2e / static_cast<double>(t) : 0.0;
    for (int i0 = 0; i0 < s.count; i0 += kThreads / 64) {
        const int i = i0 + wave;
        if (i < s.count) {
            const int64_t row = s.first + i;
            Verdict v{};
            v.row = i;
            v.p = join_parts(a, 0, row, c);
            v.token = -1;
            if (i + 1 < s.count) {
                const int next = a.tokens[row + 1];
                const bool in = next >= 0 && next < a.n;
                bool keep;
                if (!draws) {
                    keep = in && v.p.m > -INFINITY && static_cast<uint32_t>(next) == v.p.at;
                } else {
                    double p = 0.0, q = 1.0;
                    if (in && v.p.m > -INFINITY) p = weight(logit(row_at<T>(a, 0, row).x, next), v.p.m, c) / v.p.z;
                    if (a.x[1]) {
                        v.q = join_parts(a, 1, row, kLog2e);
                        q = in && v.q.m > -INFINITY ? weight(logit(row_at<D>(a, 1, row).x, next), v.q.m, kLog2e) / v.q.z : 0.0;
                    }
                    keep = in && static_cast<double>(a.u_accept[row]) * q < p;
                }
                v.refused = !keep;
                v.token = in ? next : -1;
            }
            if ((threadIdx.x & 63) == 0) lds[wave] = v;
        }
        __syncthreads();
        for (int w = 0; w < kThreads / 64; ++w)
            if (i0 + w < s.count && (lds[w].refused || i0 + w + 1 == s.count)) return lds[w];
        __syncthreads();
    }
    return Verdict{};  // no rows: not reached
}

// What a token is drawn by, of a part of the deciding row: max(p - q, 0) where a
// token was refused, p where none was or where nothing is left of it.
template <typename T, typename D>
struct Left {
    static constexpr int VL = LogitRow<T>::VL, kVec = kLogits / VL;
    LogitRow<T> x;
    LogitRow<D> y;
    double c, pz, qz;
    float pm, qm;
    int token;  // that a drafter without draft rows named, -1: none
    bool minus;
    __device__ __forceinline__ Left(const VerifyArgs &a, const SeqRows &s, const Verdict &v, float t, bool residual)
        : x(row_at<T>(a, 0, s.first + v.row)), y(row_at<D>(a, a.x[1] ? 1 : 0, s.first + v.row)) {
        c = kLog2e / static_cast<double>(t);
        pm = v.p.m, pz = 1.0 / v.p.z;
        qm = v.q.m, qz = 1.0 / v.q.z;
        minus = residual && a.x[1] && v.q.m > -INFINITY;
        token = residual && !a.x[1] ? v.token : -1;
    }
    // The draft's values at the places of vector q of x.
    __device__ __forceinline__ void beside(int q, float (&g)[VL]) const {
        if (LogitRow<D>::VL == VL && x.shift == y.shift) {
            const u32x4_t v = y.load(q);
#pragma unroll
            for (int e = 0; e < VL; ++e) g[e] = y.at(v, e);
        } else {
#pragma unroll
            for (int e = 0; e < VL; ++e) {
                const int i = x.first(q) + e;
                g[e] = i >= 0 && i < y.n ? logit(y.x, i) : -INFINITY;
            }
        }
    }
    // Of the elements of vector q; places outside the row have none.  The products
    // are rounded before they are subtracted, so that equal p and q leave nothing.
    __device__ __forceinline__ void weights(int q, double (&r)[VL]) const {
#pragma clang fp contract(off)
        const u32x4_t v = x.load(q);
        float g[VL];
        if (minus) beside(q, g);
#pragma unroll
        for (int e = 0; e < VL; ++e) {
            const int i = x.first(q) + e;
            r[e] = i >= 0 && i < x.n && i != token ? weight(x.at(v, e), pm, c) * pz : 0.0;
            if (minus) r[e] = fmax(r[e] - weight(g[e], qm, kLog2e) * qz, 0.0);
        }
    }
    // A thread's sums of a part, by vectors: those of all threads' k-th follow
    // each other, then the k + 1-st.
    __device__ __forceinline__ void sums(int part, double (&s)[kVec]) const {
#pragma unroll
        for (int k = 0; k < kVec; ++k) {
            double r[VL];
            weights(part * (kPartLogits / VL) + k * kThreads + static_cast<int>(threadIdx.x), r);
            s[k] = 0.0;
#pragma unroll
            for (int e = 0; e < VL; ++e) s[k] += r[e];
        }
    }
};

// A part's sum, to every thread; lds: a double of each wavefront.
template <typename L>
__device__ __forceinline__ double part_sum(const L &left, int part, double *lds) {
    double s[L::kVec], sum = 0.0;
    left.sums(part, s);
#pragma unroll
    for (int k = 0; k < L::kVec; ++k) sum += s[k];
    sum = wave_sum(sum);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = sum;
    __syncthreads();
    return lds[0] + lds[1] + lds[2] + lds[3];
}

// Sums of max(p - q, 0) over the parts of a sequence's refusing row.
template <typename T, typename D>
__global__ __launch_bounds__(kThreads) void verify_left_kernel(VerifyArgs a) {
    __shared__ Verdict lds[kThreads / 64];
    __shared__ double waves[kThreads / 64];
    const SeqRows s = seq_rows(a.r, blockIdx.y);
    const float t = heat(a, blockIdx.y);
    if (s.count == 0 || !(t > 0.f)) return;
    const Verdict v = decide<T, D>(a, s, t, lds);
    if (!v.refused || v.p.m == -INFINITY) return;
    const Left<T, D> left(a, s, v, t, true);
    const double sum = part_sum(left, blockIdx.x, waves);
    if (threadIdx.x == 0) a.left[static_cast<int64_t>(blockIdx.y) * a.parts + blockIdx.x] = sum;
}

// Inclusive sums over a wavefront's lanes.
__device__ __forceinline__ double wave_scan(double v) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const uint64_t u = __double_as_longlong(v);
        const uint32_t lo = __shfl_up(static_cast<uint32_t>(u), off, 64), hi = __shfl_up(static_cast<uint32_t>(u >> 32), off, 64);
        if (lane >= off) v += __longlong_as_double(static_cast<long long>(static_cast<uint64_t>(hi) << 32 | lo));
    }
    return v;
}

// The next token of a sequence: the part in which the cumulative sum passes
// u' of the whole, in it the wavefront's vectors, the lane, the element.  Sums that
// are made in two orders differ by roundings: where none passes, the last with
// any weight is taken, so that a token of weight 0 never is.
constexpr int kMaxParts = ((1 << 24) + 7 + kPartLogits - 1) / kPartLogits;
template <typename T, typename D>
__global__ __launch_bounds__(kThreads) void verify_next_kernel(VerifyArgs a) {
    using L = Left<T, D>;
    constexpr int kWaves = kThreads / 64, kSegs = L::kVec * kWaves;
    __shared__ Verdict lds[kWaves];
    __shared__ double mass[kMaxParts], waves[kWaves], seg[kSegs];
    __shared__ int chosen;
    __shared__ double before;
    const int64_t b = blockIdx.x;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const SeqRows s = seq_rows(a.r, b);
    const float t = heat(a, b);
    Verdict v{};
    if (s.count) v = decide<T, D>(a, s, t, lds);
    if (tid == 0) {
        a.accepted[b] = v.row;
        if (a.lens_out) a.lens_out[b] = a.lens[b] - (s.count ? s.count - 1 - v.row : 0);
    }
    if (!s.count || v.p.m == -INFINITY || !(t > 0.f)) {
        if (tid == 0) a.next[b] = !s.count || v.p.m == -INFINITY ? -1 : static_cast<int32_t>(v.p.at);
        return;
    }
    const Part *const parts = a.part + (s.first + v.row) * static_cast<int64_t>(a.parts);
    for (int residual = v.refused ? 1 : 0; residual >= 0; --residual) {
        const L left(a, s, v, t, residual != 0);
        // the parts' weights: p's from the first pass, less a token that was named
        for (int i = tid; i < a.parts; i += kThreads)
            mass[i] = left.minus ? a.left[b * a.parts + i] : parts[i].m == -INFINITY ? 0.0 : parts[i].sum * weight(parts[i].m, v.p.m, left.c) * left.pz;
        if (left.token >= 0) {
            const int i = (left.token + left.x.shift) / kPartLogits;
            const double m = part_sum(left, i, waves);
            if (tid == 0) mass[i] = m;
        }
        __syncthreads();
        if (wave == 0) {
            double total = 0.0;
            for (int i = lane; i < a.parts; i += 64) total += mass[i];
            total = wave_sum(total);
            const double want = static_cast<double>(a.u_next[b]) * total;
            double cum = 0.0, at = 0.0;
            int last = -1;
            for (int i0 = 0; i0 < a.parts; i0 += 64) {
                const double m = i0 + lane < a.parts ? mass[i0 + lane] : 0.0, end = cum + wave_scan(m);
                const uint64_t has = __ballot(m > 0.0), past = __ballot(m > 0.0 && end > want);
                if (has | past) {
                    const int i = past ? __ffsll(static_cast<long long>(past)) - 1 : 63 - __clzll(static_cast<long long>(has));
                    last = i0 + i;
                    at = __shfl(end, i, 64) - __shfl(m, i, 64);
                    if (past) break;
                }
                cum = __shfl(end, 63, 64);
            }
            if (lane == 0) chosen = last, before = want - at;
        }
        __syncthreads();
        const int part = chosen;
        double want = before;
        if (part < 0) {  // nothing left of p: drawn from p itself
            __syncthreads();
            continue;
        }
        double sum[L::kVec];
        left.sums(part, sum);
#pragma unroll
        for (int k = 0; k < L::kVec; ++k) {
            const double w = wave_sum(sum[k]);
            if (lane == 0) seg[k * kWaves + wave] = w;
        }
        __syncthreads();
        int at = -1;
        bool passed = false;
        double cum = 0.0, start = 0.0;
        for (int i = 0; i < kSegs && !passed; ++i) {
            if (seg[i] > 0.0) at = i, start = cum, passed = cum + seg[i] > want;
            cum += seg[i];
        }
        if (at % kWaves == wave) {
            const int q = part * (kPartLogits / L::VL) + at / kWaves * kThreads + tid;
            double r[L::VL], mine = 0.0;
            left.weights(q, r);
#pragma unroll
            for (int e = 0; e < L::VL; ++e) mine += r[e];
            const double end = start + wave_scan(mine);
            const uint64_t has = __ballot(mine > 0.0), past = __ballot(mine > 0.0 && end > want);
            const int from = past ? __ffsll(static_cast<long long>(past)) - 1 : 63 - __clzll(static_cast<long long>(has));
            if (lane == from) {
                double c2 = end - mine;
                int token = -1;
                bool done = false;
#pragma unroll
                for (int e = 0; e < L::VL; ++e) {
                    c2 += r[e];
                    if (!done && r[e] > 0.0) token = left.x.first(q) + e, done = c2 > want;
                }
                a.next[b] = token;
            }
        }
        return;
    }
}

template <typename T, typename D>
int launch_verify(const VerifyArgs &a, unsigned seqs, hipStream_t s) {
    int st = OURO_OK;
    if (a.r.max_new) {
        hipLaunchKernelGGL((verify_part_kernel<T, D>), dim3(a.parts, (a.x[1] ? 2 : 1) * a.r.max_new, seqs), dim3(kThreads), 0, s, a);
        if ((st = check_launch("verify_part_kernel"))) return st;
    }
    if (a.x[1] && a.r.max_new > 1) {
        hipLaunchKernelGGL((verify_left_kernel<T, D>), dim3(a.parts, seqs), dim3(kThreads), 0, s, a);
        if ((st = check_launch("verify_left_kernel"))) return st;
    }
    hipLaunchKernelGGL((verify_next_kernel<T, D>), dim3(seqs), dim3(kThreads), 0, s, a);
    return check_launch("verify_next_kernel");
}

// A part's logits begin at a multiple of 16 bytes, before the row's first where
// that is not one: up to 7 places more than the row has.
size_t parts_of(size_t n) { return (n + 7 + kPartLogits - 1) / kPartLogits; }
size_t up(size_t x) { return (x + 255) & ~size_t{255}; }

}  // namespace
}  // namespace ouro

using namespace ouro;

extern "C" {

size_t ouro_verify_drafts_workspace_bytes(size_t seqs, size_t rows, size_t n) {
    const size_t parts = parts_of(n);
    return up(2 * rows * parts * sizeof(Part)) + up(seqs * parts * sizeof(double));
}

int ouro_verify_drafts(const void *logits, int dtype, size_t row_stride, const void *draft, int draft_dtype, size_t draft_stride,
                       const int32_t *tokens, const int32_t *cu, size_t seqs, size_t rows, size_t max_new, size_t n,
                       const float *temperature, const float *u_accept, const float *u_next, const int32_t *lens, int32_t *accepted,
                       int32_t *next, int32_t *lens_out, void *ws, void *stream) {
    OURO_REQUIRE_INIT();
    const char *const me = "ouro_verify_drafts";
    if (!logits || !tokens || !u_accept || !u_next || !accepted || !next || (lens_out && !lens))
        return fail(OURO_ERR_INVALID_ARG, "%s: NULL argument", me);
    if ((dtype != OURO_DT_F32 && dtype != OURO_DT_BF16) || (draft && draft_dtype != OURO_DT_F32 && draft_dtype != OURO_DT_BF16))
        return fail(OURO_ERR_INVALID_ARG, "%s: dtypes %d and %d", me, dtype, draft_dtype);
    if (n < 1 || n >= (1u << 24)) return fail(OURO_ERR_SHAPE, "%s: %zu logits a row (1 .. 2^24 - 1)", me, n);
    VerifyArgs a{};
    int st = new_rows(tokens, cu, seqs, rows, max_new, 0, me, &a.r);
    if (st) return st;
    a.r.lens = nullptr;
    if (a.r.max_new > 32767) return fail(OURO_ERR_SHAPE, "%s: %d rows of a sequence (up to 32767)", me, a.r.max_new);
    if (!row_stride) row_stride = n;
    if (!draft_stride) draft_stride = n;
    if (row_stride < n || draft_stride < n || row_stride > (size_t{1} << 32) || draft_stride > (size_t{1} << 32))
        return fail(OURO_ERR_SHAPE, "%s: a stride shorter than its row, or past 2^32", me);
    const bool half = dtype == OURO_DT_BF16, dhalf = draft && draft_dtype == OURO_DT_BF16;
    if (reinterpret_cast<uintptr_t>(logits) & (half ? 1 : 3) || reinterpret_cast<uintptr_t>(draft) & (dhalf ? 1 : 3))
        return fail(OURO_ERR_ALIGN, "%s: rows must start at multiples of their element", me);
    if (!seqs) return OURO_OK;
    a.x[0] = logits, a.x[1] = draft;
    a.stride[0] = static_cast<int64_t>(row_stride), a.stride[1] = static_cast<int64_t>(draft_stride);
    a.tokens = tokens, a.lens = lens, a.temperature = temperature, a.u_accept = u_accept, a.u_next = u_next;
    a.accepted = accepted, a.next = next, a.lens_out = lens_out;
    a.n = static_cast<int>(n), a.parts = static_cast<int>(parts_of(n));
    const size_t need = ouro_verify_drafts_workspace_bytes(seqs, rows, n);
    if (need && !ws && !(ws = workspace(need, stream))) return OURO_ERR_HIP;
    a.part = static_cast<Part *>(ws);
    a.left = reinterpret_cast<double *>(static_cast<unsigned char *>(ws) + up(2 * rows * static_cast<size_t>(a.parts) * sizeof(Part)));
    const unsigned B = static_cast<unsigned>(seqs);
    hipStream_t s = as_stream(stream);
    if (half) return dhalf ? launch_verify<uint16_t, uint16_t>(a, B, s) : launch_verify<uint16_t, float>(a, B, s);
    return dhalf ? launch_verify<float, uint16_t>(a, B, s) : launch_verify<float, float>(a, B, s);
}

}  // extern "C"
