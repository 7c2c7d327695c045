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
// exponentials, sums and comparisons are made in 64 bits, exponentials within 1.1e-12:
// once in some million.  The logits are read in their own type, and it is their
// differences that are scaled.
#include "logits.hpp"

#include "kv_cache.hpp"

#include <cmath>

namespace ouro {
namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kSegLogits = 2048;  // logits of a segment: 32 a lane of a wavefront
constexpr double kLog2e = 1.4426950408889634;

// Maximum, its lowest index and the sum of e^((x - m) / T) of a segment of a row.
struct Seg {
    double sum;
    float m;
    uint32_t at;
};
static_assert(sizeof(Seg) == 16, "Seg: workspace layout");

// A row's, brought together.
struct Sums {
    double z;
    float m;
    uint32_t at;
};
// What a sequence came to: its deciding row (relative), whether that refused its
// token, the row's sums of p and q, the token (-1: none in the vocabulary).
struct Verdict {
    Sums p, q;
    int32_t row, refused, token, pad;
};
static_assert(sizeof(Verdict) == 48, "Verdict: workspace layout");

struct VerifyArgs {
    NewRows r;
    const void *x[2];  // logits, draft
    int64_t stride[2];
    const int32_t *tokens, *lens;
    const float *temperature, *u_accept, *u_next;
    int32_t *accepted, *next, *lens_out;
    Seg *seg;          // [2][rows][segs]
    double *left;      // [seqs][segs]: sums of max(p - q, 0)
    Verdict *verdict;  // [seqs], NULL where the last launch judges the rows itself
    int32_t n, segs;
};
static_assert(sizeof(VerifyArgs) == 160, "VerifyArgs: kernel argument layout");

// 2^y, y finite: y = k + f, |f| <= 1/2, and the polynomial of degree 8 that equals 2^f
// at the nine Chebyshev points of [-1/2, 1/2], within 1.1e-12 of it between them and 1
// at 0.
__device__ __forceinline__ double exp2_finite(double y) {
    const double k = rint(y), f = y - k;
    double s = 0x1.63d136366db24p-20;
    s = fma(s, f, 0x1.00dc4a532fb8ep-16);
    s = fma(s, f, 0x1.4308ac85aa947p-13);
    s = fma(s, f, 0x1.5d8745a728441p-10);
    s = fma(s, f, 0x1.3b2ab7181b755p-7);
    s = fma(s, f, 0x1.c6b08dd6fd234p-5);
    s = fma(s, f, 0x1.ebfbdff823cedp-3);
    s = fma(s, f, 0x1.62e42fef84cf0p-1);
    s = fma(s, f, 1.0);
    return __builtin_amdgcn_ldexp(s, static_cast<int>(k));
}
// 2^y, 0 below 2^-1074 and for NaN.
__device__ __forceinline__ double exp2_64(double y) { return exp2_finite(fmax(y, -2000.0)); }
// 2^y, 0 at 2^-1000 and below and for NaN, so that a product of what is not 0 never is: the
// upper half of y becomes that of -2000.  (A sum against its largest term does not see
// what this leaves out, and does without: 2 us of verify_segments_kernel's 65.)
__device__ __forceinline__ double exp2_held(double y) {
    return exp2_finite(__hiloint2double(y > -1000.0 ? __double2hiint(y) : static_cast<int>(0xc09f4000u), __double2loint(y)));
}
// e^((x - m) / T), c = log2 e / T, x <= m: 1 where x = m, infinite or not.
__device__ __forceinline__ double weight(float x, float m, double c) {
    return x == m ? 1.0 : exp2_held((static_cast<double>(x) - static_cast<double>(m)) * c);
}
// Lane `lane`'s value, the same lane for all.
__device__ __forceinline__ double lane64(double v, int lane) {
    const uint64_t u = __double_as_longlong(v);
    const uint32_t lo = __builtin_amdgcn_readlane(static_cast<uint32_t>(u), lane), hi = __builtin_amdgcn_readlane(static_cast<uint32_t>(u >> 32), lane);
    return __longlong_as_double(static_cast<long long>(static_cast<uint64_t>(hi) << 32 | lo));
}
// v plus that of the lane that a data-parallel move names, 0 where it names none.
template <int Ctrl, int Rows>
__device__ __forceinline__ double plus_dpp(double v) {
    const uint64_t u = __double_as_longlong(v);
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, static_cast<uint32_t>(u), Ctrl, Rows, 0xf, false);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, static_cast<uint32_t>(u >> 32), Ctrl, Rows, 0xf, false);
    return v + __longlong_as_double(static_cast<long long>(static_cast<uint64_t>(hi) << 32 | lo));
}
// Inclusive sums over a wavefront's lanes: over each row of 16 lanes by moves of 1,
// 2, 4 and 8, then the last lane of rows 0 and 2 to rows 1 and 3, and lane 31 to
// both of them.  (Lane exchanges through LDS instead: 0.5 us a sum.)
__device__ __forceinline__ double wave_scan(double v) {
    v = plus_dpp<0x111, 0xf>(v);
    v = plus_dpp<0x112, 0xf>(v);
    v = plus_dpp<0x114, 0xf>(v);
    v = plus_dpp<0x118, 0xf>(v);
    v = plus_dpp<0x142, 0xa>(v);
    return plus_dpp<0x143, 0xc>(v);
}
__device__ __forceinline__ double wave_sum(double v) { return lane64(wave_scan(v), 63); }
// Over the 64 lanes: within rows of 16 by moves, across them by swaps.
template <typename F>
__device__ __forceinline__ uint32_t wave_join(uint32_t v, F f) {
    v = f(v, __builtin_amdgcn_update_dpp(0, v, 0x128, 0xf, 0xf, false));
    v = f(v, __builtin_amdgcn_update_dpp(0, v, 0x141, 0xf, 0xf, false));
    v = f(v, __builtin_amdgcn_update_dpp(0, v, 0x4E, 0xf, 0xf, false));
    v = f(v, __builtin_amdgcn_update_dpp(0, v, 0xB1, 0xf, 0xf, false));
    const auto a = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    v = f(a[0], a[1]);
    const auto b = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return f(b[0], b[1]);
}
__device__ __forceinline__ float wave_max(float v) {
    return __uint_as_float(wave_join(__float_as_uint(v), [](uint32_t a, uint32_t b) { return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b))); }));
}
__device__ __forceinline__ uint32_t wave_min(uint32_t v) {
    return wave_join(v, [](uint32_t a, uint32_t b) { return min(a, b); });
}
// The likeliest token is taken where the temperature is not above 0.
__device__ __forceinline__ float heat(const VerifyArgs &a, int64_t b) { return a.temperature ? a.temperature[b] : 1.f; }

template <typename T>
__device__ __forceinline__ LogitRow<T> row_at(const VerifyArgs &a, int which, int64_t row) {
    return LogitRow<T>(static_cast<const T *>(a.x[which]) + row * a.stride[which], a.n);
}

// A segment by one wavefront: its maximum and, as the row is drawn from or not,
// the sum against it or the maximum's lowest index.
template <typename T>
__device__ __forceinline__ void segment(const VerifyArgs &a, int which, int64_t row, int seg, float t, Seg *out) {
    constexpr int VL = LogitRow<T>::VL, kVec = 32 / VL;
    const int lane = threadIdx.x & 63;
    const LogitRow<T> x = row_at<T>(a, which, row);
    const int q0 = seg * (kSegLogits / VL) + lane;
    u32x4_t v[kVec];
#pragma unroll
    for (int k = 0; k < kVec; ++k) v[k] = x.load(q0 + 64 * k);
    float m = -INFINITY;
#pragma unroll
    for (int k = 0; k < kVec; ++k)
#pragma unroll
        for (int e = 0; e < VL; ++e) m = fmaxf(m, x.raw(v[k], e));  // passes over a NaN
    m = wave_max(m);
    double sum = 0.0;
    uint32_t at = 0xffffffffu;
    if (!(t > 0.f) && m > -INFINITY) {
#pragma unroll
        for (int k = 0; k < kVec; ++k)
#pragma unroll
            for (int e = 0; e < VL; ++e)
                if (x.raw(v[k], e) == m) at = min(at, static_cast<uint32_t>(x.first(q0 + 64 * k) + e));
        at = wave_min(at);
    } else if (m == INFINITY) {
#pragma unroll
        for (int k = 0; k < kVec; ++k)
#pragma unroll
            for (int e = 0; e < VL; ++e) sum += x.raw(v[k], e) == m ? 1.0 : 0.0;
        sum = wave_sum(sum);
    } else if (m > -INFINITY) {
        const double c = kLog2e / static_cast<double>(t), md = static_cast<double>(m);
#pragma unroll
        for (int k = 0; k < kVec; ++k)
#pragma unroll
            for (int e = 0; e < VL; ++e) sum += exp2_64((static_cast<double>(x.raw(v[k], e)) - md) * c);
        sum = wave_sum(sum);
    }
    if (lane == 0) *out = Seg{sum, m, at};
}

// A wavefront a segment, of the target's rows and then of the drafter's.  No
// barrier and no LDS: what a wavefront waits for is its 8 KiB of logits.  64
// sequences of up to four drafted tokens over 248320 logits, 308 MB (the drafter's rows of
// greedy sequences are not read): 65 us at 4.7 TB/s where a copy has 5 (18 instructions in
// 64 bits a logit are some 35 of it; workgroups of 8192 logits and a polynomial of degree
// 11 took 107).
template <typename T, typename D>
__global__ __launch_bounds__(kThreads) void verify_segments_kernel(VerifyArgs a) {
    const int which = static_cast<int>(blockIdx.y) / a.r.max_new, i = static_cast<int>(blockIdx.y) % a.r.max_new;
    const int seg = static_cast<int>(blockIdx.x) * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const SeqRows s = seq_rows(a.r, blockIdx.z);
    if (i >= s.count - which || seg >= a.segs) return;  // the last row has no token to judge
    const float t = heat(a, blockIdx.z);
    if (which && !(t > 0.f)) return;
    const int64_t row = s.first + i;
    Seg *out = a.seg + (static_cast<int64_t>(which) * a.r.rows + row) * a.segs + seg;
    if (which)
        segment<D>(a, 1, row, seg, 1.f, out);
    else
        segment<T>(a, 0, row, seg, t, out);
}

// A row's segments brought together by one wavefront, to each of its lanes.
__device__ __forceinline__ Sums join_segments(const VerifyArgs &a, int which, int64_t row, bool draws, double c) {
    const Seg *p = a.seg + (static_cast<int64_t>(which) * a.r.rows + row) * a.segs;
    const int lane = threadIdx.x & 63;
    constexpr int kHeld = 2;  // of a lane, that are read once
    Seg held[kHeld];
    Sums s{0.0, -INFINITY, 0xffffffffu};
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
        held[i] = Seg{0.0, -INFINITY, 0xffffffffu};
        if (lane + 64 * i < a.segs) held[i] = p[lane + 64 * i];
    }
#pragma unroll
    for (int i = 0; i < kHeld; ++i) s.m = fmaxf(s.m, held[i].m);
    for (int i = lane + 64 * kHeld; i < a.segs; i += 64) s.m = fmaxf(s.m, p[i].m);
    s.m = wave_max(s.m);
    auto add = [&](const Seg &x) {
        if (x.m == -INFINITY) return;
        if (draws) s.z += x.sum * weight(x.m, s.m, c);
        if (x.m == s.m) s.at = min(s.at, x.at);
    };
#pragma unroll
    for (int i = 0; i < kHeld; ++i) add(held[i]);
    for (int i = lane + 64 * kHeld; i < a.segs; i += 64) add(p[i]);
    if (draws)
        s.z = wave_sum(s.z);
    else
        s.at = wave_min(s.at);
    return s;
}

// The rows of a sequence judged, a wavefront each, up to the first that refuses.
template <typename T, typename D>
__device__ __forceinline__ Verdict decide(const VerifyArgs &a, const SeqRows &s, float t, Verdict *lds) {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const bool draws = t > 0.f;
    const double c = draws ? kLog2e / static_cast<double>(t) : 0.0;
    for (int i0 = 0; i0 < s.count; i0 += kWaves) {
        const int i = i0 + wave;
        if (i < s.count) {
            const int64_t row = s.first + i;
            const bool judges = i + 1 < s.count;
            const int next = judges ? a.tokens[row + 1] : -1;
            const bool in = next >= 0 && next < a.n;
            float x = -INFINITY, y = -INFINITY, u = 0.f;
            if (in && draws) {  // on their way while the segments are joined
                u = a.u_accept[row];
                x = logit(row_at<T>(a, 0, row).x, next);
                if (a.x[1]) y = logit(row_at<D>(a, 1, row).x, next);
            }
            Verdict v{};
            v.row = i;
            v.p = join_segments(a, 0, row, draws, c);
            if (judges && draws && a.x[1]) v.q = join_segments(a, 1, row, true, kLog2e);
            v.token = in ? next : -1;
            if (judges) {
                bool keep = in && v.p.m > -INFINITY;
                if (!draws) {
                    keep = keep && static_cast<uint32_t>(next) == v.p.at;
                } else if (keep) {
                    const double q = !a.x[1] ? 1.0 : v.q.m > -INFINITY ? weight(y, v.q.m, kLog2e) / v.q.z : 0.0;
                    keep = static_cast<double>(u) * q < weight(x, v.p.m, c) / v.p.z;
                }
                v.refused = !keep;
            }
            if ((threadIdx.x & 63) == 0) lds[wave] = v;
        }
        __syncthreads();
        for (int w = 0; w < kWaves; ++w)
            if (i0 + w < s.count && (lds[w].refused || i0 + w + 1 == s.count)) return lds[w];
        __syncthreads();
    }
    return Verdict{};  // no rows: not reached
}

// A distribution's values, e^((x - m) / T) / z.  The difference comes first here as in
// the sums: x c - m c with either product rounded is off by 2^-53 |m| / T, which is
// anything where the largest of many logits is a mask's 1e30 or T is 1e-18.
struct Share {
    double c, m, z;  // log2 e / T, the maximum, 1 / z
    float top;        // +inf where m is: the mass is that of the +inf logits, else NaN
    __device__ __forceinline__ Share() {}
    __device__ __forceinline__ Share(const Sums &s, double scale) : c(scale), m(static_cast<double>(s.m)), z(1.0 / s.z), top(s.m == INFINITY ? INFINITY : NAN) {}
    // Of a logit as it lies there: 0 for NaN and -inf.
    __device__ __forceinline__ double of(float x) const {
#pragma clang fp contract(off)
        if (top == INFINITY) return x == top ? z : 0.0;
        return exp2_held((static_cast<double>(x) - m) * c) * z;
    }
};

// What a token is drawn by: max(p - q, 0) where one was refused, p where none was
// or where nothing is left of it.
template <typename T, typename D>
struct Left {
    static constexpr int VL = LogitRow<T>::VL;
    LogitRow<T> x;
    LogitRow<D> y;
    Share p, q;
    int token;  // that a drafter without draft rows named, -1: none
    bool minus;
    __device__ __forceinline__ Left(const VerifyArgs &a, const SeqRows &s, const Verdict &v, float t, bool residual)
        : x(row_at<T>(a, 0, s.first + v.row)), y(row_at<D>(a, a.x[1] ? 1 : 0, s.first + v.row)), p(v.p, kLog2e / static_cast<double>(t)) {
        minus = residual && a.x[1] && v.q.m > -INFINITY;
        if (minus) q = Share(v.q, kLog2e);
        token = residual && !a.x[1] ? v.token : -1;
    }
    // The draft's values at the places of vector q of x.
    __device__ __forceinline__ void beside(int q, float (&g)[VL]) const {
        if (LogitRow<D>::VL == VL && x.shift == y.shift) {
            const u32x4_t v = y.load(q);
#pragma unroll
            for (int e = 0; e < VL; ++e) g[e] = y.raw(v, e);
        } else {
#pragma unroll
            for (int e = 0; e < VL; ++e) {
                const int i = x.first(q) + e;
                g[e] = i >= 0 && i < y.n ? logit(y.x, i) : -INFINITY;
            }
        }
    }
    // Of the elements of vector at; places outside the row hold -inf.  Both products
    // are rounded before they are subtracted, so that equal p and q leave nothing.
    __device__ __forceinline__ void weights(int at, double (&r)[VL]) const {
#pragma clang fp contract(off)
        const u32x4_t v = x.load(at);
        float g[VL];
        if (minus) beside(at, g);
#pragma unroll
        for (int e = 0; e < VL; ++e) {
            r[e] = p.of(x.raw(v, e));
            if (minus) r[e] = fmax(r[e] - q.of(g[e]), 0.0);
            if (token >= 0 && x.first(at) + e == token) r[e] = 0.0;
        }
    }
    // A lane's sum of vectors q, q + 64, ..
    template <int N>
    __device__ __forceinline__ double sum(int q) const {
        double s = 0.0;
#pragma unroll
        for (int k = 0; k < N; ++k) {
            double r[VL];
            weights(q + 64 * k, r);
#pragma unroll
            for (int e = 0; e < VL; ++e) s += r[e];
        }
        return s;
    }
};

__device__ __forceinline__ void say(const VerifyArgs &a, int64_t b, const SeqRows &s, int kept) {
    a.accepted[b] = kept;
    if (a.lens_out) a.lens_out[b] = a.lens[b] - (s.count ? s.count - 1 - kept : 0);
}

// Every workgroup of a sequence judges its rows (all wait for the same few
// kilobytes); where a token was refused each wavefront then sums max(p - q, 0)
// over a segment of that row.  64 sequences of up to four drafted tokens over
// 248320 logits, some 90 MB of refusing rows: 34 us; the judging in a launch of
// its own 8 + 25 us where this took 33, and one launch more, two segments a wavefront 43.
template <typename T, typename D>
__global__ __launch_bounds__(kThreads) void verify_left_kernel(VerifyArgs a) {
    constexpr int VL = Left<T, D>::VL;
    __shared__ Verdict lds[kWaves];
    const int64_t b = blockIdx.y;
    const SeqRows s = seq_rows(a.r, b);
    const float t = heat(a, b);
    if (s.count == 0) return;  // whole workgroup
    const Verdict v = decide<T, D>(a, s, t, lds);
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        a.verdict[b] = v;
        say(a, b, s, v.row);
    }
    const int seg = static_cast<int>(blockIdx.x) * kWaves + static_cast<int>(threadIdx.x >> 6);
    if (!v.refused || !(t > 0.f) || v.p.m == -INFINITY || seg >= a.segs) return;
    const Left<T, D> left(a, s, v, t, true);
    const double sum = wave_sum(left.template sum<32 / VL>(seg * (kSegLogits / VL) + (threadIdx.x & 63)));
    if ((threadIdx.x & 63) == 0) a.left[b * a.segs + seg] = sum;
}

// The next token of a sequence: the segment in which the cumulative sum passes u'
// of the whole, in it the wavefront's quarter, the lane, the element.  Sums that
// are made in two orders differ by roundings: where none passes, the last with
// any weight is taken, so that a token of weight 0 never is.
template <typename T, typename D>
__global__ __launch_bounds__(kThreads) void verify_next_kernel(VerifyArgs a) {
    using L = Left<T, D>;
    constexpr int VL = L::VL, kQuarter = kSegLogits / kWaves / VL, kVec = kQuarter / 64;
    __shared__ Verdict lds[kWaves];
    __shared__ double part[kWaves * kVec];
    const int64_t b = blockIdx.x;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const SeqRows s = seq_rows(a.r, b);
    const float t = heat(a, b);
    Verdict v{};
    if (s.count) v = a.verdict ? a.verdict[b] : decide<T, D>(a, s, t, lds);
    if (tid == 0 && (!a.verdict || !s.count)) say(a, b, s, v.row);
    if (!s.count || v.p.m == -INFINITY || !(t > 0.f)) {
        if (tid == 0) a.next[b] = !s.count || v.p.m == -INFINITY ? -1 : static_cast<int32_t>(v.p.at);
        return;
    }
    const Seg *const segs = a.seg + (s.first + v.row) * static_cast<int64_t>(a.segs);
    for (int residual = v.refused ? 1 : 0; residual >= 0; --residual) {
        const L left(a, s, v, t, residual != 0);
        // the segment of a token that was named, without it
        int named = -1;
        double rest = 0.0;
        if (left.token >= 0) {
            named = (left.token + left.x.shift) / kSegLogits;
            const double sum = wave_sum(left.template sum<kVec>(named * (kSegLogits / VL) + wave * kQuarter + lane));
            if (lane == 0) part[wave] = sum;
            __syncthreads();
            for (int w = 0; w < kWaves; ++w) rest += part[w];
            __syncthreads();
        }
        // the segments' weights: p's from the first pass
        auto mass = [&](int i) {
            if (i >= a.segs) return 0.0;
            if (left.minus) return a.left[b * a.segs + i];
            if (i == named) return rest;
            const Seg x = segs[i];
            return x.m == -INFINITY ? 0.0 : x.sum * weight(x.m, v.p.m, left.p.c) * left.p.z;
        };
        double total = 0.0, want, cum = 0.0, at = 0.0;
        for (int i = lane; i < a.segs; i += 64) total += mass(i);
        want = static_cast<double>(a.u_next[b]) * wave_sum(total);
        int seg = -1;
        for (int i0 = 0; i0 < a.segs; i0 += 64) {
            const double m = mass(i0 + lane), end = cum + wave_scan(m);
            const uint64_t has = __ballot(m > 0.0), past = __ballot(m > 0.0 && end > want);
            if (has) {
                const int i = past ? __ffsll(static_cast<long long>(past)) - 1 : 63 - __clzll(static_cast<long long>(has));
                seg = i0 + i;
                at = lane64(end, i) - lane64(m, i);
                if (past) break;
            }
            cum = lane64(end, 63);
        }
        if (seg < 0) continue;  // nothing left of p: drawn from p itself
        want -= at;
        const int q0 = seg * (kSegLogits / VL) + wave * kQuarter + lane;
        double r[kVec][VL], mine[kVec];
#pragma unroll
        for (int k = 0; k < kVec; ++k) {
            left.weights(q0 + 64 * k, r[k]);
            mine[k] = 0.0;
#pragma unroll
            for (int e = 0; e < VL; ++e) mine[k] += r[k][e];
            const double w = wave_sum(mine[k]);
            if (lane == 0) part[wave * kVec + k] = w;
        }
        __syncthreads();
        int from = -1;
        bool passed = false;
        cum = 0.0;
        double start = 0.0;
        for (int i = 0; i < kWaves * kVec && !passed; ++i) {
            if (part[i] > 0.0) from = i, start = cum, passed = cum + part[i] > want;
            cum += part[i];
        }
        if (from < 0 && tid == 0) a.next[b] = -1;  // as below
#pragma unroll
        for (int k = 0; k < kVec; ++k)
            if (from == wave * kVec + k) {
                const double end = start + wave_scan(mine[k]);
                const uint64_t has = __ballot(mine[k] > 0.0), past = __ballot(mine[k] > 0.0 && end > want);
                const int who = past ? __ffsll(static_cast<long long>(past)) - 1 : 63 - __clzll(static_cast<long long>(has));
                if (lane == who) {
                    double c2 = end - mine[k];
                    int token = -1;
                    bool done = false;
#pragma unroll
                    for (int e = 0; e < VL; ++e) {
                        c2 += r[k][e];
                        if (!done && r[k][e] > 0.0) token = left.x.first(q0 + 64 * k) + e, done = c2 > want;
                    }
                    a.next[b] = token;
                }
            }
        return;
    }
    // Not reached where sequences have rows of their own: p has its maximum's mass.  Rows
    // that two share hold the sums of one, which may have been greedy and made none.
    if (tid == 0) a.next[b] = -1;
}

template <typename T, typename D>
int launch_verify(VerifyArgs a, unsigned seqs, hipStream_t s) {
    const unsigned groups = static_cast<unsigned>((a.segs + kWaves - 1) / kWaves);
    int st = OURO_OK;
    if (a.r.max_new) {
        hipLaunchKernelGGL((verify_segments_kernel<T, D>), dim3(groups, (a.x[1] ? 2 : 1) * a.r.max_new, seqs), dim3(kThreads), 0, s, a);
        if ((st = check_launch("verify_segments_kernel"))) return st;
    }
    if (a.x[1] && a.r.max_new > 1) {
        hipLaunchKernelGGL((verify_left_kernel<T, D>), dim3(groups, seqs), dim3(kThreads), 0, s, a);
        if ((st = check_launch("verify_left_kernel"))) return st;
    } else {
        a.verdict = nullptr;
    }
    hipLaunchKernelGGL((verify_next_kernel<T, D>), dim3(seqs), dim3(kThreads), 0, s, a);
    return check_launch("verify_next_kernel");
}

// A row's segments begin at a multiple of 16 bytes, before its first logit where
// that is not one: up to 7 places more than the row has.
size_t segs_of(size_t n) { return (n + 7 + kSegLogits - 1) / kSegLogits; }
struct VerifyWs {
    size_t left, verdict, bytes;
};
VerifyWs verify_ws(size_t seqs, size_t rows, size_t n) {
    auto up = [](size_t x) { return (x + 255) & ~size_t{255}; };
    VerifyWs w{};
    w.left = up(2 * rows * segs_of(n) * sizeof(Seg));
    w.verdict = w.left + up(seqs * segs_of(n) * sizeof(double));
    w.bytes = w.verdict + up(seqs * sizeof(Verdict));
    return w;
}

}  // namespace
}  // namespace ouro

using namespace ouro;

extern "C" {

size_t ouro_verify_drafts_workspace_bytes(size_t seqs, size_t rows, size_t n) { return verify_ws(seqs, rows, n).bytes; }

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
    a.n = static_cast<int>(n), a.segs = static_cast<int>(segs_of(n));
    const VerifyWs w = verify_ws(seqs, rows, n);
    if (!ws && !(ws = workspace(w.bytes, stream))) return OURO_ERR_HIP;
    unsigned char *const p = static_cast<unsigned char *>(ws);
    a.seg = reinterpret_cast<Seg *>(p);
    a.left = reinterpret_cast<double *>(p + w.left);
    a.verdict = reinterpret_cast<Verdict *>(p + w.verdict);
    const unsigned B = static_cast<unsigned>(seqs);
    hipStream_t s = as_stream(stream);
    if (half) return dhalf ? launch_verify<uint16_t, uint16_t>(a, B, s) : launch_verify<uint16_t, float>(a, B, s);
    return dhalf ? launch_verify<float, uint16_t>(a, B, s) : launch_verify<float, float>(a, B, s);
}

}  // extern "C"
