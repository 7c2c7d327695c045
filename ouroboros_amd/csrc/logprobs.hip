// logprobs.hip - log probabilities of given tokens from rows of logits, with
// their rank, the entropy and the likeliest alternatives.
//
// Of a row x: m = max x, l = sum e^(x - m), lse = m + ln l,
//   logprob(t) = (x_t - m) - ln l,
//   entropy    = ln l - (1 / l) sum e^(x - m) (x - m),
//   rank(t)    = the number of tokens ahead of t by (larger x, lower index),
// the alternatives in that order.  A NaN counts as -inf (finite_argmax passes
// over it too, infer/mod.rs:70-83), x - m as 0 where x = m (so that m = +inf
// shares the mass among the +inf logits), e^(x - m) (x - m) as 0 where
// e^(x - m) = 0.
#include "common.hpp"

namespace ouro {
namespace {

constexpr int kThreads = 256;
constexpr int kLogits = 32;                 // logits of a thread
constexpr int kPartLogits = kThreads * kLogits;
constexpr int kRowParts = 4;                // parts of a row that one workgroup takes whole, where rows are few
constexpr unsigned kFewRows = 512;          // such workgroups that the chip holds at once
constexpr int kSegs = kThreads / 16;        // segments of a part: 16 lanes each
constexpr int kJoin = 1024;                 // threads that join a row's parts
constexpr int kGroups = 256;                // groups of its segments
constexpr int kCap = 2048;                  // candidates that the choice of alternatives holds

struct ScoreArgs {
    const void *x;
    int64_t stride;
    const int32_t *target;
    float *logprob, *entropy, *lse, *top_logprob;
    int32_t *rank, *top_id;
    float4 *part;              // [rows][parts]: m, l, s, tokens ahead (as bits)
    unsigned long long *seg;   // [rows][parts * kSegs]: each segment's largest key
    int32_t n, k, parts, pad;
};
// passed by value to kernels: the host and device passes must lay it out alike
static_assert(sizeof(ScoreArgs) == 104, "ScoreArgs: kernel argument layout");

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));

template <typename T>
__device__ __forceinline__ float logit(const T *x, int64_t i) {
    float v;
    if constexpr (sizeof(T) == 4)
        v = x[i];
    else
        v = bf16_bits_to_f32(x[i]);
    return v != v ? -INFINITY : v;
}

// A row in 16-byte vectors from the last multiple of 16 bytes at or before its
// start: vector q holds elements q VL - shift .. q VL - shift + VL - 1.
template <typename T>
struct Row {
    static constexpr int VL = 16 / sizeof(T);
    static constexpr int kVec = kLogits / VL;         // vectors of a thread
    static constexpr int kPart = kPartLogits / VL;    // and of a part
    const T *x;
    int n, shift;
    __device__ __forceinline__ Row(const ScoreArgs &a, int64_t row) : x(static_cast<const T *>(a.x) + row * a.stride), n(a.n) {
        shift = static_cast<int>((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
    }
    __device__ __forceinline__ int first(int q) const { return q * VL - shift; }
    // Vector q as bits: whole where it lies in the row, else its elements one by
    // one with -inf in the places of others.
    __device__ __forceinline__ u32x4_t load(int q) const {
        const int e0 = first(q);
        if (e0 >= 0 && e0 + VL <= n) return *reinterpret_cast<const u32x4_t *>(x + e0);
        u32x4_t r;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            if constexpr (sizeof(T) == 4) {
                const int e = e0 + w;
                r[w] = e >= 0 && e < n ? __float_as_uint(x[e]) : 0xff800000u;
            } else {
                const int e = e0 + 2 * w;
                const uint32_t lo = e >= 0 && e < n ? x[e] : 0xff80u, hi = e + 1 >= 0 && e + 1 < n ? x[e + 1] : 0xff80u;
                r[w] = lo | hi << 16;
            }
        }
        return r;
    }
    // Element e of a vector as it is, and with NaN as -inf.
    static __device__ __forceinline__ float raw(const u32x4_t &v, int e) {
        if constexpr (sizeof(T) == 4) return __uint_as_float(v[e]);
        return __uint_as_float(e & 1 ? v[e >> 1] & 0xffff0000u : v[e >> 1] << 16);
    }
    static __device__ __forceinline__ float at(const u32x4_t &v, int e) {
        const float f = raw(v, e);
        return f != f ? -INFINITY : f;
    }
};

// Over the 16 lanes of a row of the wavefront, to each of them.
template <typename F>
__device__ __forceinline__ uint32_t row16(uint32_t v, F f) {
    v = f(v, __builtin_amdgcn_update_dpp(0, v, 0x128, 0xf, 0xf, false));
    v = f(v, __builtin_amdgcn_update_dpp(0, v, 0x141, 0xf, 0xf, false));
    v = f(v, __builtin_amdgcn_update_dpp(0, v, 0x4E, 0xf, 0xf, false));
    return f(v, __builtin_amdgcn_update_dpp(0, v, 0xB1, 0xf, 0xf, false));
}
__device__ __forceinline__ float row16_max(float v) {
    return __uint_as_float(row16(__float_as_uint(v), [](uint32_t a, uint32_t b) { return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b))); }));
}

// (m, l, s) of two sets of logits: l = sum e^(x - m), s = sum e^(x - m) (x - m).
__device__ __forceinline__ void merge(float &m, float &l, float &s, float m2, float l2, float s2) {
    const float M = fmaxf(m, m2);
    const float d1 = m == M ? 0.f : m - M, d2 = m2 == M ? 0.f : m2 - M;  // -inf where a set is empty beside the other
    const float f1 = expf(d1), f2 = expf(d2);
    s = (f1 > 0.f ? f1 * (s + d1 * l) : 0.f) + (f2 > 0.f ? f2 * (s2 + d2 * l2) : 0.f);
    l = f1 * l + f2 * l2;
    m = M;
}

// What a row's sums say, written by one thread; g the given token, xt its logit.
__device__ __forceinline__ void finish(const ScoreArgs &a, int64_t row, int g, float xt, float m, float l, float s, int ahead) {
    const float ln = logf(l);
    const bool empty = m == -INFINITY, given = g >= 0 && g < a.n;
    if (a.lse) a.lse[row] = empty ? -INFINITY : m + ln;
    if (a.entropy) a.entropy[row] = empty ? 0.f : ln - s / l;
    if (a.logprob) a.logprob[row] = !given ? 0.f : empty ? -INFINITY : (xt == m ? 0.f : xt - m) - ln;
    if (a.rank) a.rank[row] = given ? ahead : -1;
}

// The sums of a wavefront's lanes joined, to each of them; their maximum.
__device__ __forceinline__ float join_lanes(float m, float &l, float &s, int &ahead) {
    float M = m;
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) M = fmaxf(M, xor_shfl(M, off));
    if (M != -INFINITY) merge(m, l, s, M, 0.f, 0.f);  // against the largest
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) {
        l += xor_shfl(l, off);
        s += xor_shfl(s, off);
        ahead += xor_shfl(ahead, off);
    }
    return M;
}

// One workgroup a part of a row, its logits in registers: the wavefront's
// maximum, then the sums against it, then the tokens ahead of the given one
// and (Top) the largest key of each segment, that is of the vectors of 16
// lanes.  A row of one part is finished here.
//
// Bound by memory once the rows fill the chip: 512 rows of 248320 fp32 logits
// in 90 us (5.6 TB/s), 64 in 16 (4.0), 1009 rows of 32003 bf16 in 19 (3.4; of
// that 9 are the vector instructions, 12 a logit with its exponential).  A
// part of 8192 logits leaves each thread its 32 in registers, so that the
// maximum is known before the first exponential and nothing is read twice; 16
// bits hold twice as many in as many registers, but unpacked they take 183 and
// the launch of bf16 rows 40 us.
template <typename T, bool Top, int Parts>
__global__ __launch_bounds__(Parts * kThreads) void logprobs_part_kernel(ScoreArgs a) {
    constexpr int VL = Row<T>::VL, kVec = Row<T>::kVec, kPart = Row<T>::kPart;
    __shared__ float4 waves[Parts * kThreads / 64];
    const int tid = threadIdx.x % kThreads;
    const int64_t row = blockIdx.y;
    const Row<T> x(a, row);
    const int group = Parts == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x / kThreads);
    const int q0 = (static_cast<int>(blockIdx.x) * Parts + group) * kPart;
    u32x4_t v[kVec];
#pragma unroll
    for (int j = 0; j < kVec; ++j) {
        const int q = q0 + kThreads * j + tid;
        v[j] = u32x4_t{0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u};
        if constexpr (sizeof(T) == 2) v[j] = u32x4_t{0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u};
        if (x.first(q) < a.n) v[j] = x.load(q);
    }
    const int g = a.target ? a.target[row] : -1;
    const float xt = g >= 0 && g < a.n ? logit(x.x, g) : 0.f;
    const bool given = a.rank && g >= 0 && g < a.n;
    float mt = -INFINITY;
#pragma unroll
    for (int j = 0; j < kVec; ++j)
#pragma unroll
        for (int e = 0; e < VL; ++e) mt = fmaxf(mt, Row<T>::raw(v[j], e));  // passes over a NaN
    const float ms = row16_max(mt);
    float m = fmaxf(ms, xor_shfl(ms, 16));
    m = fmaxf(m, xor_shfl(m, 32));
    float l = 0.f, s = 0.f;
    if (m == INFINITY) {  // shared by the logits that are +inf
        for (int j = 0; j < kVec; ++j)
#pragma unroll
            for (int e = 0; e < VL; ++e) l += Row<T>::raw(v[j], e) == INFINITY ? 1.f : 0.f;
    } else if (m != -INFINITY) {
#pragma unroll
        for (int j = 0; j < kVec; ++j) {
            float lj = 0.f, sj = 0.f;  // short chains
#pragma unroll
            for (int e = 0; e < VL; ++e) {
                // the maximum takes a NaN and -inf alike to where e^d = 0 and e^d d = 0
                const float d = fmaxf(Row<T>::raw(v[j], e) - m, -3e38f);
                const float p = __builtin_amdgcn_exp2f(d * 1.4426950408889634f);
                lj += p;
                sj += p * d;
            }
            l += lj;
            s += sj;
        }
    }
    // tokens ahead, counted for the wavefront in scalar registers
    int ahead = 0;
    if (given) {
        const int lo = x.first(q0), hi = x.first(q0 + kPart);  // the part's elements
        if (xt != -INFINITY && hi <= g) {
#pragma unroll
            for (int j = 0; j < kVec; ++j)
#pragma unroll
                for (int e = 0; e < VL; ++e) ahead += __popcll(__ballot(Row<T>::raw(v[j], e) >= xt));
        } else if (lo > g) {
#pragma unroll
            for (int j = 0; j < kVec; ++j)
#pragma unroll
                for (int e = 0; e < VL; ++e) ahead += __popcll(__ballot(Row<T>::raw(v[j], e) > xt));
        } else {
            for (int j = 0; j < kVec; ++j)
#pragma unroll
                for (int e = 0; e < VL; ++e) {
                    const int i = x.first(q0 + kThreads * j + tid) + e;
                    const float f = Row<T>::at(v[j], e);
                    ahead += __popcll(__ballot(f > xt || (f == xt && i >= 0 && i < g)));
                }
        }
    }
    if constexpr (Top) {
        // the segment's largest logit at its lowest index
        uint32_t at = 0xffffffffu;
#pragma unroll
        for (int j = kVec - 1; j >= 0; --j)
#pragma unroll
            for (int e = VL - 1; e >= 0; --e)
                if (Row<T>::at(v[j], e) == ms) at = static_cast<uint32_t>(x.first(q0 + kThreads * j + tid) + e);
        at = row16(at, [](uint32_t p, uint32_t q) { return p < q ? p : q; });
        if (tid % 16 == 0)
            a.seg[(row * a.parts + blockIdx.x) * kSegs + tid / 16] = ms == -INFINITY ? 0ull : argmax_key(ms, at);
    }
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) {
        l += xor_shfl(l, off);
        s += xor_shfl(s, off);
    }
    if ((tid & 63) == 0) waves[threadIdx.x >> 6] = make_float4(m, l, s, __int_as_float(ahead));
    __syncthreads();
    // a part's wavefronts in order, by one lane
    if (threadIdx.x >= (Parts > 1 ? 64 : 1)) return;
    if (Parts == 1 || threadIdx.x < Parts) {
        const int w0 = threadIdx.x * (kThreads / 64);
        m = waves[w0].x, l = waves[w0].y, s = waves[w0].z, ahead = __float_as_int(waves[w0].w);
#pragma unroll
        for (int w = 1; w < kThreads / 64; ++w) {
            const float4 o = waves[w0 + w];
            if (o.x != -INFINITY) merge(m, l, s, o.x, o.y, o.z);
            ahead += __float_as_int(o.w);
        }
    } else {
        m = -INFINITY, l = s = 0.f, ahead = 0;
    }
    if constexpr (Parts > 1) {  // the lanes' sums as the other launch joins them
        const float M = join_lanes(m, l, s, ahead);
        if (threadIdx.x == 0) finish(a, row, g, xt, M, l, s, ahead);
        return;
    }
    if (a.parts == 1 && !a.k)
        finish(a, row, g, xt, m, l, s, ahead);
    else
        a.part[row * a.parts + blockIdx.x] = make_float4(m, l, s, __int_as_float(ahead));
}

// One workgroup a row: the parts' sums joined, and the k alternatives chosen.
//
// A lower bound of the k-th largest key: the k-th largest of the groups' largest
// (a group has every 256th segment).  Few segments reach it, and only their
// logits are read again: those at or above the bound become candidates.  Where
// they are more than kCap, the bound is raised by bisection (keys are unique, so
// some bound leaves k to kCap of them).  The candidates' places are their ranks
// among each other.
//
// A row of fewer segments than k (16 a part of 8192 logits: up to 8192 logits
// for k over 16, 24576 for k over 48) has no such bound: all its logits are
// candidates, or what a bisection of them leaves, and their ranks cost their
// number squared.  64 rows of 8000 logits take 14.4 us with k = 16 and 78 with 17
// to 64, of 2000 14.4 and 90, of 24000 24.7 with 48 and 86 with 64.
//
// Bound by latency, a chain of loads and barriers: 6.5 us for one row of 248320
// (31 parts) with 20 alternatives, 10 for 512 rows with 8.  1024 threads because
// the reread segments are loads in flight: 10.8 us with 256; 256 groups because
// with 64 and k = 64 the least of the groups' largest is the bound, which
// hundreds of segments reach: the whole call 32 us against 17.
template <typename T>
__global__ __launch_bounds__(kJoin) void logprobs_join_kernel(ScoreArgs a) {
    __shared__ unsigned long long cand[kCap];
    __shared__ int32_t list[kCap];
    __shared__ unsigned long long bound;
    __shared__ float m_all, ln_all;
    __shared__ int n_cand, n_list, ahead_of[kGroups];
    constexpr int VL = Row<T>::VL, kVec = Row<T>::kVec, kPart = Row<T>::kPart;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t row = blockIdx.x;
    const Row<T> x(a, row);
    const int ns = a.parts * kSegs;
    const unsigned long long *seg = a.seg + row * ns;
    // the groups' largest keys: thread t takes segments t, t + kJoin, ..: group t % kGroups
    unsigned long long first = 0;  // the thread's first segment's key
    const int g = a.target ? a.target[row] : -1;
    float4 part = make_float4(-INFINITY, 0.f, 0.f, 0.f);
    if (wave == 1 && lane < a.parts) part = a.part[row * a.parts + lane];
    if (a.k) {
        first = tid < ns ? seg[tid] : 0ull;
        unsigned long long best = first;
        for (int i = tid + kJoin; i < ns; i += kJoin) best = argmax_key_max(best, seg[i]);
        cand[tid] = best;
    }
    const float xt = g >= 0 && g < a.n ? logit(x.x, g) : 0.f;
    if (a.k) __syncthreads();
    if (wave == 1) {
        // the sums, a part a lane
        float m = part.x, l = part.y, s = part.z;
        int ahead = __float_as_int(part.w);
        for (int p = lane + 64; p < a.parts; p += 64) {
            const float4 o = a.part[row * a.parts + p];
            if (o.x != -INFINITY) merge(m, l, s, o.x, o.y, o.z);
            ahead += __float_as_int(o.w);
        }
        const float M = join_lanes(m, l, s, ahead);
        if (lane == 0) {
            finish(a, row, g, xt, M, l, s, ahead);
            m_all = M;
            ln_all = logf(l);
        }
    }
    if (!a.k) return;
    // group g: the keys that threads g, g + kGroups, .. hold
    if (tid < kGroups) {
        unsigned long long best = cand[tid];
#pragma unroll
        for (int i = kGroups; i < kJoin; i += kGroups) best = argmax_key_max(best, cand[tid + i]);
        cand[kJoin + tid] = best;
        ahead_of[tid] = 0;
    }
    if (tid == 0) {
        bound = 1;  // every logit above -inf, where fewer than k groups have one
        n_list = n_cand = 0;
    }
    __syncthreads();
    const unsigned long long *group = cand + kJoin, mine = group[tid % kGroups];
    {
        // its rank among a quarter of the groups
        constexpr int kShare = kGroups * kGroups / kJoin;
        const int from = tid / kGroups * kShare;
        int before = 0;
#pragma unroll 16
        for (int i = 0; i < kShare; ++i) before += group[from + i] > mine;
        atomicAdd(&ahead_of[tid % kGroups], before);
    }
    __syncthreads();
    if (tid < kGroups && mine && ahead_of[tid] == a.k - 1) bound = mine;  // keys are unique
    __syncthreads();
    const unsigned long long least = bound;
    unsigned long long lo = least, hi = ~0ull, cur = least;
    bool by_value = true;  // the first raise goes past the bound's own value
    int c;
    for (;;) {
        // the segments that reach the bound, then their logits that do
        for (int i = tid; i < ns; i += kJoin)
            if ((i == tid ? first : seg[i]) >= cur) {
                const int at = atomicAdd(&n_list, 1);
                if (at < kCap) list[at] = i;
            }
        __syncthreads();
        const int nl = n_list;
        if (nl <= kCap) {
            for (int u = tid; u < nl * 16 * kVec; u += kJoin) {
                const int i = list[u / (16 * kVec)], w = u % (16 * kVec);
                const int q = i / kSegs * kPart + i % kSegs * 16 + (w >> 4) * kThreads + (w & 15);
                if (x.first(q) >= a.n) continue;
                const u32x4_t v = x.load(q);
#pragma unroll
                for (int e = 0; e < VL; ++e) {
                    const float f = Row<T>::at(v, e);
                    if (f == -INFINITY) continue;
                    const unsigned long long key = argmax_key(f, static_cast<unsigned>(x.first(q) + e));
                    if (key >= cur) {
                        const int at = atomicAdd(&n_cand, 1);
                        if (at < kCap) cand[at] = key;
                    }
                }
            }
        }
        __syncthreads();
        c = nl <= kCap ? n_cand : kCap + 1;  // a segment in the list has a candidate at least
        if (c <= kCap && (c >= a.k || cur == least)) break;
        if (c > kCap)
            lo = cur;
        else
            hi = cur;
        if (by_value && c > kCap)
            cur = (lo | 0xffffffffull) + 1;  // above every key of this value
        else
            cur = lo + (hi - lo) / 2;
        by_value = false;
        __syncthreads();
        if (tid == 0) n_list = n_cand = 0;
        __syncthreads();
    }
    const float mm = m_all, ln = ln_all;
    for (int i = c + tid; i < a.k; i += kJoin) {
        a.top_id[row * a.k + i] = -1;
        a.top_logprob[row * a.k + i] = -INFINITY;
    }
    for (int i = tid; i < c; i += kJoin) {
        const unsigned long long mine = cand[i];
        int before = 0;
        for (int j = 0; j < c; ++j) before += cand[j] > mine;
        if (before < a.k) {
            const uint32_t u = static_cast<uint32_t>(mine >> 32);  // the logit, as argmax_key ordered it
            const float f = __uint_as_float(u & 0x80000000u ? u ^ 0x80000000u : ~u);
            a.top_id[row * a.k + before] = argmax_index(mine);
            a.top_logprob[row * a.k + before] = (f == mm ? 0.f : f - mm) - ln;
        }
    }
}

template <typename T>
int launch(const ScoreArgs &a, unsigned rows, hipStream_t s) {
    // Few rows of few parts take one launch, of the same sums in the same order.
    // (32003 bf16 logits: 1 row 5.5 us, 7.9 with two; 256 rows 8.9 and 11.7; 512
    // 15.2 and 16.4; 1009 rows 25.8 and 22.8, the launch then runs in two rounds)
    const bool whole = !a.k && a.parts > 1 && a.parts <= kRowParts && rows <= kFewRows;
    for (unsigned r = 0; r < rows; r += 65535) {  // grid y
        ScoreArgs b = a;
        const unsigned m = rows - r < 65535 ? rows - r : 65535;
        b.x = static_cast<const T *>(a.x) + r * a.stride;
        b.target = a.target ? a.target + r : nullptr;
        auto move = [&](auto *p) { return p ? p + r : p; };
        b.logprob = move(a.logprob), b.rank = move(a.rank), b.entropy = move(a.entropy), b.lse = move(a.lse);
        if (a.k) b.top_id = a.top_id + static_cast<size_t>(r) * a.k, b.top_logprob = a.top_logprob + static_cast<size_t>(r) * a.k;
        if (a.k)
            hipLaunchKernelGGL((logprobs_part_kernel<T, true, 1>), dim3(a.parts, m), dim3(kThreads), 0, s, b);
        else if (whole)
            hipLaunchKernelGGL((logprobs_part_kernel<T, false, kRowParts>), dim3(1, m), dim3(kRowParts * kThreads), 0, s, b);
        else
            hipLaunchKernelGGL((logprobs_part_kernel<T, false, 1>), dim3(a.parts, m), dim3(kThreads), 0, s, b);
        int st = check_launch("logprobs_part_kernel");
        if (st) return st;
        if (a.k || (a.parts > 1 && !whole)) {
            hipLaunchKernelGGL(logprobs_join_kernel<T>, dim3(m), dim3(a.k ? kJoin : 128), 0, s, b);
            if ((st = check_launch("logprobs_join_kernel"))) return st;
        }
    }
    return OURO_OK;
}

// Parts of a row that may start anywhere in a vector, and the workspace of a
// launch of up to 65535 rows.
int parts_of(size_t n, size_t size) {
    const size_t vl = 16 / size, vectors = (n + 2 * (vl - 1)) / vl, part = kPartLogits / vl;
    return static_cast<int>((vectors + part - 1) / part);
}
struct ScoreWs {
    size_t seg, bytes;
};
ScoreWs score_ws(size_t rows, int parts, size_t k) {
    if (rows > 65535) rows = 65535;
    if (!k && parts == 1) return {0, 0};
    ScoreWs w{};
    w.seg = (rows * parts * sizeof(float4) + 255) & ~size_t{255};
    w.bytes = w.seg + (k ? rows * parts * kSegs * sizeof(unsigned long long) : 0);
    return w;
}

}  // namespace
}  // namespace ouro

using namespace ouro;

extern "C" {

size_t ouro_token_logprobs_workspace_bytes(size_t rows, size_t n, size_t k) {
    const int a = parts_of(n, 4), b = parts_of(n, 2);
    return score_ws(rows, a > b ? a : b, k).bytes;
}

int ouro_token_logprobs(const void *logits, int dtype, size_t rows, size_t n, size_t row_stride, const int32_t *targets,
                        size_t k, float *logprob, int32_t *rank, float *entropy, float *lse, int32_t *top_id,
                        float *top_logprob, void *ws, void *stream) {
    OURO_REQUIRE_INIT();
    const char *const me = "ouro_token_logprobs";
    if (!logits) return fail(OURO_ERR_INVALID_ARG, "%s: logits are NULL", me);
    if (dtype != OURO_DT_F32 && dtype != OURO_DT_BF16) return fail(OURO_ERR_INVALID_ARG, "%s: dtype %d", me, dtype);
    if (!n || n >= (1u << 24)) return fail(OURO_ERR_SHAPE, "%s: rows of %zu logits (1 .. 2^24 - 1)", me, n);
    if (rows > 0x7fffffff) return fail(OURO_ERR_SHAPE, "%s: %zu rows", me, rows);
    if (!row_stride) row_stride = n;
    if (row_stride < n) return fail(OURO_ERR_SHAPE, "%s: rows of %zu logits %zu apart", me, n, row_stride);
    if (k > 64) return fail(OURO_ERR_SHAPE, "%s: %zu alternatives (up to 64)", me, k);
    if (k && (!top_id || !top_logprob)) return fail(OURO_ERR_INVALID_ARG, "%s: alternatives without a place", me);
    if ((logprob || rank) && !targets) return fail(OURO_ERR_INVALID_ARG, "%s: logprob and rank need targets", me);
    if (reinterpret_cast<uintptr_t>(logits) % (dtype == OURO_DT_F32 ? 4 : 2))
        return fail(OURO_ERR_ALIGN, "%s: logits off their type's alignment", me);
    if (!rows) return OURO_OK;
    const bool half = dtype == OURO_DT_BF16;
    ScoreArgs a{};
    a.x = logits, a.stride = static_cast<int64_t>(row_stride), a.target = targets;
    a.logprob = logprob, a.entropy = entropy, a.lse = lse, a.top_logprob = top_logprob, a.rank = rank, a.top_id = top_id;
    a.n = static_cast<int32_t>(n), a.k = static_cast<int32_t>(k), a.parts = parts_of(n, half ? 2 : 4);
    const ScoreWs w = score_ws(rows, a.parts, k);
    if (w.bytes) {
        if (!ws && !(ws = workspace(w.bytes, stream))) return OURO_ERR_HIP;
        unsigned char *p = static_cast<unsigned char *>(ws);
        a.part = reinterpret_cast<float4 *>(p);
        if (k) a.seg = reinterpret_cast<unsigned long long *>(p + w.seg);
    }
    return half ? launch<uint16_t>(a, static_cast<unsigned>(rows), as_stream(stream))
                : launch<float>(a, static_cast<unsigned>(rows), as_stream(stream));
}

}  // extern "C"
