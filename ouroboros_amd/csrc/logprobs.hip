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
constexpr int kVec = 8;                     // 16-byte vectors of a thread
constexpr int kPart = kThreads * kVec;      // vectors of a workgroup: 32 KiB of logits
constexpr int kSegs = kThreads / 16;        // segments of a part: 16 lanes each
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
    // Element e of a vector, NaN as -inf.
    static __device__ __forceinline__ float at(const u32x4_t &v, int e) {
        float f;
        if constexpr (sizeof(T) == 4)
            f = __uint_as_float(v[e]);
        else
            f = __uint_as_float(e & 1 ? v[e >> 1] & 0xffff0000u : v[e >> 1] << 16);
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

// What a row's sums say, written by one thread.
template <typename T>
__device__ __forceinline__ void finish(const ScoreArgs &a, int64_t row, float m, float l, float s, int ahead) {
    const float ln = logf(l);
    const bool empty = m == -INFINITY;
    const int g = a.target ? a.target[row] : -1;
    const bool given = g >= 0 && g < a.n;
    if (a.lse) a.lse[row] = empty ? -INFINITY : m + ln;
    if (a.entropy) a.entropy[row] = empty ? 0.f : ln - s / l;
    if (a.logprob) {
        const float xt = given ? logit(static_cast<const T *>(a.x) + row * a.stride, g) : 0.f;
        a.logprob[row] = !given ? 0.f : empty ? -INFINITY : (xt == m ? 0.f : xt - m) - ln;
    }
    if (a.rank) a.rank[row] = given ? ahead : -1;
}

// One workgroup a part of a row, its logits in registers: the wavefront's
// maximum, then the sums against it, then the tokens ahead of the given one
// and (Top) the largest key of each segment, that is of the vectors of 16
// lanes.  A row of one part is finished here.
template <typename T, bool Top>
__global__ __launch_bounds__(kThreads) void logprobs_part_kernel(ScoreArgs a) {
    constexpr int VL = Row<T>::VL;
    __shared__ float4 waves[kThreads / 64];
    const int tid = threadIdx.x;
    const int64_t row = blockIdx.y;
    const Row<T> x(a, row);
    const int q0 = static_cast<int>(blockIdx.x) * kPart;
    u32x4_t v[kVec];
#pragma unroll
    for (int j = 0; j < kVec; ++j) {
        const int q = q0 + kThreads * j + tid;
        v[j] = u32x4_t{0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u};
        if constexpr (sizeof(T) == 2) v[j] = u32x4_t{0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u};
        if (x.first(q) < a.n) v[j] = x.load(q);
    }
    const int g = a.target ? a.target[row] : -1;
    const bool given = a.rank && g >= 0 && g < a.n;
    const float xt = given ? logit(x.x, g) : 0.f;
    float mt = -INFINITY;
#pragma unroll
    for (int j = 0; j < kVec; ++j)
#pragma unroll
        for (int e = 0; e < VL; ++e) mt = fmaxf(mt, Row<T>::at(v[j], e));
    const float ms = row16_max(mt);
    float m = fmaxf(ms, xor_shfl(ms, 16));
    m = fmaxf(m, xor_shfl(m, 32));
    float l = 0.f, s = 0.f;
    if (m == INFINITY) {
#pragma unroll
        for (int j = 0; j < kVec; ++j)
#pragma unroll
            for (int e = 0; e < VL; ++e) l += Row<T>::at(v[j], e) == INFINITY ? 1.f : 0.f;
    } else if (m != -INFINITY) {
#pragma unroll
        for (int j = 0; j < kVec; ++j) {
            float lj = 0.f, sj = 0.f;  // short chains
#pragma unroll
            for (int e = 0; e < VL; ++e) {
                const float d = fmaxf(Row<T>::at(v[j], e) - m, -3e38f);  // e^d (-inf) would be 0 (-inf)
                const float p = __builtin_amdgcn_exp2f(d * 1.4426950408889634f);
                lj += p;
                sj += p * d;
            }
            l += lj;
            s += sj;
        }
    }
    int ahead = 0;
    if (given) {
        const int lo = x.first(q0), hi = x.first(q0 + kPart);  // the part's elements, shift aside
        if (hi <= g) {
#pragma unroll
            for (int j = 0; j < kVec; ++j)
#pragma unroll
                for (int e = 0; e < VL; ++e) ahead += Row<T>::at(v[j], e) >= xt;
            if (xt == -INFINITY) {  // the places of no element are -inf too
                ahead = 0;
                for (int j = 0; j < kVec; ++j)
                    for (int e = 0; e < VL; ++e) ahead += x.first(q0 + kThreads * j + tid) + e >= 0;
            }
        } else if (lo > g) {
#pragma unroll
            for (int j = 0; j < kVec; ++j)
#pragma unroll
                for (int e = 0; e < VL; ++e) ahead += Row<T>::at(v[j], e) > xt;
        } else {
#pragma unroll
            for (int j = 0; j < kVec; ++j)
#pragma unroll
                for (int e = 0; e < VL; ++e) {
                    const int i = x.first(q0 + kThreads * j + tid) + e;
                    const float f = Row<T>::at(v[j], e);
                    ahead += f > xt || (f == xt && i >= 0 && i < g);
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
        ahead += xor_shfl(ahead, off);
    }
    if ((tid & 63) == 0) waves[tid >> 6] = make_float4(m, l, s, __int_as_float(ahead));
    __syncthreads();
    if (tid) return;
#pragma unroll
    for (int w = 1; w < kThreads / 64; ++w) {
        const float4 o = waves[w];
        if (o.x != -INFINITY) merge(m, l, s, o.x, o.y, o.z);
        ahead += __float_as_int(o.w);
    }
    if (a.parts == 1 && !a.k)
        finish<T>(a, row, m, l, s, ahead);
    else
        a.part[row * a.parts + blockIdx.x] = make_float4(m, l, s, __int_as_float(ahead));
}

// One workgroup a row: the parts' sums joined, and the k alternatives chosen.
//
// A lower bound of the k-th largest key: the k-th largest of 64 groups' largest
// (a group has every 64th segment).  Few segments reach it, and only their
// logits are read again: those at or above the bound become candidates.  Where
// ties or a skewed row make them more than kCap, the bound is raised by
// bisection (keys are unique, so some bound leaves k to kCap of them).  The
// candidates' places are their ranks among each other.
template <typename T>
__global__ __launch_bounds__(kThreads) void logprobs_join_kernel(ScoreArgs a) {
    __shared__ unsigned long long cand[kCap];
    __shared__ unsigned long long group[64];
    __shared__ unsigned long long bound;
    __shared__ float m_all, ln_all;
    __shared__ float4 sums[kThreads / 64];
    __shared__ int count;
    constexpr int VL = Row<T>::VL;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t row = blockIdx.x;
    const Row<T> x(a, row);
    const int ns = a.parts * kSegs;
    const unsigned long long *seg = a.seg + row * ns;
    // the groups' largest keys: thread t takes segments t, t + 256, ..: group t % 64
    if (a.k) {
        unsigned long long best = 0;
        for (int i = tid; i < ns; i += kThreads) best = argmax_key_max(best, seg[i]);
        cand[tid] = best;
    }
    // the sums, a part a thread
    float m = -INFINITY, l = 0.f, s = 0.f;
    int ahead = 0;
    for (int p = tid; p < a.parts; p += kThreads) {
        const float4 o = a.part[row * a.parts + p];
        if (o.x != -INFINITY) merge(m, l, s, o.x, o.y, o.z);
        ahead += __float_as_int(o.w);
    }
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) {
        const float m2 = xor_shfl(m, off), l2 = xor_shfl(l, off), s2 = xor_shfl(s, off);
        if (m2 != -INFINITY || m != -INFINITY) {
            // the same order of the two on both lanes, so that they agree
            float ma = lane & off ? m2 : m, la = lane & off ? l2 : l, sa = lane & off ? s2 : s;
            merge(ma, la, sa, lane & off ? m : m2, lane & off ? l : l2, lane & off ? s : s2);
            m = ma, l = la, s = sa;
        }
        ahead += xor_shfl(ahead, off);
    }
    if (lane == 0) sums[wave] = make_float4(m, l, s, __int_as_float(ahead));
    __syncthreads();
    if (tid == 0) {
        for (int w = 1; w < kThreads / 64; ++w) {
            const float4 o = sums[w];
            if (o.x != -INFINITY) merge(m, l, s, o.x, o.y, o.z);
            ahead += __float_as_int(o.w);
        }
        finish<T>(a, row, m, l, s, ahead);
        m_all = m;
        ln_all = logf(l);
    }
    if (!a.k) return;
    if (tid < 64) group[tid] = argmax_key_max(argmax_key_max(cand[tid], cand[tid + 64]), argmax_key_max(cand[tid + 128], cand[tid + 192]));
    if (tid == 0) bound = 1;  // every logit above -inf, where fewer than k groups have one
    __syncthreads();
    if (tid < 64) {
        const unsigned long long mine = group[tid];
        int before = 0;
        for (int i = 0; i < 64; ++i) before += group[i] > mine;
        if (mine && before == a.k - 1) bound = mine;  // keys are unique
    }
    __syncthreads();
    const unsigned long long least = bound;
    unsigned long long lo = least, hi = ~0ull, cur = least;
    bool by_value = true;  // the first raise goes past the bound's own value
    int c;
    for (;;) {
        __syncthreads();
        if (tid == 0) count = 0;
        __syncthreads();
        // wavefront w looks at segments 64 w .. , and reads each that reaches the bound
        for (int i0 = 64 * wave; i0 < ns; i0 += kThreads) {
            const bool in = i0 + lane < ns && seg[i0 + lane] >= cur;
            unsigned long long set = __ballot(in);
            while (set) {
                const int i = i0 + __ffsll(set) - 1;
                set &= set - 1;
                const int base = i / kSegs * kPart + i % kSegs * 16;
                for (int u = lane; u < 16 * kVec; u += 64) {
                    const int q = base + (u >> 4) * kThreads + (u & 15);
                    if (x.first(q) >= a.n) continue;
                    const u32x4_t v = x.load(q);
#pragma unroll
                    for (int e = 0; e < VL; ++e) {
                        const float f = Row<T>::at(v, e);
                        if (f == -INFINITY) continue;
                        const unsigned long long key = argmax_key(f, static_cast<unsigned>(x.first(q) + e));
                        if (key >= cur) {
                            const int at = atomicAdd(&count, 1);
                            if (at < kCap) cand[at] = key;
                        }
                    }
                }
            }
        }
        __syncthreads();
        c = count;
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
    }
    const float mm = m_all, ln = ln_all;
    for (int i = tid; i < a.k; i += kThreads)
        if (i >= c) {
            a.top_id[row * a.k + i] = -1;
            a.top_logprob[row * a.k + i] = -INFINITY;
        }
    for (int i = tid; i < c; i += kThreads) {
        const unsigned long long mine = cand[i];
        int before = 0;
        for (int j = 0; j < c; ++j) before += cand[j] > mine;
        if (before < a.k) {
            const int id = argmax_index(mine);
            const float f = logit(x.x, id);
            a.top_id[row * a.k + before] = id;
            a.top_logprob[row * a.k + before] = (f == mm ? 0.f : f - mm) - ln;
        }
    }
}

template <typename T>
int launch(const ScoreArgs &a, unsigned rows, hipStream_t s) {
    for (unsigned r = 0; r < rows; r += 65535) {  // grid y
        ScoreArgs b = a;
        const unsigned m = rows - r < 65535 ? rows - r : 65535;
        b.x = static_cast<const T *>(a.x) + r * a.stride;
        b.target = a.target ? a.target + r : nullptr;
        auto move = [&](auto *p) { return p ? p + r : p; };
        b.logprob = move(a.logprob), b.rank = move(a.rank), b.entropy = move(a.entropy), b.lse = move(a.lse);
        if (a.k) b.top_id = a.top_id + static_cast<size_t>(r) * a.k, b.top_logprob = a.top_logprob + static_cast<size_t>(r) * a.k;
        if (a.k)
            hipLaunchKernelGGL((logprobs_part_kernel<T, true>), dim3(a.parts, m), dim3(kThreads), 0, s, b);
        else
            hipLaunchKernelGGL((logprobs_part_kernel<T, false>), dim3(a.parts, m), dim3(kThreads), 0, s, b);
        int st = check_launch("logprobs_part_kernel");
        if (st) return st;
        if (a.k || a.parts > 1) {
            hipLaunchKernelGGL(logprobs_join_kernel<T>, dim3(m), dim3(kThreads), 0, s, b);
            if ((st = check_launch("logprobs_join_kernel"))) return st;
        }
    }
    return OURO_OK;
}

// Parts of a row that may start anywhere in a vector, and the workspace of a
// launch of up to 65535 rows.
int parts_of(size_t n, size_t size) {
    const size_t vl = 16 / size, vectors = (n + 2 * (vl - 1)) / vl;
    return static_cast<int>((vectors + kPart - 1) / kPart);
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
    return score_ws(rows, parts_of(n, 4), k).bytes;  // fp32 rows have the most parts
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
