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

struct ScoreArgs {
    const void *x;
    int64_t stride;
    const int32_t *target;
    float *logprob, *entropy, *lse, *top_logprob;
    int32_t *rank, *top_id;
    int32_t n, k;
};
// passed by value to kernels: the host and device passes must lay it out alike
static_assert(sizeof(ScoreArgs) == 80, "ScoreArgs: kernel argument layout");

template <typename T>
__device__ __forceinline__ float logit(const T *x, int64_t i) {
    float v;
    if constexpr (sizeof(T) == 4)
        v = x[i];
    else
        v = bf16_bits_to_f32(x[i]);
    return v != v ? -INFINITY : v;
}

__device__ __forceinline__ float block_max(float v, float *tmp) {
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) v = fmaxf(v, xor_shfl(v, off));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) tmp[threadIdx.x >> 6] = v;
    __syncthreads();
    for (int w = 0; w < kThreads / 64; ++w) v = fmaxf(v, tmp[w]);
    return v;
}
__device__ __forceinline__ float block_sum(float v, float *tmp) {
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) v += xor_shfl(v, off);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) tmp[threadIdx.x >> 6] = v;
    __syncthreads();
    float s = 0.f;
    for (int w = 0; w < kThreads / 64; ++w) s += tmp[w];
    return s;
}

// One workgroup a row: the maximum, the sums, then the alternatives one after
// another, each the largest key below the one before.
template <typename T>
__global__ __launch_bounds__(kThreads) void logprobs_kernel(ScoreArgs a) {
    __shared__ float tmp[kThreads / 64];
    __shared__ unsigned long long last;
    const int t = threadIdx.x;
    const int64_t row = blockIdx.x;
    const T *x = static_cast<const T *>(a.x) + row * a.stride;
    float m = -INFINITY;
    for (int i = t; i < a.n; i += kThreads) m = fmaxf(m, logit(x, i));
    m = block_max(m, tmp);
    const int g = a.target ? a.target[row] : -1;
    const bool given = g >= 0 && g < a.n;
    const float xt = given ? logit(x, g) : 0.f;
    float l = 0.f, s = 0.f;
    int ahead = 0;
    for (int i = t; i < a.n; i += kThreads) {
        const float v = logit(x, i), dv = v == m ? 0.f : v - m, e = expf(dv);
        l += e;
        if (e > 0.f) s += e * dv;
        ahead += v > xt || (v == xt && i < g);
    }
    l = block_sum(l, tmp);
    s = block_sum(s, tmp);
    const float ahead_all = block_sum(static_cast<float>(ahead), tmp);  // n < 2^24: exact
    const float ln = logf(l);
    const bool empty = m == -INFINITY;
    if (t == 0) {
        if (a.lse) a.lse[row] = m + ln;
        if (a.entropy) a.entropy[row] = empty ? 0.f : ln - s / l;
        if (a.logprob) a.logprob[row] = !given ? 0.f : empty ? -INFINITY : (xt == m ? 0.f : xt - m) - ln;
        if (a.rank) a.rank[row] = given ? static_cast<int32_t>(ahead_all) : -1;
    }
    unsigned long long before = ~0ull;
    for (int k = 0; k < a.k; ++k) {
        unsigned long long best = 0;
        for (int i = t; i < a.n; i += kThreads) {
            const float v = logit(x, i);
            const unsigned long long key = argmax_key(v, static_cast<unsigned>(i));
            if (v != -INFINITY && key < before) best = argmax_key_max(best, key);
        }
        best = argmax_block_key(best);
        if (t == 0) last = best;
        __syncthreads();
        before = last;
        if (t == 0) {
            const int id = before ? argmax_index(before) : -1;
            const float v = id >= 0 ? logit(x, id) : -INFINITY;
            a.top_id[row * a.k + k] = id;
            a.top_logprob[row * a.k + k] = id < 0 ? -INFINITY : (v == m ? 0.f : v - m) - ln;
        }
        __syncthreads();
    }
}

}  // namespace
}  // namespace ouro

using namespace ouro;

extern "C" {

size_t ouro_token_logprobs_workspace_bytes(size_t rows, size_t n, size_t k) {
    (void)rows;
    (void)n;
    (void)k;
    return 0;
}

int ouro_token_logprobs(const void *logits, int dtype, size_t rows, size_t n, size_t row_stride, const int32_t *targets,
                        size_t k, float *logprob, int32_t *rank, float *entropy, float *lse, int32_t *top_id,
                        float *top_logprob, void *ws, void *stream) {
    OURO_REQUIRE_INIT();
    (void)ws;
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
    ScoreArgs a{logits, static_cast<int64_t>(row_stride), targets, logprob, entropy, lse, top_logprob, rank, top_id,
                static_cast<int32_t>(n), static_cast<int32_t>(k)};
    const dim3 grid(static_cast<unsigned>(rows));
    if (dtype == OURO_DT_F32)
        hipLaunchKernelGGL(logprobs_kernel<float>, grid, dim3(kThreads), 0, as_stream(stream), a);
    else
        hipLaunchKernelGGL(logprobs_kernel<uint16_t>, grid, dim3(kThreads), 0, as_stream(stream), a);
    return check_launch("logprobs_kernel");
}

}  // extern "C"
