// kv_evict.hip - a caller's paged key-value cache cut to a budget by
// accumulated attention weight.
//
// Of a head's n slots, ordered by (position among the newest, weight, lower
// slot), the first `keep` stay.  Attention does not depend on the order of the
// slots, so nothing is shifted: the i-th slot below `keep` that goes is filled
// from the i-th slot at or above `keep` that stays.  Every source is at or
// above `keep` and every destination below it, so the moves have no order
// among them, and there are at most min(keep, n - keep).
#include "kv_cache.hpp"

namespace ouro {
namespace {

struct EvictArgs {
    KvView c;
    const float *weight;
    const int32_t *pos, *lens;
    float *weight_out;
    int32_t *pos_out, *lens_out, *slot_from;  // slot_from [seqs][heads][keep]
    int32_t *hole, *mover;                    // [seqs][heads][keep]: the slots to fill, and those that fill them, in order
    int32_t *moves;                           // [seqs][heads]
    int32_t heads, slots, slots_out, max_len, keep, recent;
};
// passed by value to kernels: the host and device passes must lay it out alike
static_assert(sizeof(EvictArgs) == 176, "EvictArgs: kernel argument layout");

// A weight as an unsigned of the same order: NaN lowest, -0 as +0.
__device__ __forceinline__ uint32_t weight_order(float w) {
    if (w != w) return 0u;
    const uint32_t u = __float_as_uint(w == 0.f ? 0.f : w);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

constexpr int kThreads = 256;

// Sum of v over the workgroup, to every thread.
__device__ __forceinline__ int block_sum(int v, int *tmp) {
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) v += xor_shfl(v, off);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) tmp[threadIdx.x >> 6] = v;
    __syncthreads();
    int s = 0;
    for (int w = 0; w < kThreads / 64; ++w) s += tmp[w];
    return s;
}
// Exclusive prefix of a flag over the workgroup; *total gets the sum.
__device__ __forceinline__ int block_rank(bool f, int *tmp, int *total) {
    const unsigned long long bal = __ballot(f);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    __syncthreads();
    if (lane == 0) tmp[wave] = __popcll(bal);
    __syncthreads();
    int before = __popcll(bal & ((1ull << lane) - 1)), all = 0;
    for (int w = 0; w < kThreads / 64; ++w) {
        if (w < wave) before += tmp[w];
        all += tmp[w];
    }
    *total = all;
    return before;
}

// The choice of one (head, sequence): a workgroup finds the weight of the last
// slot that stays bit by bit, then walks the slots in order.
__global__ __launch_bounds__(kThreads) void kv_choose_kernel(EvictArgs a) {
    __shared__ int tmp[kThreads / 64];
    const int hs = blockIdx.x, t = threadIdx.x;
    const int64_t b = blockIdx.y, row = b * a.heads + hs;
    const int n = max(0, min(a.lens[b], a.max_len));
    const float *w = a.weight + row * a.slots;
    const int32_t *pos = a.pos + row * a.slots;
    int32_t *from = a.slot_from + row * a.keep, *hole = a.hole + row * a.keep, *mover = a.mover + row * a.keep;
    float *w_out = a.weight_out + row * a.slots_out;
    int32_t *pos_out = a.pos_out + row * a.slots_out;
    if (hs == 0 && t == 0) a.lens_out[b] = min(n, a.keep);
    for (int j = t; j < a.keep; j += kThreads) from[j] = j < n ? j : -1;
    if (n <= a.keep) {
        if (t == 0) a.moves[row] = 0;
        if (w_out != w)
            for (int j = t; j < n; j += kThreads) w_out[j] = w[j], pos_out[j] = pos[j];
        return;
    }
    // the newest: positions past max - recent
    int newest = INT32_MIN;
    for (int j = t; j < n; j += kThreads) newest = max(newest, pos[j]);
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) newest = max(newest, xor_shfl(newest, off));
    if ((t & 63) == 0) tmp[t >> 6] = newest;
    __syncthreads();
    for (int i = 0; i < kThreads / 64; ++i) newest = max(newest, tmp[i]);
    const int64_t line = static_cast<int64_t>(newest) - a.recent;
    int mine = 0;
    for (int j = t; j < n; j += kThreads) mine += pos[j] > line;
    const int recents = block_sum(mine, tmp);
    // whichever class is cut: the newest alone where they fill the budget,
    // else the others
    const bool cut = recents >= a.keep;
    const int need = cut ? a.keep : a.keep - recents;
    uint32_t T = 0;
    for (int bit = 31; bit >= 0; --bit) {
        const uint32_t c = T | (1u << bit);
        mine = 0;
        for (int j = t; j < n; j += kThreads) mine += (pos[j] > line) == cut && weight_order(w[j]) >= c;
        if (block_sum(mine, tmp) >= need) T = c;
    }
    mine = 0;
    for (int j = t; j < n; j += kThreads) mine += (pos[j] > line) == cut && weight_order(w[j]) > T;
    const int ties = need - block_sum(mine, tmp);
    int tied = 0, holes = 0, movers = 0;
    for (int j0 = 0; j0 < n; j0 += kThreads) {
        const int j = j0 + t;
        const bool live = j < n;
        const bool is_new = live && pos[j] > line;
        const uint32_t o = live ? weight_order(w[j]) : 0u;
        const bool in_class = live && is_new == cut;
        int all;
        const int r = tied + block_rank(in_class && o == T, tmp, &all);
        tied += all;
        const bool stays = live && ((is_new && !cut) || (in_class && (o > T || (o == T && r < ties))));
        const int i = holes + block_rank(live && !stays && j < a.keep, tmp, &all);
        holes += all;
        if (live && !stays && j < a.keep) hole[i] = j;
        const int k = movers + block_rank(stays && j >= a.keep, tmp, &all);
        movers += all;
        if (stays && j >= a.keep) mover[k] = j;
    }
    __syncthreads();
    for (int i = t; i < movers; i += kThreads) from[hole[i]] = mover[i];
    __syncthreads();
    for (int j = t; j < a.keep; j += kThreads) {
        const int src = from[j];
        w_out[j] = w[src];
        pos_out[j] = pos[src];
    }
    if (t == 0) a.moves[row] = movers;
}

// One workgroup a (kv head, sequence) and share of its moves: whole rows of k and v.
template <typename C>
__global__ __launch_bounds__(kThreads) void kv_move_kernel(EvictArgs a) {
    const int h = blockIdx.y, lane = threadIdx.x & 63;
    const int64_t b = blockIdx.z, row = b * a.heads + (a.heads > 1 ? h : 0);
    const int n = a.moves[row];
    const int32_t *mover = a.mover + row * a.keep, *hole = a.hole + row * a.keep;
    for (int i = blockIdx.x * 4 + (threadIdx.x >> 6); i < n; i += 4 * gridDim.x) {
        const int64_t src = kv_slot(a.c, b, mover[i]), dst = kv_slot(a.c, b, hole[i]);
        if (src < 0 || dst < 0) continue;
        const int64_t o = h * a.c.head_stride;
        for (int e = lane; e < a.c.d; e += 64) {
            static_cast<C *>(a.c.k)[dst + o + e] = static_cast<const C *>(a.c.k)[src + o + e];
            static_cast<C *>(a.c.v)[dst + o + e] = static_cast<const C *>(a.c.v)[src + o + e];
        }
    }
}

size_t evict_ws_bytes(size_t seqs, size_t heads, size_t keep) {
    return (seqs * heads * (3 * keep + 1) * sizeof(int32_t) + 255) & ~size_t{255};
}

}  // namespace
}  // namespace ouro

using namespace ouro;

extern "C" {

size_t ouro_kv_evict_workspace_bytes(size_t seqs, size_t heads, size_t max_len, size_t keep) {
    (void)max_len;
    return evict_ws_bytes(seqs, heads, keep);
}

int ouro_kv_evict(const ouro_kv_cache *cache, const ouro_kv_history *history, const int32_t *lens, size_t seqs,
                  size_t max_len, size_t keep, size_t recent, const ouro_kv_history *left, int32_t *lens_out,
                  int32_t *slot_from, void *ws, void *stream) {
    OURO_REQUIRE_INIT();
    const char *const me = "ouro_kv_evict";
    EvictArgs a{};
    int st = kv_view(cache, me, &a.c);
    if (st) return st;
    if (!history || !lens || !lens_out) return fail(OURO_ERR_INVALID_ARG, "%s: NULL argument", me);
    if (lens_out == lens) return fail(OURO_ERR_INVALID_ARG, "%s: lens_out is lens (heads read it while it would be written)", me);
    if (!left) left = history;
    if (seqs > 65535) return fail(OURO_ERR_SHAPE, "%s: %zu sequences (up to 65535)", me, seqs);
    if (max_len > static_cast<size_t>(cache->max_pages) * cache->page_tokens || max_len > (1u << 30))
        return fail(OURO_ERR_SHAPE, "%s: %zu slots of %d pages of %d tokens", me, max_len, cache->max_pages, cache->page_tokens);
    if (keep < 1 || keep > (1u << 30) || recent > (1u << 30)) return fail(OURO_ERR_SHAPE, "%s: keep %zu, recent %zu", me, keep, recent);
    if ((st = kv_check_history(history, cache->n_head_kv, max_len, me))) return st;
    if ((st = kv_check_history(left, cache->n_head_kv, keep < max_len ? keep : max_len, me))) return st;
    if (left->heads != history->heads) return fail(OURO_ERR_SHAPE, "%s: histories of %d and %d heads", me, history->heads, left->heads);
    if ((left->weight == history->weight) != (left->pos == history->pos) ||
        (left->weight == history->weight && left->slots != history->slots))
        return fail(OURO_ERR_INVALID_ARG, "%s: the history left is neither the history nor apart from it", me);
    if (!seqs) return OURO_OK;
    const size_t heads = history->heads, need = evict_ws_bytes(seqs, heads, keep);
    if (!ws && !(ws = workspace(need, stream))) return OURO_ERR_HIP;
    int32_t *w = static_cast<int32_t *>(ws);
    a.weight = history->weight, a.pos = history->pos, a.lens = lens;
    a.weight_out = left->weight, a.pos_out = left->pos, a.lens_out = lens_out;
    a.moves = w;
    a.hole = w + seqs * heads;
    a.mover = a.hole + seqs * heads * keep;
    a.slot_from = slot_from ? slot_from : a.mover + seqs * heads * keep;
    a.heads = static_cast<int>(heads), a.slots = history->slots, a.slots_out = left->slots;
    a.max_len = static_cast<int>(max_len), a.keep = static_cast<int>(keep), a.recent = static_cast<int>(recent);
    hipStream_t s = as_stream(stream);
    hipLaunchKernelGGL(kv_choose_kernel, dim3(a.heads, static_cast<unsigned>(seqs)), dim3(kThreads), 0, s, a);
    if ((st = check_launch("kv_choose_kernel"))) return st;
    if (keep >= max_len) return OURO_OK;  // nothing to move
    const size_t most = keep < max_len - keep ? keep : max_len - keep;
    const dim3 grid(static_cast<unsigned>((most + 15) / 16), a.c.n_head_kv, static_cast<unsigned>(seqs));
    if (cache->dtype == OURO_DT_BF16)
        hipLaunchKernelGGL(kv_move_kernel<uint16_t>, grid, dim3(kThreads), 0, s, a);
    else
        hipLaunchKernelGGL(kv_move_kernel<float>, grid, dim3(kThreads), 0, s, a);
    return check_launch("kv_move_kernel");
}

}  // extern "C"
