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
    int2 *move;                               // [seqs][heads][most]: a slot to fill, and the slot that fills it
    int32_t *moves;                           // [seqs][heads]
    int32_t heads, slots, slots_out, max_len, keep, recent, most, vecs;  // vecs: 16-byte vectors of a row
};
// passed by value to kernels: the host and device passes must lay it out alike
static_assert(sizeof(EvictArgs) == 176, "EvictArgs: kernel argument layout");

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));

// Orders of slots in one unsigned: 0 of what goes whatever its weight,
// 0xffffffff of what stays whatever its weight, between them a weight's (NaN
// lowest, -0 as +0).
constexpr uint32_t kGoes = 0u, kStays = 0xffffffffu, kLeast = 1u, kMost = 0xff800000u;
__device__ __forceinline__ uint32_t weight_order(float w) {
    if (w != w) return kLeast;
    const uint32_t u = __float_as_uint(w == 0.f ? 0.f : w);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// Over lanes 0 .. W - 1 of each 16 (W 4 or 16), to each of them.
template <int W, typename F>
__device__ __forceinline__ int row_join(int v, F f) {
    if constexpr (W == 16) {
        v = f(v, __builtin_amdgcn_update_dpp(0, v, 0x128, 0xf, 0xf, false));
        v = f(v, __builtin_amdgcn_update_dpp(0, v, 0x141, 0xf, 0xf, false));
    }
    v = f(v, __builtin_amdgcn_update_dpp(0, v, 0x4E, 0xf, 0xf, false));
    return f(v, __builtin_amdgcn_update_dpp(0, v, 0xB1, 0xf, 0xf, false));
}

// Copies rows of k and v of one (kv head, sequence): `lanes` lanes a row, from
// the pair `first` on in steps of `step`.
__device__ __forceinline__ void move_rows(const EvictArgs &a, int64_t b, int h, const int2 *move, int n, int first, int step, int lane) {
    for (int i = first; i < n; i += step) {
        const int2 m = move[i];
        const int64_t dst = kv_slot(a.c, b, m.x), src = kv_slot(a.c, b, m.y);
        if (src < 0 || dst < 0 || lane >= a.vecs) continue;
        const int64_t size = a.c.elem;
        const char *k = static_cast<const char *>(a.c.k), *v = static_cast<const char *>(a.c.v);
        const int64_t from = (src + h * a.c.head_stride) * size + lane * 16, to = (dst + h * a.c.head_stride) * size + lane * 16;
        const u32x4_t x = *reinterpret_cast<const u32x4_t *>(k + from), y = *reinterpret_cast<const u32x4_t *>(v + from);
        *reinterpret_cast<u32x4_t *>(static_cast<char *>(a.c.k) + to) = x;
        *reinterpret_cast<u32x4_t *>(static_cast<char *>(a.c.v) + to) = y;
    }
}

// The choice of one (head, sequence) by one workgroup of W wavefronts, each
// with a run of slots in order, 64 R of them in registers (longer runs are read
// again at each pass).  The order of the last slot that stays is searched for
// with three counts a round; counts are of ballots, and a round's are joined
// through LDS with one barrier.  Moves: the workgroup copies the rows too.
template <int W, int R, bool Moves>
__global__ __launch_bounds__(W * 64) void kv_choose_kernel(EvictArgs a) {
    constexpr int kThreads = W * 64;
    __shared__ int4 tmp[2][W];
    const int hs = blockIdx.x, t = threadIdx.x, lane = t & 63;
    const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int64_t b = blockIdx.y, row = b * a.heads + hs;
    const int n = max(0, min(a.lens[b], a.max_len)), keep = a.keep;
    const float *weight = a.weight + row * a.slots;
    const int32_t *pos = a.pos + row * a.slots;
    int32_t *from = a.slot_from + row * keep;
    float *w_out = a.weight_out + row * a.slots_out;
    int32_t *pos_out = a.pos_out + row * a.slots_out;
    const bool apart = w_out != weight;
    if (hs == 0 && t == 0) a.lens_out[b] = min(n, keep);
    if (n <= keep) {
        for (int j = t; j < keep; j += kThreads) from[j] = j < n ? j : -1;
        if (!Moves && t == 0) a.moves[row] = 0;
        if (apart)
            for (int j = t; j < n; j += kThreads) w_out[j] = weight[j], pos_out[j] = pos[j];
        return;
    }
    int round = 0;
    // A wavefront's counts joined: the sums over all wavefronts, and those over
    // the ones before it.
    int4 all, before;
    auto join = [&](int x, int y, int z) {
        int4 *buf = tmp[round++ & 1];  // a wavefront is at most one round ahead
        if (lane == 0) buf[wave] = make_int4(x, y, z, 0);
        __syncthreads();
        const int4 o = buf[lane % W];
        auto add = [](int p, int q) { return p + q; };
        const bool is = lane % W < wave;
        all = make_int4(row_join<W>(o.x, add), row_join<W>(o.y, add), row_join<W>(o.z, add), 0);
        before = make_int4(row_join<W>(is ? o.x : 0, add), row_join<W>(is ? o.y : 0, add), row_join<W>(is ? o.z : 0, add), 0);
    };
    const int run = ((n + kThreads - 1) / kThreads) * 64;  // slots of a wavefront
    const int j0 = wave * run, end = min(n, j0 + run);
    float w[R];
    int32_t p[R];
    uint32_t o[R];
    auto load = [&](int c) {
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const int j = j0 + c + i * 64 + lane;
            w[i] = 0.f, p[i] = INT32_MIN;
            if (c + i * 64 < run && j < end) w[i] = weight[j], p[i] = pos[j];
        }
    };
    const bool once = run <= 64 * R;
    // the newest: positions past max - recent
    load(0);
    int newest = INT32_MIN;
    for (int c = 0; c < run; c += 64 * R) {
        if (c) load(c);
#pragma unroll
        for (int i = 0; i < R; ++i) newest = max(newest, p[i]);
    }
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) newest = max(newest, xor_shfl(newest, off));
    {
        int4 *buf = tmp[round++ & 1];
        if (lane == 0) buf[wave].x = newest;
        __syncthreads();
        newest = row_join<W>(buf[lane % W].x, [](int x, int y) { return x > y ? x : y; });
    }
    const int64_t line = static_cast<int64_t>(newest) - a.recent;
    int news = 0;
    for (int c = 0; c < run; c += 64 * R) {
        if (!once) load(c);
#pragma unroll
        for (int i = 0; i < R; ++i) {
            if (c + i * 64 >= run) break;
            news += __popcll(__ballot(j0 + c + i * 64 + lane < end && p[i] > line));
        }
    }
    join(news, 0, 0);
    // whichever class is cut: the newest alone where they fill the budget, else the others
    const bool cut = all.x >= keep;
    auto orders = [&](int c) {
        if (!once) load(c);
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const bool is_new = p[i] > line;
            o[i] = is_new == cut ? weight_order(w[i]) : is_new ? kStays : kGoes;
            if (j0 + c + i * 64 + lane >= end) o[i] = kGoes;
        }
    };
    if (once) orders(0);
    // the largest order that `keep` slots reach: in lo .. hi
    uint32_t lo = kLeast, hi = kMost;
    int ties = 0;      // how many at the order itself stay
    bool exact = false;
    while (lo < hi) {
        const uint32_t q = max(1u, (hi - lo) >> 2), c1 = lo + q, c2 = c1 + q, c3 = c2 + q;
        int n1 = 0, n2 = 0, n3 = 0;
        for (int c = 0; c < run; c += 64 * R) {
            if (!once) orders(c);
#pragma unroll
            for (int i = 0; i < R; ++i) {
                if (c + i * 64 >= run) break;
                n1 += __popcll(__ballot(o[i] >= c1));
                n2 += __popcll(__ballot(o[i] >= c2));
                n3 += __popcll(__ballot(o[i] >= c3));
            }
        }
        join(n1, n2, n3);
        const int m1 = __builtin_amdgcn_readfirstlane(all.x), m2 = __builtin_amdgcn_readfirstlane(all.y), m3 = __builtin_amdgcn_readfirstlane(all.z);
        if (m1 == keep || m2 == keep || m3 == keep) {  // exactly those above lo stay
            lo = (m1 == keep ? c1 : m2 == keep ? c2 : c3) - 1;
            exact = true;
            break;
        }
        if (m3 >= keep)
            lo = c3;
        else if (m2 >= keep)
            lo = c2, hi = c3 - 1;
        else if (m1 >= keep)
            lo = c1, hi = c2 - 1;
        else
            hi = c1 - 1;
    }
    int tied = 0;  // those at lo in the wavefronts before
    if (!exact) {
        int above = 0, at = 0;
        for (int c = 0; c < run; c += 64 * R) {
            if (!once) orders(c);
#pragma unroll
            for (int i = 0; i < R; ++i) {
                if (c + i * 64 >= run) break;
                above += __popcll(__ballot(o[i] > lo));
                at += __popcll(__ballot(o[i] == lo));
            }
        }
        join(above, at, 0);
        ties = keep - all.x;
        tied = before.y;
    }
    // those that go below `keep`, those that stay from it on
    const unsigned long long below = (1ull << lane) - 1;
    auto stays = [&](int i, int &seen) {
        const bool is = !exact && o[i] == lo;
        const unsigned long long bal = __ballot(is);
        const int r = seen + __popcll(bal & below);
        seen += __popcll(bal);
        return o[i] > lo || (is && r < ties);
    };
    int holes = 0, movers = 0, seen = tied;
    for (int c = 0; c < run; c += 64 * R) {
        if (!once) orders(c);
#pragma unroll
        for (int i = 0; i < R; ++i) {
            if (c + i * 64 >= run) break;
            const int j = j0 + c + i * 64 + lane;
            const bool s = stays(i, seen);
            holes += __popcll(__ballot(!s && j < end && j < keep));
            movers += __popcll(__ballot(s && j >= keep));
        }
    }
    join(holes, movers, 0);
    const int moves = all.y;
    holes = before.x, movers = before.y, seen = tied;
    int2 *move = a.move + row * a.most;
    for (int c = 0; c < run; c += 64 * R) {
        if (!once) orders(c);
#pragma unroll
        for (int i = 0; i < R; ++i) {
            if (c + i * 64 >= run) break;
            const int j = j0 + c + i * 64 + lane;
            const bool s = stays(i, seen);
            const bool hole = !s && j < end && j < keep, mover = s && j >= keep;
            const unsigned long long hb = __ballot(hole), mb = __ballot(mover);
            if (hole) move[holes + __popcll(hb & below)].x = j;
            if (mover) move[movers + __popcll(mb & below)].y = j;
            holes += __popcll(hb);
            movers += __popcll(mb);
            if (s && j < keep) {
                from[j] = j;
                if (apart) w_out[j] = w[i], pos_out[j] = p[i];
            }
        }
    }
    __syncthreads();
    for (int i = t; i < moves; i += kThreads) {
        const int2 m = move[i];
        from[m.x] = m.y;
        w_out[m.x] = weight[m.y];
        pos_out[m.x] = pos[m.y];
    }
    if constexpr (Moves) {
        const int lanes = a.vecs <= 16 ? 16 : a.vecs <= 32 ? 32 : 64;
        const int h0 = a.heads > 1 ? hs : 0, h1 = a.heads > 1 ? hs + 1 : a.c.n_head_kv;
        for (int h = h0; h < h1; ++h) move_rows(a, b, h, move, moves, t / lanes, kThreads / lanes, t % lanes);
    } else if (t == 0) {
        a.moves[row] = moves;
    }
}

constexpr int kMoveThreads = 256;

// One workgroup a (kv head, sequence) and share of its moves.
__global__ __launch_bounds__(kMoveThreads) void kv_move_kernel(EvictArgs a) {
    const int lanes = a.vecs <= 16 ? 16 : a.vecs <= 32 ? 32 : 64;
    const int h = blockIdx.y, t = threadIdx.x;
    const int64_t b = blockIdx.z, row = b * a.heads + (a.heads > 1 ? h : 0);
    const int groups = kMoveThreads / lanes;
    move_rows(a, b, h, a.move + row * a.most, a.moves[row], blockIdx.x * groups + t / lanes, gridDim.x * groups, t % lanes);
}

constexpr size_t kFew = 64;  // moves a sequence and head up to which the choosing workgroup makes them

// Moves of a (sequence, head) at the most.
size_t most_moves(size_t max_len, size_t keep) {
    const size_t gone = max_len > keep ? max_len - keep : 0;
    return keep < gone ? keep : gone;
}
size_t evict_ws_bytes(size_t seqs, size_t heads, size_t max_len, size_t keep) {
    return (seqs * heads * (most_moves(max_len, keep) * sizeof(int2) + (keep + 1) * sizeof(int32_t)) + 255) & ~size_t{255};
}

template <bool Moves>
void choose(const EvictArgs &a, unsigned seqs, hipStream_t s) {
    const dim3 grid(a.heads, seqs);
    if (a.max_len <= 2048)
        hipLaunchKernelGGL((kv_choose_kernel<4, 8, Moves>), grid, dim3(256), 0, s, a);
    else
        hipLaunchKernelGGL((kv_choose_kernel<16, 16, Moves>), grid, dim3(1024), 0, s, a);
}

}  // namespace
}  // namespace ouro

using namespace ouro;

extern "C" {

size_t ouro_kv_evict_workspace_bytes(size_t seqs, size_t heads, size_t max_len, size_t keep) {
    return evict_ws_bytes(seqs, heads, max_len, keep);
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
    const size_t heads = history->heads, most = most_moves(max_len, keep), need = evict_ws_bytes(seqs, heads, max_len, keep);
    if (!ws && !(ws = workspace(need, stream))) return OURO_ERR_HIP;
    a.weight = history->weight, a.pos = history->pos, a.lens = lens;
    a.weight_out = left->weight, a.pos_out = left->pos, a.lens_out = lens_out;
    a.move = static_cast<int2 *>(ws);
    a.moves = reinterpret_cast<int32_t *>(a.move + seqs * heads * most);
    a.slot_from = slot_from ? slot_from : a.moves + seqs * heads;
    a.heads = static_cast<int>(heads), a.slots = history->slots, a.slots_out = left->slots;
    a.max_len = static_cast<int>(max_len), a.keep = static_cast<int>(keep), a.recent = static_cast<int>(recent);
    a.most = static_cast<int>(most), a.vecs = a.c.d * a.c.elem / 16;
    hipStream_t s = as_stream(stream);
    if (most <= kFew) {
        choose<true>(a, static_cast<unsigned>(seqs), s);
        return check_launch("kv_choose_kernel");
    }
    choose<false>(a, static_cast<unsigned>(seqs), s);
    if ((st = check_launch("kv_choose_kernel"))) return st;
    const unsigned rows = kMoveThreads / (a.vecs <= 16 ? 16 : a.vecs <= 32 ? 32 : 64);
    const dim3 grid(static_cast<unsigned>((most + rows - 1) / rows), a.c.n_head_kv, static_cast<unsigned>(seqs));
    hipLaunchKernelGGL(kv_move_kernel, grid, dim3(kMoveThreads), 0, s, a);
    return check_launch("kv_move_kernel");
}

}  // extern "C"
