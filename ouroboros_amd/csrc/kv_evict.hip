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
    int32_t *pos_out, *lens_out, *slot_from;  // slot_from [seqs][heads][n_from]
    int2 *move;                               // [seqs][heads][most]: a slot to fill, and the slot that fills it
    int32_t *moves;                           // [seqs][heads]
    int32_t heads, slots, slots_out, max_len, keep, recent, most, vecs;  // vecs: 16-byte vectors of a row
    int32_t n_from, pad;  // n_from: keep, in the workspace no more than max_len
};
// passed by value to kernels: the host and device passes must lay it out alike
static_assert(sizeof(EvictArgs) == 184, "EvictArgs: kernel argument layout");

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));

// Orders of slots in one unsigned: 0 of what goes whatever its weight,
// 0xffffffff of what stays whatever its weight, between them a weight's (NaN
// lowest, -0 as +0).
constexpr uint32_t kGoes = 0u, kStays = 0xffffffffu, kLeast = 1u, kMost = 0xff800000u;
__device__ __forceinline__ uint32_t weight_order(float w) {
    const uint32_t u = __float_as_uint(w + 0.f);
    return w != w ? kLeast : u ^ (static_cast<uint32_t>(static_cast<int32_t>(u) >> 31) | 0x80000000u);
}

// Lanes of the mask below this one.
__device__ __forceinline__ int rank_in(unsigned long long mask) {
    return __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(mask >> 32), __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(mask), 0));
}

// Over the 16 lanes of a row of the wavefront, to each of them.
template <typename F>
__device__ __forceinline__ int row_join(int v, F f) {
    v = f(v, __builtin_amdgcn_update_dpp(0, v, 0x128, 0xf, 0xf, false));
    v = f(v, __builtin_amdgcn_update_dpp(0, v, 0x141, 0xf, 0xf, false));
    v = f(v, __builtin_amdgcn_update_dpp(0, v, 0x4E, 0xf, 0xf, false));
    return f(v, __builtin_amdgcn_update_dpp(0, v, 0xB1, 0xf, 0xf, false));
}

// Copies rows of k and v of one (kv head, sequence), lanes of 16 bytes, from the
// pair `first` on in steps of `step`.
__device__ __forceinline__ void move_rows(const EvictArgs &a, int64_t b, int h, const int2 *move, int n, int first, int step, int lane) {
    if (lane >= a.vecs) return;
    const int64_t head = h * a.c.head_stride * a.c.elem + lane * 16;
    char *k = static_cast<char *>(a.c.k) + head, *v = static_cast<char *>(a.c.v) + head;
    for (int i = first; i < n; i += step) {
        const int2 m = move[i];
        const int64_t dst = kv_slot(a.c, b, m.x) * a.c.elem, src = kv_slot(a.c, b, m.y) * a.c.elem;
        if (src < 0 || dst < 0) continue;  // a hole, which the caller promised not to have: no access through it
        const u32x4_t x = *reinterpret_cast<const u32x4_t *>(k + src), y = *reinterpret_cast<const u32x4_t *>(v + src);
        // not kept by the caches, which whoever reads the row next is not behind
        // (100 MB moved: 27.5 us, 33.1 with plain stores, 30.9 with loads past them too)
        __builtin_nontemporal_store(x, reinterpret_cast<u32x4_t *>(k + dst));
        __builtin_nontemporal_store(y, reinterpret_cast<u32x4_t *>(v + dst));
    }
}

constexpr int kThreads = 1024, kWaves = kThreads / 64;
constexpr int kBinBits = 11, kBins = 1 << kBinBits, kCopies = 4;  // bins of a count, and how many lanes' counts share one

// The choice of one (head, sequence) by one workgroup of 16 wavefronts, each
// with a run of slots in order, 64 R of them in registers (longer runs, past
// 16384 places with the up to 63 before slot 0, are read again at each pass:
// the whole call for 4 rows of 16384 slots cut to 2048 25 us, to 2000 40, 4 of
// 16385 42, of 40000 67).  The runs' blocks of 64 start so that one starts at
// slot `keep`: what a block's slots may become is the same for all of them.  The
// order of the last slot that stays is found from counts in bins, from the
// largest order down, first of all orders, then of the bin that holds it.
// Moves: the workgroup copies the rows too.
//
// Bound by instructions and barriers: a pass over 16384 slots costs a workgroup
// 256 cycles for each instruction a slot takes, a barrier about 400.  Four rows
// of 16384 slots, a workgroup each: 17.5 us, of which the counts in bins 4, the
// two passes over what stays 5, loads 2.  64 rows of 1025 slots, 4 heads: 7.8 us
// with the launch.  Counting thresholds with ballots, 12 rounds of three, took
// 14 us more.
template <int R, bool Moves>
__global__ __launch_bounds__(kThreads) void kv_choose_kernel(EvictArgs a) {
    __shared__ int4 tmp[2][kWaves];
    __shared__ __align__(16) int bins[kBins * kCopies];
    __shared__ int4 found;
    const int hs = blockIdx.x, t = threadIdx.x, lane = t & 63;
    const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int64_t b = blockIdx.y, row = b * a.heads + hs;
    const int n = max(0, min(a.lens[b], a.max_len)), keep = a.keep;
    const float *weight = a.weight + row * a.slots;
    const int32_t *pos = a.pos + row * a.slots;
    int32_t *from = a.slot_from + row * a.n_from;
    float *w_out = a.weight_out + row * a.slots_out;
    int32_t *pos_out = a.pos_out + row * a.slots_out;
    const bool apart = w_out != weight;
    if (hs == 0 && t == 0) a.lens_out[b] = min(n, keep);
    if (n <= keep) {
        for (int j = t; j < a.n_from; j += kThreads) from[j] = j < n ? j : -1;
        if (!Moves && t == 0) a.moves[row] = 0;
        if (apart)
            for (int j = t; j < n; j += kThreads) w_out[j] = weight[j], pos_out[j] = pos[j];
        return;
    }
    for (int i = t; i < kBins; i += kThreads) reinterpret_cast<int4 *>(bins)[i] = make_int4(0, 0, 0, 0);
    int round = 0;
    // A wavefront's counts joined: the sums over all wavefronts, and those over
    // the ones before it.
    int4 all, before;
    auto join = [&](int x, int y, int z) __attribute__((always_inline)) {
        int4 *buf = tmp[round++ & 1];  // a wavefront is at most one round ahead
        if (lane == 0) buf[wave] = make_int4(x, y, z, 0);
        __syncthreads();
        const int4 o = buf[lane % kWaves];
        auto add = [](int p, int q) { return p + q; };
        const bool is = lane % kWaves < wave;
        all = make_int4(row_join(o.x, add), row_join(o.y, add), row_join(o.z, add), 0);
        before = make_int4(row_join(is ? o.x : 0, add), row_join(is ? o.y : 0, add), row_join(is ? o.z : 0, add), 0);
    };
    const int front = -keep & 63;  // places before slot 0
    const int run = (n + front + kThreads - 1) / kThreads * 64;  // places of a wavefront
    const int j0 = wave * run - front;
    float w[R];
    uint32_t u[R];  // the position, then how far it is behind the newest
    uint32_t o[R];
    auto slot = [&](int c, int i) __attribute__((always_inline)) { return c + i * 64 < run && static_cast<uint32_t>(j0 + c + i * 64 + lane) < static_cast<uint32_t>(n); };
    auto load = [&](int c) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < R; ++i) {
            w[i] = 0.f, u[i] = static_cast<uint32_t>(INT32_MIN);
            if (slot(c, i)) w[i] = weight[j0 + c + i * 64 + lane], u[i] = pos[j0 + c + i * 64 + lane];
        }
    };
    const bool once = run <= 64 * R;
    // the newest: positions past max - recent
    load(0);
    int newest = INT32_MIN;
    for (int c = 0; c < run; c += 64 * R) {
        if (c) load(c);
#pragma unroll
        for (int i = 0; i < R; ++i) newest = max(newest, static_cast<int>(u[i]));
    }
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) newest = max(newest, xor_shfl(newest, off));
    {
        int4 *buf = tmp[round++ & 1];
        if (lane == 0) buf[wave].x = newest;
        __syncthreads();
        newest = row_join(buf[lane % kWaves].x, [](int x, int y) { return x > y ? x : y; });
    }
    // new: newest - pos < recent, a difference that 32 bits hold unsigned
    const uint32_t recent = a.recent;
    auto behind = [&](int c) __attribute__((always_inline)) {
        if (!once) load(c);
#pragma unroll
        for (int i = 0; i < R; ++i) u[i] = slot(c, i) ? newest - u[i] : 0xffffffffu;
    };
    int news = 0;
    for (int c = 0; c < run; c += 64 * R) {
        behind(c);
#pragma unroll
        for (int i = 0; i < R; ++i) news += __popcll(__ballot(u[i] < recent));
    }
    join(news, 0, 0);
    // whichever class is cut: the newest alone where they fill the budget, else the others
    const bool cut = all.x >= keep;
    const uint32_t other = cut ? kGoes : kStays;
    auto orders = [&](int c) __attribute__((always_inline)) {
        if (!once) behind(c);
#pragma unroll
        for (int i = 0; i < R; ++i) {
            o[i] = (u[i] < recent) == cut ? weight_order(w[i]) : other;
            if (!slot(c, i)) o[i] = kGoes;
        }
    };
    if (once) orders(0);
    // the largest order that `keep` slots reach, in lo .. hi
    uint32_t lo = kLeast, hi = kMost;
    int need = cut ? keep : keep - all.x;  // slots of lo .. hi that stay
    bool exact = false;
    for (;;) {
        const int shift = max(0, 32 - static_cast<int>(__clz(hi - lo)) - kBinBits);
        for (int c = 0; c < run; c += 64 * R) {
            if (!once) orders(c);
#pragma unroll
            for (int i = 0; i < R; ++i) {
                if (c + i * 64 >= run) break;
                if (o[i] - lo <= hi - lo) atomicAdd(&bins[((hi - o[i]) >> shift) * kCopies + lane % kCopies], 1);
            }
        }
        __syncthreads();
        int mine[kBins / kThreads], sum = 0;
#pragma unroll
        for (int i = 0; i < kBins / kThreads; ++i) {
            int4 *bin = reinterpret_cast<int4 *>(bins) + t * (kBins / kThreads) + i;
            const int4 q = *bin;
            *bin = make_int4(0, 0, 0, 0);
            sum += mine[i] = q.x + q.y + q.z + q.w;
        }
        int up = sum;  // over the lanes up to this one
        up += __builtin_amdgcn_update_dpp(0, up, 0x111, 0xf, 0xf, false);
        up += __builtin_amdgcn_update_dpp(0, up, 0x112, 0xf, 0xf, false);
        up += __builtin_amdgcn_update_dpp(0, up, 0x114, 0xf, 0xf, false);
        up += __builtin_amdgcn_update_dpp(0, up, 0x118, 0xf, 0xf, false);
        up += __builtin_amdgcn_update_dpp(0, up, 0x142, 0xa, 0xf, false);
        up += __builtin_amdgcn_update_dpp(0, up, 0x143, 0xc, 0xf, false);
        join(__builtin_amdgcn_readlane(up, 63), 0, 0);
        int past = before.x + up - sum;  // in the bins of larger orders
#pragma unroll
        for (int i = 0; i < kBins / kThreads; ++i) {
            if (past < need && past + mine[i] >= need) found = make_int4(t * (kBins / kThreads) + i, past, mine[i], 0);
            past += mine[i];
        }
        __syncthreads();
        const int bin = __builtin_amdgcn_readfirstlane(found.x), over = __builtin_amdgcn_readfirstlane(found.y), in = __builtin_amdgcn_readfirstlane(found.z);
        hi -= static_cast<uint32_t>(bin) << shift;
        const uint32_t width = (1u << shift) - 1;
        if (hi - lo > width) lo = hi - width;
        need -= over;
        if (need == in) {  // those of the bin stay to the last
            --lo;
            exact = true;
            break;
        }
        if (lo == hi) break;
    }
    // of those at lo, the slots up to `last` stay
    int last = -1;
    if (!exact) {
        int at = 0;
        for (int c = 0; c < run; c += 64 * R) {
            if (!once) orders(c);
#pragma unroll
            for (int i = 0; i < R; ++i) at += __popcll(__ballot(o[i] == lo));
        }
        join(at, 0, 0);
        int seen = __builtin_amdgcn_readfirstlane(before.x);
        if (seen < need && seen + at >= need)
            for (int c = 0; c < run; c += 64 * R) {
                if (!once) orders(c);
#pragma unroll
                for (int i = 0; i < R; ++i) {
                    const unsigned long long is = __ballot(o[i] == lo);
                    if (o[i] == lo && seen + rank_in(is) == need - 1) found.x = j0 + c + i * 64 + lane;
                    seen += __popcll(is);
                }
            }
        __syncthreads();
        last = __builtin_amdgcn_readfirstlane(found.x);
    }
    auto stays = [&](int c, int i) __attribute__((always_inline)) { return __ballot(o[i] > (i * 64 <= last - j0 - c - lane ? lo - 1 : lo)); };
    // those that go below `keep`, those that stay from it on
    int under = 0, over = 0;
    const int cross = keep - j0;  // the first of the run's places from `keep` on
    for (int c = 0; c < run; c += 64 * R) {
        if (!once) orders(c);
#pragma unroll
        for (int i = 0; i < R; ++i) {
            if (c + i * 64 >= run) break;
            const int s = __popcll(stays(c, i));
            if (c + i * 64 < cross)
                under += 64 - s;
            else
                over += s;
        }
    }
    if (wave == 0) under -= front;
    join(under, over, 0);
    const int moves = all.y;
    int hole = __builtin_amdgcn_readfirstlane(before.x), mover = __builtin_amdgcn_readfirstlane(before.y);
    int2 *move = a.move + row * a.most;
    for (int c = 0; c < run; c += 64 * R) {
        if (!once) orders(c);
#pragma unroll
        for (int i = 0; i < R; ++i) {
            if (c + i * 64 >= run) break;
            const int j = j0 + c + i * 64 + lane;
            const unsigned long long s = stays(c, i);
            if (c + i * 64 < cross) {
                if (s >> lane & 1) {
                    from[j] = j;
                    if (apart) w_out[j] = w[i], pos_out[j] = newest - u[i];
                }
                unsigned long long goes = ~s;
                if (i == 0 && j0 + c < 0) goes &= ~0ull << front;
                if (goes) {
                    if (goes >> lane & 1) move[hole + rank_in(goes)].x = j;
                    hole += __popcll(goes);
                }
            } else if (s) {
                if (s >> lane & 1) move[mover + rank_in(s)].y = j;
                mover += __popcll(s);
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

// One workgroup a (kv head, sequence) and share of its moves: bound by memory,
// 100 MB read and written in 19 us, about a large copy's rate.  Four rows in
// flight a lane instead of one took as long.
__global__ __launch_bounds__(kMoveThreads) void kv_move_kernel(EvictArgs a) {
    const int lanes = a.vecs <= 16 ? 16 : a.vecs <= 32 ? 32 : 64;
    const int h = blockIdx.y, t = threadIdx.x;
    const int64_t b = blockIdx.z, row = b * a.heads + (a.heads > 1 ? h : 0);
    const int groups = kMoveThreads / lanes;
    move_rows(a, b, h, a.move + row * a.most, a.moves[row], blockIdx.x * groups + t / lanes, gridDim.x * groups, t % lanes);
}

// Bytes of moved rows up to which the choosing workgroup moves them itself.  64
// sequences and 4 heads: 256 moves of 512 bytes (128 KiB) 16.6 us by it, 19.9 by
// a second launch, one move 7.9 and 11.3; with one sequence 9.7 and 10.6.  512
// moves of 1 KiB take 19.0 by it and 11.8 with 4 sequences, 29.0 and 27.4 with 48.
constexpr size_t kFew = 128 << 10;

// Moves of a (sequence, head) at the most.
size_t most_moves(size_t max_len, size_t keep) {
    const size_t gone = max_len > keep ? max_len - keep : 0;
    return keep < gone ? keep : gone;
}
// The workspace: the moves, their numbers, n_from entries a row of a slot_from
// that the caller does not ask for.
size_t evict_ws_bytes(size_t seqs, size_t heads, size_t max_len, size_t keep, size_t n_from) {
    return (seqs * heads * (most_moves(max_len, keep) * sizeof(int2) + (n_from + 1) * sizeof(int32_t)) + 255) & ~size_t{255};
}

template <bool Moves>
void choose(const EvictArgs &a, unsigned seqs, hipStream_t s) {
    const dim3 grid(a.heads, seqs);
    // places of the runs: the first block may start up to 63 before slot 0.
    // Registers for fewer of them save what the unrolled passes skip: 1025 slots
    // 8.0 us with 2 a lane, 8.4 with 4; 4032 slots 15.2 with 4, 17.3 with 16.
    const int places = a.max_len + 63;
    if (places <= 2 * kThreads)
        hipLaunchKernelGGL((kv_choose_kernel<2, Moves>), grid, dim3(kThreads), 0, s, a);
    else if (places <= 4 * kThreads)
        hipLaunchKernelGGL((kv_choose_kernel<4, Moves>), grid, dim3(kThreads), 0, s, a);
    else
        hipLaunchKernelGGL((kv_choose_kernel<16, Moves>), grid, dim3(kThreads), 0, s, a);
}

}  // namespace
}  // namespace ouro

using namespace ouro;

extern "C" {

size_t ouro_kv_evict_workspace_bytes(size_t seqs, size_t heads, size_t max_len, size_t keep) {
    return evict_ws_bytes(seqs, heads, max_len, keep, keep);
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
    const size_t heads = history->heads, most = most_moves(max_len, keep);
    const size_t n_from = slot_from ? keep : keep < max_len ? keep : max_len;  // a budget may be far above every length
    if (!ws && !(ws = workspace(evict_ws_bytes(seqs, heads, max_len, keep, slot_from ? 0 : n_from), stream))) return OURO_ERR_HIP;
    a.weight = history->weight, a.pos = history->pos, a.lens = lens;
    a.weight_out = left->weight, a.pos_out = left->pos, a.lens_out = lens_out;
    a.move = static_cast<int2 *>(ws);
    a.moves = reinterpret_cast<int32_t *>(a.move + seqs * heads * most);
    a.slot_from = slot_from ? slot_from : a.moves + seqs * heads;
    a.heads = static_cast<int>(heads), a.slots = history->slots, a.slots_out = left->slots;
    a.max_len = static_cast<int>(max_len), a.keep = static_cast<int>(keep), a.recent = static_cast<int>(recent);
    a.n_from = static_cast<int>(n_from);
    a.most = static_cast<int>(most), a.vecs = a.c.d * a.c.elem / 16;
    hipStream_t s = as_stream(stream);
    if (most * (heads > 1 ? 1 : a.c.n_head_kv) * a.vecs * 32 <= kFew) {
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
