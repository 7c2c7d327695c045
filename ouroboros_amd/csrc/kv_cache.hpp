// kv_cache.hpp - what the operators on a caller's paged key-value cache share
// (kv_attend.hip, kv_evict.hip; of 8-bit codes kv8_cache.hip, kv8_attend.hip):
// the cache as a kernel sees it, and the checks of its description.
#pragma once

#include "common.hpp"

namespace ouro {

// A cache by value in a kernel's arguments.  Slot j of sequence b is token
// j % page_tokens of page pages[b * max_pages + j / page_tokens]; an id
// outside 0 .. n_pages - 1 is a hole, whose slots hold nothing.
struct KvView {
    void *k, *v;
    const int32_t *pages;
    int64_t page_stride, token_stride, head_stride;  // elements
    int32_t n_pages, max_pages, page_shift, n_head_kv, d;
    int32_t elem;  // bytes of an element
};
// passed by value to kernels: the host and device passes must lay it out alike
static_assert(sizeof(KvView) == 72, "KvView: kernel argument layout");

// Element offset of (sequence, slot) in the pools before the head's offset,
// -1 for a slot of a hole.  64 bits: a pool may pass 2^32 elements.
__device__ __forceinline__ int64_t kv_slot(const KvView &c, int64_t seq, int slot) {
    const int32_t page = c.pages[seq * c.max_pages + (slot >> c.page_shift)];
    if (page < 0 || page >= c.n_pages) return -1;
    return page * c.page_stride + (slot & ((1 << c.page_shift) - 1)) * c.token_stride;
}

// Checks a description and fills the view; `what` names the entry point.
int kv_view(const ouro_kv_cache *cache, const char *what, KvView *out);
// Checks a history of `slots` >= need slots against the cache.
int kv_check_history(const ouro_kv_history *h, int n_head_kv, size_t need, const char *what);

// A cache of 8-bit codes: element = code * scale, a scale for each block of
// 1 << block_shift slots of a page and kv head.
struct Kv8View {
    int8_t *k, *v;
    float *k_scale, *v_scale;
    const int32_t *pages;
    int64_t page_stride, token_stride, head_stride;  // bytes
    int32_t n_pages, max_pages, page_shift, block_shift, n_head_kv, d;
};
static_assert(sizeof(Kv8View) == 88, "Kv8View: kernel argument layout");

// Byte offset of token t of a page that is there, before the head's offset.
__device__ __forceinline__ int64_t kv8_row(const Kv8View &c, int32_t page, int t) {
    return page * c.page_stride + t * c.token_stride;
}
// Index of the scale of token t of a page that is there.
__device__ __forceinline__ int64_t kv8_scale(const Kv8View &c, int32_t page, int t, int head) {
    return ((static_cast<int64_t>(page) << (c.page_shift - c.block_shift)) + (t >> c.block_shift)) * c.n_head_kv + head;
}
int kv8_view(const ouro_kv8_cache *cache, const char *what, Kv8View *out);

// The newest rows of each sequence, packed one after another.
struct NewRows {
    const int32_t *lens, *cu;  // cu NULL: max_new rows each
    int32_t rows, max_new, max_len;
};
static_assert(sizeof(NewRows) == 32, "NewRows: kernel argument layout");

// A sequence's: its slots in use, its first packed row and how many it has, each
// held to its range whatever the arrays say.  Row i is slot n - count + i, none
// where that is below 0.
struct SeqRows {
    int n, first, count;
};
__device__ __forceinline__ SeqRows seq_rows(const NewRows &a, int64_t b) {
    SeqRows s;
    s.n = a.lens ? max(0, min(a.lens[b], a.max_len)) : 0;
    if (a.cu) {
        s.first = max(0, min(a.cu[b], a.rows));
        s.count = min(max(min(a.cu[b + 1], a.rows) - s.first, 0), a.max_new);
    } else {
        s.first = static_cast<int>(b) * a.max_new;
        s.count = a.max_new;
    }
    return s;
}
// Checks seqs, rows and max_new against each other and fills the view.
int new_rows(const int32_t *lens, const int32_t *cu, size_t seqs, size_t rows, size_t max_new, size_t max_len, const char *what,
             NewRows *out);

}  // namespace ouro
