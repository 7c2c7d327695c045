// kv_cache.hpp - what the operators on a caller's paged key-value cache share
// (kv_attend.hip, kv_evict.hip): the cache as a kernel sees it, and the checks
// of its description.
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

}  // namespace ouro
