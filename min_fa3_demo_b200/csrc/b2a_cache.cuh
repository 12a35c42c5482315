// The key/value cache as the kernels see it: slots of a sequence, found through a block table or in one piece.
#pragma once

#include "b2a_fwd.cuh"
#include "b2a_host.cuh"

namespace b2a {

// Strides in elements.  Offsets are 64-bit throughout: a pool of pages easily has more than 2^31 elements.
struct CacheView {
    __nv_bfloat16* k;
    __nv_bfloat16* v;
    const int* block_table;     // null: page b holds sequence b
    long long table_stride;
    long long k_stride[3];      // page, row, head
    long long v_stride[3];
    int pages;
    int page_size;
    int heads;
    int table_width;

    __device__ __forceinline__ long long capacity() const {   // slots of a sequence
        return block_table == nullptr ? page_size : static_cast<long long>(page_size) * table_width;
    }
    // Page of a slot; -1: there is none.
    __device__ __forceinline__ int page_of(int seq, long long slot) const {
        if (slot < 0 || slot >= capacity()) return -1;
        const int page = block_table == nullptr ? seq : block_table[seq * table_stride + slot / page_size];
        return page >= 0 && page < pages ? page : -1;
    }
};

// Checks a caller's cache and fills the view.
inline int make_cache_view(const b2a_cache& c, int batch, bool needs_v, CacheView* view) {
    B2A_REQUIRE(c.k != nullptr && (c.v != nullptr || !needs_v), "the cache's k and v must not be NULL");
    B2A_REQUIRE(c.pages >= 1 && c.page_size >= 1 && c.heads_k >= 1, "pages, page_size and heads_k must be positive");
    B2A_REQUIRE((reinterpret_cast<uintptr_t>(c.k) & 0xF) == 0 && (reinterpret_cast<uintptr_t>(c.v) & 0xF) == 0,
                "the cache must be 16-byte aligned");
    for (int i = 0; i < 3; ++i) {
        B2A_REQUIRE(c.k_stride[i] >= 0 && c.v_stride[i] >= 0 && c.k_stride[i] % 8 == 0 && c.v_stride[i] % 8 == 0,
                    "strides of the cache must be multiples of 8 elements");
    }
    if (c.block_table != nullptr) {
        B2A_REQUIRE(c.page_size % 8 == 0, "page_size must be a multiple of 8, got %d", c.page_size);
        B2A_REQUIRE(c.table_width >= 1 && c.table_stride >= 0, "the block table must have at least one column");
        B2A_REQUIRE(static_cast<long long>(c.page_size) * c.table_width <= INT32_MAX, "a sequence must have fewer than 2^31 slots");
    } else {
        B2A_REQUIRE(c.pages >= batch, "a cache without a block table needs a page for each sequence, got %d for %d", c.pages, batch);
    }
    view->k = static_cast<__nv_bfloat16*>(c.k);
    view->v = static_cast<__nv_bfloat16*>(c.v);
    view->block_table = c.block_table;
    view->table_stride = c.table_stride;
    for (int i = 0; i < 3; ++i) {
        view->k_stride[i] = c.k_stride[i];
        view->v_stride[i] = c.v_stride[i];
    }
    view->pages = c.pages;
    view->page_size = c.page_size;
    view->heads = c.heads_k;
    view->table_width = c.table_width;
    return B2A_OK;
}

}  // namespace b2a
