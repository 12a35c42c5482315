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
    unsigned int per_page;      // 2^32 / page_size, rounded up

    __device__ __forceinline__ int capacity() const {   // slots of a sequence
        return block_table == nullptr ? page_size : page_size * table_width;
    }
    // A slot's number in the block table, and its row there, without a division: the high half of slot * per_page is the
    // quotient or one more.
    __device__ __forceinline__ int entry_of(int slot, int* row) const {
        int at = static_cast<int>(__umulhi(static_cast<unsigned int>(slot), per_page));
        *row = slot - at * page_size;
        if (*row < 0) {
            --at;
            *row += page_size;
        }
        return at;
    }
    // Page of a slot, and its row; -1: there is none.
    __device__ __forceinline__ int page_of(int seq, long long slot, int* row) const {
        if (slot < 0 || slot >= capacity()) return -1;
        *row = static_cast<int>(slot);
        if (block_table == nullptr) return seq;
        const int page = block_table[seq * table_stride + entry_of(static_cast<int>(slot), row)];
        return page >= 0 && page < pages ? page : -1;
    }
    __device__ __forceinline__ bool has(int seq, int slot) const {
        int row;
        return page_of(seq, slot, &row) >= 0;
    }
    // Where a slot's head lies in K (V), in elements; -1: nowhere.
    __device__ __forceinline__ long long at(const long long (&stride)[3], int page, int row, int head) const {
        return page < 0 ? -1 : page * stride[0] + row * stride[1] + head * stride[2];
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
    view->per_page = c.page_size == 1 ? 0xFFFFFFFFu : 0xFFFFFFFFu / static_cast<unsigned int>(c.page_size) + 1u;
    return B2A_OK;
}

// mbar_wait for a whole warp, with one answer for all its lanes: a lane that gave up alone would leave the others waiting for it at
// the next warp-wide instruction.
__device__ __forceinline__ bool warp_wait(const WaitCtx& ctx, uint32_t bar, uint32_t parity, uint32_t tag) {
    return __all_sync(0xFFFFFFFFu, mbar_wait(ctx, bar, parity, tag));
}

// ---------------------------------------------------------------------------------------
// Work of the kernels that stream the cache once: all blocks of 128 slots of all (sequence, group of query tokens, K/V head),
// in this order, are dealt out to the CTAs in runs of equal length.  The lengths are on the device, so every CTA finds its
// own run: one warp adds up the sequences' blocks, a lane a sequence.  Nothing is handed out while the kernel runs, and no
// list has to be made by a launch before it.  Behind an item's blocks come a few that stand for what its masks, its sums
// and its results cost; a run that begins among those begins with the next item.
// ---------------------------------------------------------------------------------------
constexpr int kSlotBlock = 128;

struct CacheQueries {
    CacheView cache;
    const int* cache_lens;
    const int* cu_seqlens_q;    // null: seqlen_q tokens a sequence
    const unsigned char* mask;  // null: a chain
    long long mask_stride[2];   // bytes: sequence, row
    int batch;
    int seqlen_q;               // most tokens of a sequence
    int total_q;
    int heads_q;
    int group;                  // query heads of a K/V head
    int item_tokens;            // query tokens of an item
    int min_run;                // fewest blocks of a run
    int item_extra;             // what beginning and ending an item costs, in blocks
    int limit_slots;            // slots behind these do not exist (weights with fewer of them than the cache)
};

struct CacheSeq {
    int q_begin;     // row of the first token
    int n;           // query tokens
    int len;         // slots before them
    int slots;       // slots with them
    int bad;         // the lengths do not fit the cache or the batch; what does is used
};

__device__ __forceinline__ CacheSeq cache_seq(const CacheQueries& p, int b) {
    CacheSeq s;
    long long begin = static_cast<long long>(b) * p.seqlen_q, end = begin + p.seqlen_q;
    const long long len = p.cache_lens[b];
    if (p.cu_seqlens_q != nullptr) {
        begin = p.cu_seqlens_q[b];
        end = p.cu_seqlens_q[b + 1];
    }
    s.bad = begin < 0 || end < begin || end > p.total_q || end - begin > p.seqlen_q;
    const long long n = s.bad ? 0 : end - begin;
    const long long cap = min(p.cache.capacity(), p.limit_slots);
    s.q_begin = static_cast<int>(begin);
    s.n = static_cast<int>(n);
    s.len = static_cast<int>(min(max(len, 0ll), cap));
    s.slots = static_cast<int>(min(s.len + n, cap));
    s.bad |= len < 0 || len + n > cap;
    return s;
}

__device__ __forceinline__ int cache_items(const CacheQueries& p, const CacheSeq& s) {
    return s.n > 0 ? (s.n - 1) / p.item_tokens + 1 : 0;     // item_tokens may be any bound that a caller gave
}

// Blocks that item `rt` of a sequence sees; at least one, so that rows that see nothing are written too.
__device__ __forceinline__ int cache_item_blocks(const CacheQueries& p, const CacheSeq& s, int rt) {
    int slots = s.slots;
    if (p.mask == nullptr && (rt + 1ll) * p.item_tokens < s.n) slots = min(slots, s.len + (rt + 1) * p.item_tokens);
    return max(1, (slots + kSlotBlock - 1) / kSlotBlock);
}

__device__ __forceinline__ long long cache_seq_blocks(const CacheQueries& p, const CacheSeq& s) {
    const int items = cache_items(p, s);
    long long blocks = 0;
    if (p.mask != nullptr) {
        blocks = items > 0 ? static_cast<long long>(items) * cache_item_blocks(p, s, 0) : 0;
    } else {
        for (int rt = 0; rt < items; ++rt) blocks += cache_item_blocks(p, s, rt);
    }
    return (blocks + static_cast<long long>(items) * p.item_extra) * p.cache.heads;
}

// A CTA's run [pos, end) and where in it the walk is.  Every lane of the warp holds the same.
struct CacheWalk {
    long long pos, end, total;
    int run;                 // blocks of a whole run
    int seq, rt, head, j;    // block j of this item is next
    int blocks;              // of this item
    int bad;                 // sequences whose lengths do not fit (only the lane's own until start() has returned)
    CacheSeq s;

    __device__ __forceinline__ void start(const CacheQueries& p, int cta, int ctas, int lane) {
        auto blocks_of = [&](int b) -> long long {
            if (b >= p.batch) return 0;
            const CacheSeq q = cache_seq(p, b);
            bad |= q.bad;
            return cache_seq_blocks(p, q);
        };
        bad = 0;
        const long long first = blocks_of(lane);
        total = first;
        for (int b = lane + 32; b < p.batch; b += 32) total += blocks_of(b);
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) total += __shfl_xor_sync(0xFFFFFFFFu, total, d);
        bad = __any_sync(0xFFFFFFFFu, bad);
        run = static_cast<int>(max(static_cast<long long>(p.min_run), (total + ctas - 1) / ctas));
        pos = min(static_cast<long long>(cta) * run, total);
        end = min(pos + run, total);
        if (pos >= end) return;
        long long before = 0;
        for (int b = 0;; b += 32) {
            const long long mine = b == 0 ? first : blocks_of(b + lane);
            long long upto = mine;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const long long up = __shfl_up_sync(0xFFFFFFFFu, upto, d);
                if (lane >= d) upto += up;
            }
            const unsigned found = __ballot_sync(0xFFFFFFFFu, before + upto > pos);
            if (found != 0u) {
                const int at = __ffs(found) - 1;
                seq = b + at;
                before += __shfl_sync(0xFFFFFFFFu, upto - mine, at);
                break;
            }
            before += __shfl_sync(0xFFFFFFFFu, upto, 31);
        }
        s = cache_seq(p, seq);
        long long off = pos - before;
        rt = 0;
        blocks = cache_item_blocks(p, s, 0);
        while (off >= static_cast<long long>(blocks + p.item_extra) * p.cache.heads) {
            off -= static_cast<long long>(blocks + p.item_extra) * p.cache.heads;
            blocks = cache_item_blocks(p, s, ++rt);
        }
        head = static_cast<int>(off / (blocks + p.item_extra));
        j = static_cast<int>(off - static_cast<long long>(head) * (blocks + p.item_extra));
        if (j >= blocks) advance(p, 0);
    }
    __device__ __forceinline__ long long item_begin() const { return pos - j; }
    // Blocks [j, j + piece()) of the item are the next piece.
    __device__ __forceinline__ int piece() const { return static_cast<int>(min(static_cast<long long>(blocks - j), end - pos)); }
    __device__ __forceinline__ void advance(const CacheQueries& p, int count) {
        pos += count;
        j += count;
        if (j < blocks) return;
        pos += blocks + p.item_extra - j;
        if (pos >= end) return;
        j = 0;
        if (++head < p.cache.heads) return;
        head = 0;
        if (++rt >= cache_items(p, s)) {
            rt = 0;
            do {
                s = cache_seq(p, ++seq);   // there is one: the run has blocks left
            } while (s.n == 0);
        }
        blocks = cache_item_blocks(p, s, rt);
    }
};

// Rows of a TMA box over slots: pages of 128 slots and more are read in whole blocks, and smaller or odd ones in the largest
// power of two that never crosses the end of a page.  A cache of one piece ends in a box that TMA fills with zeros.
inline int slot_box_rows(const CacheView& c) {
    if (c.block_table == nullptr) return kSlotBlock;
    int rows = 8;
    while (rows < kSlotBlock && c.page_size % (2 * rows) == 0) rows *= 2;
    return rows;
}

inline int make_slot_map(CUtensorMap* map, const CacheView& c, bool keys, int box_rows) {
    const uint64_t sizes[3] = {static_cast<uint64_t>(c.pages), static_cast<uint64_t>(c.page_size), static_cast<uint64_t>(c.heads)};
    const long long* st = keys ? c.k_stride : c.v_stride;
    const int64_t strides[3] = {st[0], st[1], st[2]};
    return make_strided_map(map, keys ? c.k : c.v, 4, sizes, strides, 1, static_cast<uint32_t>(box_rows));
}

// Loads blocks of slots by one warp: a lane for each box of the block.  A lane asks for its page a block ahead and looks at the
// answer only when it needs it, so that neither the block table's latency nor a division is on the path.
struct SlotLoader {
    int shift, boxes;        // rows of a box, a power of two
    int page, row;
    int bad;                 // this lane met a page that does not exist

    // blocks: that are looked up and loaded together; their boxes are at most 32.
    __device__ __forceinline__ explicit SlotLoader(int box_rows, int blocks = 1) {
        shift = __ffs(box_rows) - 1;
        boxes = blocks * kSlotBlock >> shift;
        page = row = bad = 0;
    }

    __device__ __forceinline__ void look_up(const CacheView& c, int seq, int block, int slots, int lane) {
        const int slot = block * kSlotBlock + (lane << shift);
        if (lane >= boxes || slot >= slots) return;
        if (c.block_table == nullptr) {
            page = seq;
            row = slot;
            return;
        }
        const int at = c.entry_of(slot, &row);
        page = c.block_table[seq * c.table_stride + at];
    }
    // Boxes of a block that hold slots.
    __device__ __forceinline__ int count(int block, int slots) const {
        return min(boxes, max(0, (slots - block * kSlotBlock + (1 << shift) - 1) >> shift));
    }
    __device__ __forceinline__ void load(const CUtensorMap* map, uint32_t dst, uint32_t bar, int head, int n, int lane) {
        if (lane == 0) mbar_arrive_expect_tx(bar, static_cast<uint32_t>(n << shift) * 256u);
        __syncwarp();
        if (lane < n) {
            const uint32_t at = dst + static_cast<uint32_t>(lane << shift) * 128u;
            tma_load_4d(at, map, bar, 0, head, row, page);
            tma_load_4d(at + kHalfTileBytes, map, bar, 64, head, row, page);
        }
        __syncwarp();
    }
    // Before a block is loaded: whether one of its pages does not exist.  TMA fills such a box with zeros, and its slots must not
    // take part, so the CTA is told (`missing`, in shared memory, never taken back: its blocks then look up their pages).
    __device__ __forceinline__ void check(const CacheView& c, int n, int lane, uint32_t* missing) {
        const int gone = lane < n && static_cast<unsigned>(page) >= static_cast<unsigned>(c.pages);
        bad |= gone;
        if (__any_sync(0xFFFFFFFFu, gone) && lane == 0) *reinterpret_cast<volatile uint32_t*>(missing) = 1u;
        __syncwarp();
    }
};

// Checks the arguments that b2a_tree_fwd and b2a_cache_weights share.
inline int make_cache_queries(const b2a_tree_args& a, bool needs_v, CacheQueries* q) {
    const int rc = make_cache_view(a.cache, a.batch, needs_v, &q->cache);
    if (rc != B2A_OK) return rc;
    B2A_REQUIRE(a.q != nullptr && a.lse != nullptr && a.cache_lens != nullptr, "q, lse and cache_lens must not be NULL");
    B2A_REQUIRE((reinterpret_cast<uintptr_t>(a.q) & 0xF) == 0, "q must be 16-byte aligned");
    B2A_REQUIRE(a.batch >= 1 && a.seqlen_q >= 1 && a.total_q >= 1, "batch, seqlen_q and total_q must be positive");
    B2A_REQUIRE(a.heads_q >= 1 && a.heads_q % a.cache.heads_k == 0, "heads_q %% heads_k must be 0, got heads_q=%d heads_k=%d",
                a.heads_q, a.cache.heads_k);
    B2A_REQUIRE(a.heads_q / a.cache.heads_k <= kTileM, "at most %d query heads may share a K/V head, got %d", kTileM,
                a.heads_q / a.cache.heads_k);
    if (a.cu_seqlens_q == nullptr) {
        B2A_REQUIRE(static_cast<long long>(a.batch) * a.seqlen_q == a.total_q,
                    "fixed-length sizes must satisfy total_q = batch * seqlen_q");
    }
    B2A_REQUIRE(a.mask_stride[0] >= 0 && a.mask_stride[1] >= 0, "strides of tree_mask must not be negative");
    q->cache_lens = a.cache_lens;
    q->cu_seqlens_q = a.cu_seqlens_q;
    q->mask = a.tree_mask;
    q->mask_stride[0] = a.mask_stride[0];
    q->mask_stride[1] = a.mask_stride[1];
    q->batch = a.batch;
    q->seqlen_q = a.seqlen_q;
    q->total_q = a.total_q;
    q->heads_q = a.heads_q;
    q->group = a.heads_q / a.cache.heads_k;
    q->limit_slots = INT32_MAX - 2 * kSlotBlock;   // so that slot numbers of whole blocks fit in 32 bits
    return B2A_OK;
}

}  // namespace b2a
