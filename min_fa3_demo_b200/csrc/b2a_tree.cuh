// What the kernels of b2a_tree_fwd share: parameters, pieces of work, masks, and the V rows that a product must not see.
#pragma once

#include "b2a_cache.cuh"

namespace b2a {

constexpr int kTreeMaxCtas = kFwdStatusWords;

struct TreeParams {
    CacheQueries c;
    __nv_bfloat16* out;
    float* lse;
    long long lse_seq_stride;    // 0 for packed queries
    long long lse_head_stride;
    int tile_tokens;             // 128 / group
    int box_rows;
    float scale_log2;
    unsigned int* status;        // a word for each CTA, behind the header
    uint32_t timeout_ns;
    // Pieces that do not cover their item: two a CTA, the one its run begins with and the one it ends with.
    struct TreeCut* cuts;        // [CTAs]: the item that a run begins inside of
    float2* part_stat;           // [2 * CTAs][part_tiles][part_rows] (row maximum, row sum); few rows: (reference, row sum)
    float4* part_o;              // [2 * CTAs][part_tiles][32][part_rows] O before the division; few rows: [2 * CTAs][part_rows][32]
    int part_tiles;
    int part_rows;
};

struct TreeCut {
    long long first, last;       // the item's blocks in the row of all
    int run;                     // 0: the CTA's run does not begin inside an item
    int seq, q_begin, tok0, n, head;
    int pad[2];
};

// A run's share of an item.
struct TreePiece {
    int valid;
    int seq, q_begin, n, len, slots, head;
    int tok0;        // first token
    int tokens[2];   // of the two tiles
    int j0, blocks;
    int part;        // where its part goes; -1: it covers the item
};

// What tree_combine has to know of the item that this CTA's run begins inside of.
__device__ __forceinline__ TreeCut tree_cut(const TreeParams& p, const CacheWalk& walk) {
    TreeCut cut{};
    if (walk.pos < walk.end && walk.j > 0) {
        cut.first = walk.item_begin();
        cut.last = cut.first + walk.blocks;
        cut.run = walk.run;
        cut.seq = walk.seq;
        cut.q_begin = walk.s.q_begin;
        cut.tok0 = walk.rt * p.c.item_tokens;
        cut.n = walk.s.n;
        cut.head = walk.head;
    }
    return cut;
}

// The walk's next piece.
__device__ __forceinline__ TreePiece tree_piece(const TreeParams& p, const CacheWalk& walk) {
    TreePiece w{};
    w.valid = walk.pos < walk.end;
    if (w.valid) {
        w.seq = walk.seq;
        w.q_begin = walk.s.q_begin;
        w.n = walk.s.n;
        w.len = walk.s.len;
        w.slots = walk.s.slots;
        w.head = walk.head;
        w.tok0 = walk.rt * p.c.item_tokens;
        w.tokens[0] = min(p.tile_tokens, w.n - w.tok0);
        w.tokens[1] = max(0, min(p.tile_tokens, w.n - w.tok0 - p.tile_tokens));
        w.j0 = walk.j;
        w.blocks = walk.piece();
        // The item that the run begins inside of (or with), or another one, which then crosses the run's end.
        const bool other = walk.item_begin() > static_cast<long long>(blockIdx.x) * walk.run;
        w.part = w.blocks == walk.blocks ? -1 : 2 * static_cast<int>(blockIdx.x) + (other ? 1 : 0);
    }
    return w;
}

// Loads of V by one warp: the blocks of all pieces, one behind the other.
template <int kSlots, int kStages, typename Shared>
__device__ __forceinline__ void tree_load_v(const TreeParams& p, Shared& sh, const CUtensorMap* map, const WaitCtx& wctx, int lane) {
    SlotLoader loader(p.box_rows);
    uint32_t v_it = 0;
    bool ok = true;
    PH_DECL(3)   // 0 other, 1 wait for V's stage, 2 issue V
    for (uint32_t it = 0; ok; ++it) {
        const uint32_t at = it % kSlots;
        ok = warp_wait(wctx, smem_u32(&sh.piece_full[at]), (it / kSlots) & 1u, 4);
        if (!ok) break;
        const TreePiece w = sh.piece[at];
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&sh.piece_empty[at]));
        if (!w.valid) break;
        loader.look_up(p.c.cache, w.seq, w.j0, w.slots, lane);
        for (int i = 0; i < w.blocks; ++i, ++v_it) {
            SlotLoader now = loader;
            if (i + 1 < w.blocks) loader.look_up(p.c.cache, w.seq, w.j0 + i + 1, w.slots, lane);
            const int boxes = now.count(w.j0 + i, w.slots);
            const uint32_t stage = v_it % kStages;
            PH_MARK(0);
            ok = warp_wait(wctx, smem_u32(&sh.v_empty[stage]), ((v_it / kStages) & 1u) ^ 1u, 18);
            if (!ok) break;
            PH_MARK(1);
            now.load(map, smem_u32(&sh.v[stage][0]), smem_u32(&sh.v_full[stage]), w.head, boxes, lane);
            PH_MARK(2);
        }
    }
    PH_PRINT("tree load", 3);
}

__device__ __forceinline__ const unsigned char* tree_mask_row(const TreeParams& p, const TreePiece& w, int token) {
    return p.c.mask + (p.c.cu_seqlens_q == nullptr ? w.seq * p.c.mask_stride[0] + token * p.c.mask_stride[1]
                                                   : (static_cast<long long>(w.q_begin) + token) * p.c.mask_stride[1]);
}

__device__ __forceinline__ bool tree_sees(const TreeParams& p, const TreePiece& w, int token, int u) {
    return p.c.mask == nullptr ? u <= token : tree_mask_row(p, w, token)[u] != 0;
}

__device__ __forceinline__ bool bf16_not_finite(uint32_t half) { return (half & 0x7F80u) == 0x7F80u; }

// One row of a block of V in shared memory, two halves of 128 bytes: zeros behind the last slot, and of a drafted token no value
// that is not finite, since 0 * NaN is NaN.  Returns whether there was one.
__device__ __forceinline__ bool tree_clean_row(uint8_t* row, int r, bool behind) {
    // Another chunk first in each row, so that rows of 128 bytes do not meet in the same banks.
    auto chunk = [&](int c) { return reinterpret_cast<uint4*>(row + (c >> 3) * kHalfTileBytes + (((c + r) & 7) * 16)); };
    if (behind) {
#pragma unroll
        for (int c = 0; c < 16; ++c) *chunk(c) = make_uint4(0u, 0u, 0u, 0u);
        return false;
    }
    uint32_t ones = 0;      // an exponent of all ones carries into its half's sign bit
#pragma unroll
    for (int c = 0; c < 16; ++c) {
        const uint4 v = *chunk(c);
        ones |= ((v.x & 0x7F807F80u) + 0x00800080u) | ((v.y & 0x7F807F80u) + 0x00800080u) |
                ((v.z & 0x7F807F80u) + 0x00800080u) | ((v.w & 0x7F807F80u) + 0x00800080u);
    }
    if ((ones & 0x80008000u) == 0u) return false;
#pragma unroll 1
    for (int c = 0; c < 16; ++c) {
        const uint4 v = *chunk(c);
        uint32_t words[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (bf16_not_finite(words[e])) words[e] &= 0xFFFF0000u;
            if (bf16_not_finite(words[e] >> 16)) words[e] &= 0xFFFFu;
        }
        *chunk(c) = make_uint4(words[0], words[1], words[2], words[3]);
    }
    return true;
}

// b2a_tree_few.cu: the kernels for calls of at most kFewRows rows an item.  map_q's box holds all of an item's.  Us with them and
// with those of b2a_tree.cu, 32 heads over 8, sequences x slots:
//              1 x 16,384     64 x 2,048      16 x 16,384     4 x 400        32 x 1,000
//    4 rows    24.7  31.5     99.1  113.2     171.6  174.6    12.4  16.0     35.2  42.8
//   16         25.9  32.1    104.2  119.1     175.2  178.9    14.1  16.9     38.7  45.8
//   32         30.8  33.4    121.1  122.2     185.3  182.3    16.5  17.4     50.0  47.1
//   64         45.0  41.6    190.3  142.5     251.3  186.0    22.2  19.9     78.5  53.7
constexpr int kFewRows = 32;
int launch_tree_few(const CUtensorMap& map_q, const CUtensorMap& map_k, const CUtensorMap& map_v, const TreeParams& p, int ctas,
                    const DeviceInfo& dev, cudaStream_t stream);

// Adds up the pieces of items that ends of runs cut: of calls of few rows, and of the others.
int launch_tree_combine_few(const TreeParams& p, int ctas, cudaStream_t stream);
int launch_tree_combine(const TreeParams& p, int ctas, cudaStream_t stream);

struct TreeLayout {
    int ctas, tile_tokens, tiles, rows;   // rows of a tile; few rows: of an item, which is one tile
    bool few;
    size_t o, scratch;                    // of the pieces' results behind their sums, and of both
};

// What is kept after a call: header, status words and cuts.
constexpr size_t kTreeCutsAt = align_up(sizeof(WorkspaceHeader) + kFwdStatusWords * sizeof(unsigned int), 256);
constexpr size_t kTreeKept = align_up(kTreeCutsAt + kTreeMaxCtas * sizeof(TreeCut), 256);

inline TreeLayout tree_layout(int seqlen_q, int group, int sms) {
    TreeLayout t{};
    t.ctas = sms < kTreeMaxCtas ? sms : kTreeMaxCtas;
    t.few = static_cast<long long>(seqlen_q) * group <= kFewRows;
    t.tile_tokens = t.few ? seqlen_q : kTileM / group;
    t.tiles = seqlen_q > t.tile_tokens ? 2 : 1;
    t.rows = (t.tiles == 2 ? t.tile_tokens : seqlen_q) * group;
    const size_t parts = 2ull * t.ctas * t.tiles * t.rows;
    t.o = align_up(parts * sizeof(float2), 256);
    t.scratch = t.o + parts * kHeadDim * sizeof(float);
    return t;
}

// N columns of tensor memory.
template <int N>
__device__ __forceinline__ void few_ld(uint32_t taddr, uint32_t (&r)[N]) {
    if constexpr (N == 4) {
        asm volatile("tcgen05.ld.sync.aligned.32x32b.x4.b32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                     : "r"(taddr)
                     : "memory");
    } else if constexpr (N == 8) {
        asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                     : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                     : "r"(taddr)
                     : "memory");
    } else {
#pragma unroll
        for (int i = 0; i < N; i += 16) tmem_ld_x16(taddr + i, r + i);
    }
}

// Sums of N columns over the lanes of a warp, halving the columns as it halves the lanes: lane j ends with the sum of column
// j % N.
template <int N>
__device__ __forceinline__ void few_column_sums(float (&v)[N], int lane) {
#pragma unroll
    for (int d = 16; d >= N; d >>= 1) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xFFFFFFFFu, v[i], d);
    }
#pragma unroll
    for (int d = N / 2; d > 0; d >>= 1) {
        const bool upper = (lane & d) != 0;
#pragma unroll
        for (int i = 0; i < d; ++i) {
            const float low = v[i], high = v[i + d];
            v[i] = (upper ? high : low) + __shfl_xor_sync(0xFFFFFFFFu, upper ? low : high, d);
        }
    }
}

}  // namespace b2a
