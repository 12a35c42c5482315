// What attention the slots of a cache received: w[b, h, slot] += sum over the rows of K/V head h that see the slot of
// exp(scale q k - lse).
//
// The scores are made the other way round than for attention, S^T = K Q^T: a thread has a slot, its row of tensor memory the
// scores of all query rows with it, and the sum is its own.  No slot is shared by two threads or CTAs, so nothing is reduced
// between them and repeated calls give the same bits.  K is streamed once where the rows of a sequence fit two tiles of
// 128 (256 bytes a slot and head: bound by memory for up to some 128 rows, by the exponentials beyond); of more rows, two
// tiles' worth at a time go over the same few blocks, which then come from L2, and the sums wait in shared memory.
//
//   warp 0-15   sums, in four groups that take turns at the blocks: bound by the special-function unit, which they keep 83% busy
//               (2,048 tokens, 32 heads over 8, 16,384 slots before them: 377 us; two groups take 1.2 times as long; every second or
//               fourth pair of exponentials as a polynomial on the FMA pipe made it slower).  One token, 16 sequences of up to
//               8,001 slots: 152 MB in 31.2 us, 4.9 TB/s
//   warp 16     K Q^T       warp 17   plan, loads of K       warp 18   loads of Q and its lse: pages of 16 slots cost a warp some
//               1,000 clk a block to ask for, which Q must not wait behind
//
// Tensor memory (512 columns): an S^T of 128 columns for each group of warps.
#include "b2a_cache.cuh"

#include <cmath>

namespace b2a {

namespace {

constexpr int kWeightGroups = 4;       // of four warps each, which take turns at the blocks
constexpr int kWeightThreads = 128 * kWeightGroups + 96;
constexpr int kWeightKStages = kWeightGroups, kWeightQSlots = 2;
constexpr int kWeightPass = 2;        // query tiles that go over a chunk's blocks together (256 tokens, 64 heads over 8, 32,768 slots: 169 us
                                      // with two, 172 with one; two have room)
constexpr int kWeightChunk = 16;      // blocks that several passes of query tiles go over
constexpr int kWeightSlots = 4;       // pieces in flight
constexpr int kWeightMmaWarp = 4 * kWeightGroups, kWeightLoadWarp = kWeightMmaWarp + 1, kWeightQWarp = kWeightMmaWarp + 2;

struct WeightParams {
    CacheQueries c;
    const float* lse;
    long long lse_seq_stride, lse_head_stride;
    float* weights;
    long long weights_stride[2];
    int tile_tokens;
    int box_rows;
    float scale_log2;
    unsigned int* status;
    uint32_t timeout_ns;
};

struct WeightPiece {
    int valid;
    int seq, q_begin, n, len, slots, head;
    int j0, blocks;      // at most kWeightChunk
};

struct __align__(1024) WeightShared {
    uint8_t q[kWeightQSlots][kTileBytes];
    uint8_t k[kWeightKStages][kTileBytes];
    float minus_lse2[kWeightQSlots][kTileM];    // -lse * log2(e) of a tile's rows
    uint4 token_columns[kTileM];                // the columns of a tile's token
    uint32_t live[kWeightQSlots][4];            // a bit for each row that exists and has a finite lse: the others give nothing
    float sums[kWeightChunk][kTileM];
    WeightPiece piece[kWeightSlots];
    uint64_t q_full[kWeightQSlots], q_empty[kWeightQSlots];
    uint64_t k_full[kWeightKStages], k_empty[kWeightKStages];
    uint64_t s_full[kWeightGroups], s_empty[kWeightGroups];
    uint64_t piece_full[kWeightSlots], piece_empty[kWeightSlots];
    uint32_t missing;                           // the CTA has met a page that does not exist
    uint32_t tmem_base;
    uint32_t abort_flag;
};

constexpr size_t kWeightSmemBytes = sizeof(WeightShared) + 1024;
static_assert(kWeightSmemBytes <= 227 * 1024, "shared memory of a CTA");

// Of 32 columns those from a number on (which may be anything).
__host__ __device__ __forceinline__ uint32_t columns_from(int from) {
    return from <= 0 ? 0xFFFFFFFFu : from >= 32 ? 0u : 0xFFFFFFFFu << from;
}

__device__ __forceinline__ int weight_tiles(const WeightParams& p, int n) { return (n + p.tile_tokens - 1) / p.tile_tokens; }

// Not inlined: the sums' code would grow by what is hardly ever looked at (one token, 16 sequences of up to 8,001 slots: 31.7 us
// instead of 31.0).
__device__ __noinline__ bool weight_has(const WeightParams& p, int seq, int slot) { return p.c.cache.has(seq, slot); }

// Adds exp2(scale s + minus_lse2) of 16 columns, those of which `see` has a bit.
template <bool kAll>
__device__ __forceinline__ void weight_sum(const uint32_t (&s)[16], const float4* minus_lse2, float sl2, uint32_t see, float2 (&acc)[4]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float4 l4 = minus_lse2[e];
        float2 p0 = fma2(make_float2(__uint_as_float(s[4 * e]), __uint_as_float(s[4 * e + 1])), make_float2(sl2, sl2),
                         make_float2(l4.x, l4.y));
        float2 p1 = fma2(make_float2(__uint_as_float(s[4 * e + 2]), __uint_as_float(s[4 * e + 3])), make_float2(sl2, sl2),
                         make_float2(l4.z, l4.w));
        p0 = make_float2(fast_exp2(p0.x), fast_exp2(p0.y));
        p1 = make_float2(fast_exp2(p1.x), fast_exp2(p1.y));
        if (!kAll) {
            if (!((see >> (4 * e)) & 1u)) p0.x = 0.f;
            if (!((see >> (4 * e + 1)) & 1u)) p0.y = 0.f;
            if (!((see >> (4 * e + 2)) & 1u)) p1.x = 0.f;
            if (!((see >> (4 * e + 3)) & 1u)) p1.y = 0.f;
        }
        acc[(2 * e) & 3] = add2(acc[(2 * e) & 3], p0);
        acc[(2 * e + 1) & 3] = add2(acc[(2 * e + 1) & 3], p1);
    }
}

__global__ void __launch_bounds__(kWeightThreads, 1)
tree_weights(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
             const __grid_constant__ WeightParams p) {
    extern __shared__ uint8_t smem_raw[];
    WeightShared& sh = *reinterpret_cast<WeightShared*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int i = 0; i < kWeightQSlots; ++i) {
            mbar_init(smem_u32(&sh.q_full[i]), 1);
            mbar_init(smem_u32(&sh.q_empty[i]), 1 + 4 * kWeightGroups);      // the products, and the warps that read minus_lse2
        }
        for (int i = 0; i < kWeightKStages; ++i) {
            mbar_init(smem_u32(&sh.k_full[i]), 1);
            mbar_init(smem_u32(&sh.k_empty[i]), 1);
        }
        for (int i = 0; i < kWeightGroups; ++i) {
            mbar_init(smem_u32(&sh.s_full[i]), 1);
            mbar_init(smem_u32(&sh.s_empty[i]), 4);
        }
        for (int i = 0; i < kWeightSlots; ++i) {
            mbar_init(smem_u32(&sh.piece_full[i]), 1);
            mbar_init(smem_u32(&sh.piece_empty[i]), 2 + 4 * kWeightGroups);
        }
        sh.abort_flag = 0;
        sh.missing = 0;
        fence_mbar_init();
        fence_proxy_async_smem();
    }
    if (warp == kWeightMmaWarp) {
        tmem_alloc(smem_u32(&sh.tmem_base), 512);
        tmem_relinquish();
        tc_fence_before_sync();
    }
    for (int k = threadIdx.x; k < p.tile_tokens; k += kWeightThreads) {
        uint32_t columns[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) columns[c] = columns_from(k * p.c.group - 32 * c) & ~columns_from((k + 1) * p.c.group - 32 * c);
        sh.token_columns[k] = make_uint4(columns[0], columns[1], columns[2], columns[3]);
    }
    let_next_kernel_start();
    wait_for_previous_kernel();
    if (threadIdx.x == 0) {
        p.status[blockIdx.x] = 0u;
        if (blockIdx.x == 0) reinterpret_cast<int4*>(p.status)[-1] = make_int4(-static_cast<int>(gridDim.x), 0, 0, 0);
    }
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem_base = *reinterpret_cast<volatile uint32_t*>(&sh.tmem_base);
    const WaitCtx wctx{smem_u32(&sh.abort_flag), p.status, p.timeout_ns, 1u};

    // All roles go through the same order: pieces, pairs of query tiles, fours of blocks, tiles of the pair, blocks.  So each group of
    // warps has its turn before the next product for the same one.
    if (warp == kWeightLoadWarp) {
        if (lane == 0) {
            tma_prefetch_desc(&map_k);
        }
        CacheWalk walk;
        walk.start(p.c, blockIdx.x, gridDim.x, lane);
        SlotLoader loader(p.box_rows);
        loader.bad = walk.bad;
        uint32_t k_it = 0;
        bool ok = true;
        for (uint32_t it = 0; ok; ++it) {
            const uint32_t at = it % kWeightSlots;
            ok = warp_wait(wctx, smem_u32(&sh.piece_empty[at]), ((it / kWeightSlots) & 1u) ^ 1u, 1);
            if (!ok) break;
            WeightPiece w{};
            w.valid = walk.pos < walk.end;
            if (w.valid) {
                w.seq = walk.seq;
                w.q_begin = walk.s.q_begin;
                w.n = walk.s.n;
                w.len = walk.s.len;
                w.slots = walk.s.slots;
                w.head = walk.head;
                w.j0 = walk.j;
                w.blocks = min(walk.piece(), kWeightChunk);
            }
            if (lane == 0) {
                sh.piece[at] = w;
                mbar_arrive(smem_u32(&sh.piece_full[at]));
            }
            if (!w.valid) break;
            const int passes = (weight_tiles(p, w.n) + kWeightPass - 1) / kWeightPass;
            for (int pass = 0; pass < passes && ok; ++pass) {
                loader.look_up(p.c.cache, w.seq, w.j0, w.slots, lane);
                for (int i = 0; i < w.blocks; ++i, ++k_it) {
                    SlotLoader now = loader;
                    if (i + 1 < w.blocks) loader.look_up(p.c.cache, w.seq, w.j0 + i + 1, w.slots, lane);
                    const int boxes = now.count(w.j0 + i, w.slots);
                    const uint32_t stage = k_it % kWeightKStages;
                    ok = warp_wait(wctx, smem_u32(&sh.k_empty[stage]), ((k_it / kWeightKStages) & 1u) ^ 1u, 3);
                    if (!ok) break;
                    now.check(p.c.cache, boxes, lane, &sh.missing);
                    loader.bad |= now.bad;
                    now.load(&map_k, smem_u32(&sh.k[stage][0]), smem_u32(&sh.k_full[stage]), w.head, boxes, lane);
                }
            }
            if (!ok) break;
            walk.advance(p.c, w.blocks);
        }
        if (__any_sync(0xFFFFFFFFu, loader.bad) && lane == 0) set_status(wctx.status_word(), kStatusBadArg, 0x3Fu << 12);
    } else if (warp == kWeightQWarp) {
        if (lane == 0) tma_prefetch_desc(&map_q);
        uint32_t q_it = 0;
        bool ok = true;
        for (uint32_t it = 0; ok; ++it) {
            const uint32_t at = it % kWeightSlots;
            ok = warp_wait(wctx, smem_u32(&sh.piece_full[at]), (it / kWeightSlots) & 1u, 11);
            if (!ok) break;
            const WeightPiece w = sh.piece[at];
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&sh.piece_empty[at]));
            if (!w.valid) break;
            const int tiles = weight_tiles(p, w.n);
            for (int tile = 0; tile < tiles; ++tile) {
                const uint32_t slot = q_it % kWeightQSlots;
                const int tok0 = tile * p.tile_tokens, rows = min(p.tile_tokens, w.n - tok0) * p.c.group;
                // Read before the wait, which is for the last warp to be done with the tile that lies there.
                float lse[4];
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const int r = c * 32 + lane;
                    lse[c] = INFINITY;
                    if (r < rows) {
                        const int token = tok0 + r / p.c.group, head = w.head * p.c.group + r % p.c.group;
                        lse[c] = p.lse[w.seq * p.lse_seq_stride + head * p.lse_head_stride +
                                       (p.c.cu_seqlens_q == nullptr ? token : w.q_begin + token)];
                    }
                }
                ok = warp_wait(wctx, smem_u32(&sh.q_empty[slot]), ((q_it / kWeightQSlots) & 1u) ^ 1u, 2);
                if (!ok) break;
                ++q_it;
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const bool live = !isinf(lse[c]);
                    sh.minus_lse2[slot][c * 32 + lane] = live ? -lse[c] * kLog2e : 0.f;
                    const uint32_t bits = __ballot_sync(0xFFFFFFFFu, live);
                    if (lane == 0) sh.live[slot][c] = bits;
                }
                __syncwarp();
                if (lane == 0) {
                    const uint32_t bar = smem_u32(&sh.q_full[slot]), dst = smem_u32(&sh.q[slot][0]);
                    mbar_arrive_expect_tx(bar, static_cast<uint32_t>(p.tile_tokens * p.c.group) * 256u);
                    tma_load_3d(dst, &map_q, bar, 0, w.head * p.c.group, w.q_begin + tok0);
                    tma_load_3d(dst + kHalfTileBytes, &map_q, bar, 64, w.head * p.c.group, w.q_begin + tok0);
                }
                __syncwarp();
            }
        }
    } else if (warp == kWeightMmaWarp) {
        constexpr uint32_t kStep = kTileBytes >> 4;
        const uint32_t q_lo0 = desc_lo_kmajor(smem_u32(&sh.q[0][0]));
        const uint32_t k_lo0 = desc_lo_kmajor(smem_u32(&sh.k[0][0]));
        uint32_t q_it = 0, k_it = 0;
        uint32_t par = 0;       // bit x: phase of group x's S^T
        uint32_t first_group = 0;   // that takes a piece's first block: the turns go on from piece to piece
        bool ok = true;
        PH_DECL(5)   // 0 other, 1 wait K, 2 wait Q, 3 wait S, 4 issue
        for (uint32_t it = 0; ok; ++it) {
            const uint32_t at = it % kWeightSlots;
            ok = warp_wait(wctx, smem_u32(&sh.piece_full[at]), (it / kWeightSlots) & 1u, 4);
            if (!ok) break;
            const volatile WeightPiece& w = sh.piece[at];
            const int valid = __shfl_sync(0xFFFFFFFFu, w.valid, 0);
            const int blocks = __shfl_sync(0xFFFFFFFFu, w.blocks, 0);
            const int n = __shfl_sync(0xFFFFFFFFu, w.n, 0);
            if (lane == 0) mbar_arrive(smem_u32(&sh.piece_empty[at]));
            __syncwarp();
            if (!valid) break;
            const int tiles = weight_tiles(p, n);
            for (int tile0 = 0; tile0 < tiles && ok; tile0 += kWeightPass) {
                const int here = min(kWeightPass, tiles - tile0);
                for (int i0 = 0; i0 < blocks && ok; i0 += kWeightGroups) {
                    const int count = min(kWeightGroups, blocks - i0);
                    for (int t = 0; t < here && ok; ++t) {
                        const uint32_t slot = (q_it + t) % kWeightQSlots;
                        PH_MARK(0);
                        if (i0 == 0) {
                            ok = warp_wait(wctx, smem_u32(&sh.q_full[slot]), ((q_it + t) / kWeightQSlots) & 1u, 6);
                            if (!ok) break;
                        }
                        PH_MARK(2);
                        // As many columns as the tile has rows, in steps of 16.
                        const int rows = min(p.tile_tokens, n - (tile0 + t) * p.tile_tokens) * p.c.group;
                        const uint32_t idesc = make_idesc_bf16(kTileM, (rows + 15) & ~15, 0, 0);
                        for (int j = 0; j < count; ++j) {
                            const uint32_t x = (first_group + i0 + j) % kWeightGroups;
                            const uint32_t stage = (k_it + j) % kWeightKStages;
                            PH_MARK(0);
                            if (t == 0) {
                                ok = warp_wait(wctx, smem_u32(&sh.k_full[stage]), ((k_it + j) / kWeightKStages) & 1u, 5);
                                if (!ok) break;
                            }
                            PH_MARK(1);
                            ok = warp_wait(wctx, smem_u32(&sh.s_empty[x]), ((par >> x) & 1u) ^ 1u, 7);
                            if (!ok) break;
                            par ^= 1u << x;
                            PH_MARK(3);
                            tc_fence_after_sync();
                            umma_ss_kk_x8_w(tmem_base + x * 128u, k_lo0 + stage * kStep, q_lo0 + slot * kStep, idesc, 0u);
                            tc_commit_w(smem_u32(&sh.s_full[x]));
                            if (t == here - 1) tc_commit_w(smem_u32(&sh.k_empty[stage]));
                            __syncwarp();
                            PH_MARK(4);
                        }
                        if (ok && i0 + count == blocks) tc_commit_w(smem_u32(&sh.q_empty[slot]));
                    }
                    k_it += count;
                }
                q_it += here;
            }
            first_group += blocks;
        }
        PH_PRINT("weights mma", 5);
    } else {
        const int x = warp >> 2, quarter = warp & 3, r = quarter * 32 + lane;
        const uint32_t s_tmem = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16);
        const float sl2 = p.scale_log2;
        uint32_t q_it = 0, s_it = 0, first_group = 0;
        bool ok = true;
        PH_DECL(4)   // 0 other, 1 wait S, 2 sums
        for (uint32_t it = 0; ok; ++it) {
            const uint32_t at = it % kWeightSlots;
            ok = warp_wait(wctx, smem_u32(&sh.piece_full[at]), (it / kWeightSlots) & 1u, 8);
            if (!ok) break;
            const WeightPiece& w = sh.piece[at];
            if (!w.valid) break;
            const int tiles = weight_tiles(p, w.n);
            const int mine = (x - first_group) % kWeightGroups;      // this group's first block
            float* out = p.weights + w.seq * p.weights_stride[0] + w.head * p.weights_stride[1];
            for (int tile0 = 0; tile0 < tiles && ok; tile0 += kWeightPass) {
                const int here = min(kWeightPass, tiles - tile0);
                const bool last = tile0 + kWeightPass >= tiles;
                for (int i = mine; i < w.blocks; i += kWeightGroups) {
                    const int slot = (w.j0 + i) * kSlotBlock + r;
                    const bool tail = (w.j0 + i + 1) * kSlotBlock > w.len;
                    float before = 0.f;
                    if (last && slot < w.slots) before = out[slot];
                    float sum = tile0 == 0 ? 0.f : sh.sums[i][r];
                    for (int t = 0; t < here; ++t, ++s_it) {
                        const uint32_t q_slot = (q_it + t) % kWeightQSlots;
                        const int tok0 = (tile0 + t) * p.tile_tokens, tokens = min(p.tile_tokens, w.n - tok0);
                        const int rows = tokens * p.c.group;
                        // Which columns see this slot: all of them if it lies before the drafted tokens.
                        uint4 some = make_uint4(0xFFFFFFFFu, 0xFFFFFFFFu, 0xFFFFFFFFu, 0xFFFFFFFFu);
                        const int u = slot - w.len;
                        if (tail && u >= 0) {
                            some = make_uint4(0u, 0u, 0u, 0u);
                            if (slot < w.slots && p.c.mask == nullptr) {
                                const int from = max(0, u - tok0) * p.c.group;   // the first column that does
                                some = make_uint4(columns_from(from), columns_from(from - 32), columns_from(from - 64), columns_from(from - 96));
                            } else if (slot < w.slots) {
                                const unsigned char* mask = p.c.mask + u +
                                    (p.c.cu_seqlens_q == nullptr ? w.seq * p.c.mask_stride[0] + tok0 * p.c.mask_stride[1]
                                                                 : (static_cast<long long>(w.q_begin) + tok0) * p.c.mask_stride[1]);
#pragma unroll 8
                                for (int k = 0; k < tokens; ++k) {
                                    const uint4 columns = sh.token_columns[k];
                                    if (mask[k * p.c.mask_stride[1]] != 0) {
                                        some.x |= columns.x;
                                        some.y |= columns.y;
                                        some.z |= columns.z;
                                        some.w |= columns.w;
                                    }
                                }
                            }
                        }
                        PH_MARK(0);
                        ok = warp_wait(wctx, smem_u32(&sh.s_full[x]), s_it & 1u, 9);
                        if (!ok) break;
                        PH_MARK(1);
                        tc_fence_after_sync();
                        float2 acc[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) acc[e] = make_float2(0.f, 0.f);
                        const uint4 live = *reinterpret_cast<const uint4*>(&sh.live[q_slot][0]);
                        const uint32_t see[4] = {some.x & live.x, some.y & live.y, some.z & live.z, some.w & live.w};
                        const uint32_t from = s_tmem + x * 128u;
                        const float4* lse2 = reinterpret_cast<const float4*>(&sh.minus_lse2[q_slot][0]);
                        // The next 16 columns are on their way out of tensor memory while these are added up.  A tile that every
                        // slot of the warp sees whole has no bits to look at (256 tokens, 64 heads over 8, 32,768 slots: 188 us
                        // without this, 169 with).
                        uint32_t s0[16], s1[16];
                        tmem_ld_x16(from, s0);
                        if (rows > 112 && __all_sync(0xFFFFFFFFu, (see[0] & see[1] & see[2] & see[3]) == 0xFFFFFFFFu)) {
#pragma unroll
                            for (int c = 0; c < 8; ++c) {
                                tmem_wait_ld();
                                if (c < 7) tmem_ld_x16(from + (c + 1) * 16, c & 1 ? s0 : s1);
                                weight_sum<true>(c & 1 ? s1 : s0, lse2 + c * 4, sl2, 0xFFFFu, acc);
                            }
                        } else {
#pragma unroll
                            for (int c = 0; c < 8; ++c) {
                                if (c * 16 < rows) {
                                    tmem_wait_ld();
                                    if ((c + 1) * 16 < rows) tmem_ld_x16(from + (c + 1) * 16, c & 1 ? s0 : s1);
                                    const uint32_t bits = see[c >> 1] >> ((c & 1) * 16);
                                    weight_sum<false>(c & 1 ? s1 : s0, lse2 + c * 4, sl2, bits, acc);
                                }
                            }
                        }
                        const float2 both = add2(add2(acc[0], acc[1]), add2(acc[2], acc[3]));
                        tc_fence_before_sync();
                        __syncwarp();
                        if (lane == 0) {
                            mbar_arrive(smem_u32(&sh.s_empty[x]));
                            if (i + kWeightGroups >= w.blocks) mbar_arrive(smem_u32(&sh.q_empty[q_slot]));   // its last block
                        }
                        sum += both.x + both.y;
                        PH_MARK(2);
                    }
                    if (!ok) break;
                    if (!last) {
                        sh.sums[i][r] = sum;
                    } else if (slot < w.slots && (*reinterpret_cast<volatile uint32_t*>(&sh.missing) == 0u || weight_has(p, w.seq, slot))) {
                        out[slot] = before + sum;
                    }
                }
                // A group without a block here has waited for nothing yet: it may give back no tile that is still to come.
                for (int t = 0; t < here && mine >= w.blocks && ok; ++t) {
                    const uint32_t q_slot = (q_it + t) % kWeightQSlots;
                    ok = warp_wait(wctx, smem_u32(&sh.q_full[q_slot]), ((q_it + t) / kWeightQSlots) & 1u, 10);
                    if (ok && lane == 0) mbar_arrive(smem_u32(&sh.q_empty[q_slot]));
                }
                q_it += here;
            }
            if (!ok) break;
            first_group += w.blocks;
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&sh.piece_empty[at]));
        }
        PH_PRINT("weights", 3);
    }

    tc_fence_before_sync();
    __syncthreads();
    if (warp == kWeightMmaWarp) {
        tc_fence_after_sync();
        tmem_dealloc(tmem_base, 512);
    }
}

int set_weight_smem() {
    B2A_CUDA_OK(cudaFuncSetAttribute(tree_weights, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kWeightSmemBytes)));
    return B2A_OK;
}

constexpr size_t kWeightWorkspace = sizeof(WorkspaceHeader) + kFwdStatusWords * sizeof(unsigned int);

}  // namespace

}  // namespace b2a

extern "C" {

size_t b2a_cache_weights_workspace_bytes(void) { return b2a::kWeightWorkspace; }

int b2a_cache_weights(const b2a_tree_args* a, void* cuda_stream) {
    using namespace b2a;
    B2A_REQUIRE(a != nullptr, "args must not be NULL");
    WeightParams p{};
    int rc = make_cache_queries(*a, false, &p.c);
    if (rc != B2A_OK) return rc;
    B2A_REQUIRE(a->weights != nullptr && a->weights_slots >= 1, "weights must not be NULL or empty");
    B2A_REQUIRE(a->weights_stride[0] >= 0 && a->weights_stride[1] >= 0, "strides of weights must not be negative");
    B2A_REQUIRE(a->workspace != nullptr && (reinterpret_cast<uintptr_t>(a->workspace) & 0xF) == 0,
                "workspace must be a 16-byte aligned device pointer");
    if (a->workspace_bytes < kWeightWorkspace) {
        return fail(B2A_ERR_WORKSPACE_TOO_SMALL, "workspace has %zu bytes, need %zu", a->workspace_bytes, kWeightWorkspace);
    }
    DeviceInfo dev{};
    rc = current_device_info(&dev);
    if (rc != B2A_OK) return rc;
    p.tile_tokens = kTileM / p.c.group;
    p.c.item_tokens = a->seqlen_q;               // all rows of a sequence are one item
    p.c.min_run = 1;
    // Several tiles of queries begin anew with each item (0, 2, 4 blocks: 88.9, 75.3, 75.3 us for 256 rows of 32 heads against up to
    // 16,000 slots; one token for 16 sequences 30.4, 30.9, 31.2).
    p.c.item_extra = a->seqlen_q > p.tile_tokens ? 2 : 0;
    p.c.limit_slots = std::min(p.c.limit_slots, a->weights_slots);
    p.box_rows = slot_box_rows(p.c.cache);
    CUtensorMap map_q, map_k;
    const uint64_t q_sizes[2] = {static_cast<uint64_t>(a->total_q), static_cast<uint64_t>(a->heads_q)};
    rc = make_strided_map(&map_q, a->q, 3, q_sizes, a->q_stride, static_cast<uint32_t>(p.c.group), static_cast<uint32_t>(p.tile_tokens));
    if (rc == B2A_OK) rc = make_slot_map(&map_k, p.c.cache, true, p.box_rows);
    if (rc == B2A_OK) rc = once_per_device(dev.device, 7, set_weight_smem);
    if (rc != B2A_OK) return rc;
    p.lse = a->lse;
    p.lse_head_stride = a->cu_seqlens_q == nullptr ? a->seqlen_q : a->total_q;
    p.lse_seq_stride = a->cu_seqlens_q == nullptr ? static_cast<long long>(a->heads_q) * a->seqlen_q : 0;
    p.weights = a->weights;
    p.weights_stride[0] = a->weights_stride[0];
    p.weights_stride[1] = a->weights_stride[1];
    p.scale_log2 = (a->softmax_scale > 0.f ? a->softmax_scale : 1.0f / std::sqrt(static_cast<float>(kHeadDim))) * kLog2e;
    p.status = reinterpret_cast<unsigned int*>(static_cast<WorkspaceHeader*>(a->workspace) + 1);
    p.timeout_ns = wait_timeout_ns();
    const int ctas = std::min(dev.sm_count, kFwdStatusWords);
    auto kernel = tree_weights;
    B2A_CUDA_OK(launch_early(kernel, ctas, kWeightThreads, kWeightSmemBytes, static_cast<cudaStream_t>(cuda_stream), map_q, map_k, p));
    return B2A_OK;
}

}  // extern "C"
