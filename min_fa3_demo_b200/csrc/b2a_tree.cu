// Attention of drafted tokens over a cache: O = softmax(scale Q K^T + mask) V for the few rows that a decoding step has.
//
// A row (token t, query head h) sees all slots before the drafted tokens and those drafted tokens its mask names (the
// ancestors in a tree; without a mask, those up to itself).  The query heads of a K/V head share its stream: tile rows are
// 128 / group tokens of group heads.  What an item (up to 256 rows of one K/V head against its slots) costs is its slots,
// 512 bytes each, whatever the number of rows, so the kernel is bound by memory up to some 256 rows and by the softmax beyond.
// 16 sequences of 16,384 slots, 8 K/V heads, 64 rows: 1.07 GB in 186 us, 5.8 TB/s; 16 of up to 8,000 slots in pages of 16, up
// to 128 rows: 353 MB in 81 us, 4.4 TB/s; 8 of up to 16,000 slots, 512 rows: 147 GFLOP in 168 us, 0.88 PFLOP/s.
//
// Work: all items' blocks of 128 slots in a row, dealt out in equal runs, a run a CTA (CacheWalk).  An item that crosses the
// end of a run is finished by tree_combine, in fp32 and in slot order.
//
//   warp 0-3, 4-7   softmax warpgroups, one thread a row
//   warp 8          Q K^T       warp 10   P V       warp 9   plan, loads of Q and K       warp 11   loads of V
//
// An item of more than 128 rows has two tiles that use each block in turn, as in the forward.  One of at most 128 has only
// one, and its two warpgroups take turns at the blocks: each has a running maximum, a sum and an O of its own, and they are
// added up at the end of the piece through tensor memory, which both can read.  So the chain S -> softmax -> P V of one
// block overlaps the next block's, and a warp that has only a few rows has two blocks' time for each.
//
// Tensor memory (512 columns): P of the warpgroups [0,64) [192,256), S [64,192), O [256,384) [384,512).
//
// Masked slots: a score is replaced, not added to, so NaN and infinities in K that a row does not see have no effect.  V
// rows behind the last slot are zeroed in shared memory before the product (0 * NaN is NaN), and so are values of drafted
// tokens that are not finite; those are added back to the rows that see them at the end.
#include "b2a_tree.cuh"

#include <cmath>

namespace b2a {

namespace {

constexpr int kTreeThreads = 384;
constexpr int kTreeSlots = 4;       // pieces in flight between the load warp and the others
constexpr int kTreeQkWarp = 8, kTreeLoadWarp = 9, kTreePvWarp = 10, kTreeVWarp = 11;

// kTwo: items may have two tiles.  Where none has, the second tile's room goes to another stage of K (trees of up to 32 tokens, 32
// over 8 heads, 16 sequences of up to 8,000 slots: 90 us without, 87 with, 89.5 if it goes to V).
template <bool kTwo>
struct __align__(1024) TreeShared {
    static constexpr int kTiles = kTwo ? 2 : 1, kK = kTwo ? 2 : 3, kV = 2;
    uint8_t q[kTiles][kTileBytes];
    uint8_t k[kK][kTileBytes];
    uint8_t v[kV][kTileBytes];
    uint32_t seen[2][2][kTileM][4];   // warpgroup, turn, token: one bit for each slot of the block
    float2 stat[2][kTileM];           // row maximum and sum of the two warpgroups
    TreePiece piece[kTreeSlots];
    uint64_t q_full[2], q_empty[2];
    uint64_t k_full[kK], k_empty[kK];
    uint64_t v_full[kV], v_empty[kV];
    uint64_t s_full[2], s_empty, p_full[2], pv_done[2];
    uint64_t seen_full[2];
    uint64_t both_done, both_read;
    uint64_t piece_full[kTreeSlots], piece_empty[kTreeSlots];
    // Number of the last piece, of the even ones and of the odd ones, that met a drafted value that is not finite.  Of two tiles
    // the first one's warpgroup may be a piece ahead of the other's, and no more: they take S from one place in turn.
    uint32_t not_finite[2];
    uint32_t missing;                 // the CTA has met a page that does not exist
    uint32_t tmem_base;
    uint32_t abort_flag;
};

template <bool kTwo>
constexpr size_t tree_smem_bytes() { return sizeof(TreeShared<kTwo>) + 1024; }
static_assert(tree_smem_bytes<true>() <= 227 * 1024 && tree_smem_bytes<false>() <= 227 * 1024, "shared memory of a CTA");

// Whether a block goes to warpgroup x: both tiles take every block, one tile's warpgroups take turns.
__device__ __forceinline__ bool tree_takes(bool two, int i, int x) { return two || (i & 1) == x; }

// Values of drafted tokens that are not finite, added to a row that sees them: columns [column, column + 32) of O.
// Only the sign of the weight, which is positive, matters.
__device__ __forceinline__ void tree_add_not_finite(const TreeParams& p, const TreePiece& w, int token, int column, uint32_t (&t)[32]) {
    const int from = max(0, w.j0 * kSlotBlock - w.len), to = min(w.n, (w.j0 + w.blocks) * kSlotBlock - w.len);
#pragma unroll 1
    for (int u = from; u < to; ++u) {
        const long long slot = static_cast<long long>(w.len) + u;
        if (slot >= w.slots || !tree_sees(p, w, token, u)) continue;
        int row;
        const int page = p.c.cache.page_of(w.seq, slot, &row);
        if (page < 0) continue;
        const uint4* v = reinterpret_cast<const uint4*>(p.c.cache.v + p.c.cache.at(p.c.cache.v_stride, page, row, w.head) + column);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint4 eight = v[i];
            const uint32_t words[4] = {eight.x, eight.y, eight.z, eight.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int at = i * 8 + e * 2;
                if (bf16_not_finite(words[e])) t[at] = __float_as_uint(__uint_as_float(t[at]) + __uint_as_float(words[e] << 16));
                if (bf16_not_finite(words[e] >> 16)) {
                    t[at + 1] = __float_as_uint(__uint_as_float(t[at + 1]) + __uint_as_float(words[e] & 0xFFFF0000u));
                }
            }
        }
    }
}

template <bool kTwo>
__global__ void __launch_bounds__(kTreeThreads, 1)
tree_attention(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
               const __grid_constant__ CUtensorMap map_v, const __grid_constant__ TreeParams p) {
    extern __shared__ uint8_t smem_raw[];
    using Shared = TreeShared<kTwo>;
    Shared& sh = *reinterpret_cast<Shared*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(smem_u32(&sh.q_full[i]), 1);
            mbar_init(smem_u32(&sh.q_empty[i]), 1);
            mbar_init(smem_u32(&sh.s_full[i]), 1);
            mbar_init(smem_u32(&sh.p_full[i]), kTileM);
            mbar_init(smem_u32(&sh.pv_done[i]), 1);
            mbar_init(smem_u32(&sh.seen_full[i]), kTileM);
        }
        mbar_init(smem_u32(&sh.s_empty), kTileM);
        mbar_init(smem_u32(&sh.both_done), 2 * kTileM);
        mbar_init(smem_u32(&sh.both_read), 2 * kTileM);
        for (int i = 0; i < Shared::kK; ++i) {
            mbar_init(smem_u32(&sh.k_full[i]), 1);
            mbar_init(smem_u32(&sh.k_empty[i]), 1);
        }
        for (int i = 0; i < Shared::kV; ++i) {
            mbar_init(smem_u32(&sh.v_full[i]), 1);
            mbar_init(smem_u32(&sh.v_empty[i]), 1);
        }
        for (int i = 0; i < kTreeSlots; ++i) {
            mbar_init(smem_u32(&sh.piece_full[i]), 1);
            mbar_init(smem_u32(&sh.piece_empty[i]), 3 + 8);   // MMA warps, V's load warp and softmax warps
        }
        sh.abort_flag = 0;
        sh.not_finite[0] = sh.not_finite[1] = 0;
        sh.missing = 0;
        fence_mbar_init();
        fence_proxy_async_smem();
    }
    if (warp == kTreeQkWarp) {
        tmem_alloc(smem_u32(&sh.tmem_base), 512);
        tmem_relinquish();
        tc_fence_before_sync();
    }
    let_next_kernel_start();
    wait_for_previous_kernel();
    // Each CTA clears and uses a status word of its own, and CTA 0 writes the header (as the forward does).
    if (threadIdx.x == 0) {
        p.status[blockIdx.x] = 0u;
        if (blockIdx.x == 0) reinterpret_cast<int4*>(p.status)[-1] = make_int4(-static_cast<int>(gridDim.x), 0, 0, 0);
    }
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem_base = *reinterpret_cast<volatile uint32_t*>(&sh.tmem_base);
    const WaitCtx wctx{smem_u32(&sh.abort_flag), p.status, p.timeout_ns, 1u};

    if (warp >= 8) {
        reg_dealloc<72>();
        if (warp == kTreeLoadWarp) {
            // ------------------------------------------------------------ plan and loads
            if (lane == 0) {
                tma_prefetch_desc(&map_q);
                tma_prefetch_desc(&map_k);
                tma_prefetch_desc(&map_v);
            }
            CacheWalk walk;
            walk.start(p.c, blockIdx.x, gridDim.x, lane);
            if (lane == 0) p.cuts[blockIdx.x] = tree_cut(p, walk);
            SlotLoader loader(p.box_rows);
            loader.bad = walk.bad;
            uint32_t k_it = 0, q_par = 0;
            bool ok = true;
            PH_DECL(3)   // 0 other, 1 wait for K's stage, 2 issue K
            for (uint32_t it = 0; ok; ++it) {
                const uint32_t at = it % kTreeSlots;
                ok = warp_wait(wctx, smem_u32(&sh.piece_empty[at]), ((it / kTreeSlots) & 1u) ^ 1u, 1);
                if (!ok) break;
                const TreePiece w = tree_piece(p, walk);
                if (lane == 0) {
                    sh.piece[at] = w;
                    mbar_arrive(smem_u32(&sh.piece_full[at]));
                }
                if (!w.valid) break;
                auto load_q = [&](int x) {
                    ok = warp_wait(wctx, smem_u32(&sh.q_empty[x]), ((q_par >> x) & 1u) ^ 1u, 2);
                    if (!ok) return;
                    q_par ^= 1u << x;
                    if (lane == 0) {
                        const uint32_t bar = smem_u32(&sh.q_full[x]), dst = smem_u32(&sh.q[x][0]);
                        const int row = w.q_begin + w.tok0 + x * p.tile_tokens;
                        mbar_arrive_expect_tx(bar, static_cast<uint32_t>(p.tile_tokens * p.c.group) * 256u);
                        tma_load_3d(dst, &map_q, bar, 0, w.head * p.c.group, row);
                        tma_load_3d(dst + kHalfTileBytes, &map_q, bar, 64, w.head * p.c.group, row);
                    }
                    __syncwarp();
                };
                load_q(0);
                loader.look_up(p.c.cache, w.seq, w.j0, w.slots, lane);
                for (int i = 0; i < w.blocks && ok; ++i, ++k_it) {
                    SlotLoader now = loader;
                    if (i + 1 < w.blocks) loader.look_up(p.c.cache, w.seq, w.j0 + i + 1, w.slots, lane);
                    const int boxes = now.count(w.j0 + i, w.slots);
                    const uint32_t stage = k_it % Shared::kK;
                    PH_MARK(0);
                    ok = warp_wait(wctx, smem_u32(&sh.k_empty[stage]), ((k_it / Shared::kK) & 1u) ^ 1u, 3);
                    if (!ok) break;
                    PH_MARK(1);
                    now.check(p.c.cache, boxes, lane, &sh.missing);
                    loader.bad |= now.bad;
                    now.load(&map_k, smem_u32(&sh.k[stage][0]), smem_u32(&sh.k_full[stage]), w.head, boxes, lane);
                    PH_MARK(2);
                    if (kTwo && i == 0 && w.tokens[1] > 0) load_q(1);
                }
                if (!ok) break;
                walk.advance(p.c, w.blocks);
            }
            if (__any_sync(0xFFFFFFFFu, loader.bad) && lane == 0) set_status(wctx.status_word(), kStatusBadArg, 0x3Fu << 12);
            PH_PRINT("tree load", 3);
        } else if (warp == kTreeVWarp) {
            // ------------------------------------------------------------ loads of V
            tree_load_v<kTreeSlots, Shared::kV>(p, sh, &map_v, wctx, lane);
        } else if (warp == kTreeQkWarp || warp == kTreePvWarp) {
            // ------------------------------------------------------------ MMA warps
            const bool qk = warp == kTreeQkWarp;
            constexpr uint32_t idesc_qk = make_idesc_bf16(kTileM, kTileN, 0, 0);
            constexpr uint32_t idesc_pv = make_idesc_bf16(kTileM, kHeadDim, 0, 1);
            constexpr uint32_t kStageStep = kTileBytes >> 4;
            const uint32_t q_lo0 = desc_lo_kmajor(smem_u32(&sh.q[0][0]));
            const uint32_t k_lo0 = desc_lo_kmajor(smem_u32(&sh.k[0][0]));
            const uint32_t v_lo0 = desc_lo_mnmajor(smem_u32(&sh.v[0][0]));
            uint32_t kv_it = 0, s_it = 0, par = 0;
            bool ok = true;
            PH_DECL(4)   // 0 other, 1 wait K (V), 2 wait S (P), 3 issue
            for (uint32_t it = 0; ok; ++it) {
                const uint32_t at = it % kTreeSlots;
                ok = warp_wait(wctx, smem_u32(&sh.piece_full[at]), (it / kTreeSlots) & 1u, 5);
                if (!ok) break;
                const volatile TreePiece& w = sh.piece[at];
                const int valid = __shfl_sync(0xFFFFFFFFu, w.valid, 0);
                const int blocks = __shfl_sync(0xFFFFFFFFu, w.blocks, 0);
                const bool two = kTwo && __shfl_sync(0xFFFFFFFFu, w.tokens[1], 0) > 0;
                if (lane == 0) mbar_arrive(smem_u32(&sh.piece_empty[at]));
                __syncwarp();
                if (!valid) break;
                for (int i = 0; i < blocks && ok; ++i, ++kv_it) {
                    const uint32_t stages = qk ? Shared::kK : Shared::kV, stage = kv_it % stages, phase = (kv_it / stages) & 1u;
                    PH_MARK(0);
                    if (qk) {
                        ok = mbar_wait(wctx, smem_u32(&sh.k_full[stage]), phase, 6);
                        if (!ok) break;
                        PH_MARK(1);
#pragma unroll
                        for (int x = 0; x < 2; ++x) {
                            if (!tree_takes(two, i, x)) continue;
                            const int tile = two ? x : 0;
                            if (i == 0) {
                                ok = warp_wait(wctx, smem_u32(&sh.q_full[tile]), (par >> tile) & 1u, 7);
                                if (!ok) break;
                                par ^= 1u << tile;
                            }
                            // The softmax warps have taken the S before this one out of tensor memory.
                            ok = mbar_wait(wctx, smem_u32(&sh.s_empty), (s_it & 1u) ^ 1u, 8);
                            if (!ok) break;
                            PH_MARK(2);
                            ++s_it;
                            tc_fence_after_sync();
                            umma_ss_kk_x8_w(tmem_base + kFwdColS, q_lo0 + tile * kStageStep, k_lo0 + stage * kStageStep, idesc_qk, 0u);
                            tc_commit_w(smem_u32(&sh.s_full[x]));
                            if (i == blocks - 1) tc_commit_w(smem_u32(&sh.q_empty[tile]));
                            __syncwarp();
                            PH_MARK(3);
                        }
                        tc_commit_w(smem_u32(&sh.k_empty[stage]));
                    } else {
                        ok = mbar_wait(wctx, smem_u32(&sh.v_full[stage]), phase, 9);
                        if (!ok) break;
                        PH_MARK(1);
#pragma unroll
                        for (int x = 0; x < 2; ++x) {
                            if (!tree_takes(two, i, x)) continue;
                            ok = mbar_wait(wctx, smem_u32(&sh.p_full[x]), (par >> x) & 1u, 10);
                            if (!ok) break;
                            PH_MARK(2);
                            par ^= 1u << x;
                            tc_fence_after_sync();
                            umma_ts_x8_w(tmem_base + kFwdColO + x * 128u, tmem_base + kFwdColP + x * kFwdColPStep,
                                         v_lo0 + stage * kStageStep, idesc_pv, i > (two ? 0 : x) ? 1u : 0u);
                            tc_commit_w(smem_u32(&sh.pv_done[x]));
                            __syncwarp();
                            PH_MARK(3);
                        }
                        tc_commit_w(smem_u32(&sh.v_empty[stage]));
                    }
                }
            }
            PH_PRINT("tree mma", 4);
        }
    } else {
        // ---------------------------------------------------------------- softmax warpgroups
        reg_alloc<216>();
        const int x = warp >> 2;
        const int quarter = warp & 3;
        const int r = quarter * 32 + lane;
        const uint32_t lane_base = static_cast<uint32_t>(quarter * 32) << 16;
        const uint32_t s_tmem = tmem_base + lane_base + kFwdColS;
        const uint32_t p_tmem = tmem_base + lane_base + kFwdColP + static_cast<uint32_t>(x) * kFwdColPStep;
        const uint32_t o_tmem = tmem_base + lane_base + kFwdColO;
        const float sl2 = p.scale_log2;
        const int row_token = r / p.c.group;           // of the tile
        const int row_head = r - row_token * p.c.group;
        uint32_t s_cnt = 0, pv_cnt = 0, seen_cnt = 0, both_cnt = 0, kv_base = 0;
        bool ok = true;
        PH_DECL(6)   // 0 other, 1 which slots are seen, 2 wait S, 3 take S, 4 V rows and mask, 5 softmax

        for (uint32_t it = 0; ok; ++it) {
            const uint32_t at = it % kTreeSlots;
            ok = warp_wait(wctx, smem_u32(&sh.piece_full[at]), (it / kTreeSlots) & 1u, 11);
            if (!ok) break;
            const TreePiece& w = sh.piece[at];
            auto release = [&]() {
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&sh.piece_empty[at]));
            };
            if (!w.valid) break;
            const bool two = kTwo && w.tokens[1] > 0;
            const int tile = two ? x : 0;
            const int tokens = w.tokens[tile];
            const int rows = tokens * p.c.group;
            const bool row_valid = r < rows;
            const bool active = quarter * 32 < rows;      // the warp has a row at all
            const int token = w.tok0 + tile * p.tile_tokens + row_token;
            const bool masked = p.c.mask != nullptr;

            float m_used = -INFINITY;   // running reference maximum (raw score units)
            float l = 0.f;              // running row sum relative to m_used
            const int first = two ? 0 : x, step = two ? 1 : 2;
            for (int i = first; i < w.blocks; i += step) {
                const int base = (w.j0 + i) * kSlotBlock;
                const bool tail = base + kSlotBlock > w.len;   // drafted tokens, or no slots any more
                uint32_t* seen = nullptr;
                PH_MARK(0);
                if (tail && masked) {
                    // Which slots of the block each token sees: a warp's lanes are 32 slots.  Eight tokens' bytes at a time.
                    const int slot = base + quarter * 32 + lane, u = slot - w.len;
                    const bool ask = slot < w.slots && u >= 0 && u < w.n, always = u < 0 && slot < w.slots;
                    const unsigned char* byte = tree_mask_row(p, w, w.tok0 + tile * p.tile_tokens) + (ask ? u : 0);
                    seen = &sh.seen[x][seen_cnt & 1u][0][0];
                    for (int t0 = 0; t0 < tokens; t0 += 8) {
                        uint32_t yes[8];
#pragma unroll
                        for (int t = 0; t < 8; ++t) {
                            yes[t] = always ? 1u : 0u;
                            if (ask && t0 + t < tokens) yes[t] = byte[(t0 + t) * p.c.mask_stride[1]];
                        }
#pragma unroll
                        for (int t = 0; t < 8; ++t) {
                            const uint32_t word = __ballot_sync(0xFFFFFFFFu, yes[t] != 0u);
                            if (lane == 0 && t0 + t < tokens) seen[(t0 + t) * 4 + quarter] = word;
                        }
                    }
                    __syncwarp();
                    mbar_arrive(smem_u32(&sh.seen_full[x]));
                }
                PH_MARK(1);
                ok = mbar_wait(wctx, smem_u32(&sh.s_full[x]), s_cnt & 1u, 12);
                if (!ok) break;
                PH_MARK(2);
                ++s_cnt;
                tc_fence_after_sync();
                float s[kTileN];
                if (active) {
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        uint32_t t[32];
                        tmem_ld_x32(s_tmem + c * 32, t);
#pragma unroll
                        for (int e = 0; e < 32; ++e) s[c * 32 + e] = __uint_as_float(t[e]);
                    }
                    tmem_wait_ld();
                }
                tc_fence_before_sync();
                mbar_arrive(smem_u32(&sh.s_empty));
                PH_MARK(3);

                const bool begins = i == first;
                bool pv_pending = !begins;
                auto wait_pv = [&]() -> bool {
                    if (!mbar_wait(wctx, smem_u32(&sh.pv_done[x]), pv_cnt & 1u, 15)) return false;
                    ++pv_cnt;
                    tc_fence_after_sync();
                    pv_pending = false;
                    return true;
                };

                if (tail) {
                    if (masked) {
                        ok = warp_wait(wctx, smem_u32(&sh.seen_full[x]), seen_cnt & 1u, 13);
                        if (!ok) break;
                        ++seen_cnt;
                    }
                    // V row r of the block (whichever warpgroup's product with it comes first): behind the last slot
                    // zeros, and of drafted tokens no value that is not finite.
                    const int slot = base + r;
                    const bool look = slot >= w.len && slot < w.slots && (w.n > 1 || masked);
                    if (!two || x == 0) {
                        // A barrier tells the last phase from the one before it, no more: the V that lay in this stage two
                        // blocks ago has to have come, which the product with it proves.
                        if (pv_pending) {
                            ok = wait_pv();
                            if (!ok) break;
                        }
                        const uint32_t stage = (kv_base + i) % Shared::kV;
                        ok = warp_wait(wctx, smem_u32(&sh.v_full[stage]), ((kv_base + i) / Shared::kV) & 1u, 14);
                        if (!ok) break;
                        if (slot >= w.slots || look) {
                            if (tree_clean_row(&sh.v[stage][r * 128], r, slot >= w.slots)) {
                                *reinterpret_cast<volatile uint32_t*>(&sh.not_finite[it & 1u]) = it + 1;
                            }
                        }
                        fence_proxy_async_smem();
                    }
                }
                if (active && tail) {
                    // One bit per visible slot of 32.
                    const int lim = min(w.slots, w.len + token + 1) - base;
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        uint32_t bits;
                        if (masked) {
                            bits = seen[min(row_token, tokens - 1) * 4 + c];
                        } else {
                            const int vis = min(max(lim - c * 32, 0), 32);
                            bits = vis == 32 ? 0xFFFFFFFFu : (1u << vis) - 1u;
                        }
#pragma unroll
                        for (int e = 0; e < 32; ++e) {
                            if (!((bits >> e) & 1u)) s[c * 32 + e] = -INFINITY;
                        }
                    }
                }
                // Asked by the whole warp: the flag may go up, for a block still to come, between two lanes' looks.
                if (__builtin_expect(__any_sync(0xFFFFFFFFu, *reinterpret_cast<volatile uint32_t*>(&sh.missing) != 0u), 0)) {
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        const uint32_t bits = __ballot_sync(0xFFFFFFFFu, p.c.cache.has(w.seq, base + c * 32 + lane));
#pragma unroll
                        for (int e = 0; e < 32; ++e) {
                            if (!((bits >> e) & 1u)) s[c * 32 + e] = -INFINITY;
                        }
                    }
                }

                PH_MARK(4);
                if (!active) {
                    // None of the warp's rows exists; it keeps step, and its P and O are never looked at.
                    if (pv_pending) {
                        ok = wait_pv();
                        if (!ok) break;
                    }
                    mbar_arrive(smem_u32(&sh.p_full[x]));
                    continue;
                }
                float bm;
                {
                    float m[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) m[e] = s[e];
#pragma unroll
                    for (int e = 8; e < kTileN; ++e) m[e & 7] = fmaxf(m[e & 7], s[e]);
                    bm = fmaxf(max3(max3(m[0], m[1], m[2]), m[3], m[4]), max3(m[5], m[6], m[7]));
                }
                const float m_new = fmaxf(m_used, bm);
                if (begins) {
                    m_used = m_new;
                } else if (__any_sync(0xFFFFFFFFu, row_valid && (m_new - m_used) * sl2 > kRescaleThreshold)) {
                    // O is scaled only when the maximum has moved by a factor of 2^8: the division at the end uses the same
                    // one.  Rows of the tile that do not exist have no say: what lies there differs from call to call.
                    const float factor = m_new == -INFINITY ? 1.f : fast_exp2((m_used - m_new) * sl2);
                    l *= factor;
                    m_used = m_new;
                    if (pv_pending) {         // a block that ends a sequence has waited already
                        ok = wait_pv();
                        if (!ok) break;
                    }
#pragma unroll 1
                    for (int c = 0; c < 4; ++c) {
                        uint32_t t[32];
                        tmem_ld_x32(o_tmem + x * 128 + c * 32, t);
                        tmem_wait_ld();
#pragma unroll
                        for (int e = 0; e < 32; ++e) t[e] = __float_as_uint(__uint_as_float(t[e]) * factor);
                        tmem_st_x32(o_tmem + x * 128 + c * 32, t);
                    }
                }
                // P stays below 1 however far the maximum has moved since, so that no product with a finite V overflows.
                const float neg_m = m_used == -INFINITY ? 0.f : -m_used * sl2 - kRescaleThreshold;
                const float2 sl2v = make_float2(sl2, sl2), negv = make_float2(neg_m, neg_m);
                float2 acc0 = make_float2(0.f, 0.f), acc1 = make_float2(0.f, 0.f);
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    uint32_t t[32];
#pragma unroll
                    for (int e = 0; e < 32; e += 2) {
                        const float2 x0 = fma2(make_float2(s[c * 64 + 2 * e], s[c * 64 + 2 * e + 1]), sl2v, negv);
                        const float2 x1 = fma2(make_float2(s[c * 64 + 2 * e + 2], s[c * 64 + 2 * e + 3]), sl2v, negv);
                        const float2 p0 = make_float2(fast_exp2(x0.x), fast_exp2(x0.y));
                        const float2 p1 = make_float2(fast_exp2(x1.x), fast_exp2(x1.y));
                        acc0 = add2(acc0, p0);
                        acc1 = add2(acc1, p1);
                        // P is rounded to bf16 for the product: 2^-9 of a term on average, as much as the rounding of out.
                        t[e] = pack_bf16x2(p0.x, p0.y);
                        t[e + 1] = pack_bf16x2(p1.x, p1.y);
                    }
                    if (c == 0 && pv_pending) {
                        ok = wait_pv();
                        if (!ok) break;
                    }
                    tmem_st_x32(p_tmem + c * 32, t);
                }
                if (!ok) break;
                l += (acc0.x + acc0.y) + (acc1.x + acc1.y);
                tmem_wait_st();
                tc_fence_before_sync();
                mbar_arrive(smem_u32(&sh.p_full[x]));
                PH_MARK(5);
            }
            if (!ok) break;
            kv_base += w.blocks;
            if (w.blocks > first) {
                ok = mbar_wait(wctx, smem_u32(&sh.pv_done[x]), pv_cnt & 1u, 15);
                if (!ok) break;
                ++pv_cnt;
                tc_fence_after_sync();
            }

            // One tile: the two warpgroups' parts, O = a0 O0 + a1 O1; each does half of the columns.
            float a0 = 1.f, a1 = 0.f;
            if (!two) {
                sh.stat[x][r] = make_float2(m_used, l);
                tc_fence_before_sync();
                mbar_arrive(smem_u32(&sh.both_done));
                ok = warp_wait(wctx, smem_u32(&sh.both_done), both_cnt & 1u, 16);
                if (!ok) break;
                tc_fence_after_sync();
                const float2 s0 = sh.stat[0][r], s1 = sh.stat[1][r];
                m_used = fmaxf(s0.x, s1.x);
                a0 = s0.x == m_used ? 1.f : fast_exp2((s0.x - m_used) * sl2);
                a1 = s1.x == m_used ? 1.f : fast_exp2((s1.x - m_used) * sl2);
                l = s0.y * a0 + s1.y * a1;
                if (w.blocks == 1) a1 = 0.f;
            }
            if (active) {
                const bool not_finite = *reinterpret_cast<volatile uint32_t*>(&sh.not_finite[it & 1u]) == it + 1;
                // A sum of 0: the row sees nothing (or only what is -inf).  NaN stays NaN.
                const float inv = l == 0.f ? 0.f : 1.f / l;
                const bool whole = w.part < 0;
                if (row_valid && (two || x == 0)) {
                    if (whole) {
                        const float lse = l == 0.f ? -INFINITY : (m_used * sl2 + kRescaleThreshold + fast_log2(l)) * kLn2;
                        const int head = w.head * p.c.group + row_head;
                        p.lse[w.seq * p.lse_seq_stride + head * p.lse_head_stride +
                              (p.c.cu_seqlens_q == nullptr ? token : w.q_begin + token)] = lse;
                    } else {
                        p.part_stat[(static_cast<long long>(w.part) * Shared::kTiles + tile) * p.part_rows + r] = make_float2(m_used, l);
                    }
                }
                __nv_bfloat16* o_row = p.out + ((static_cast<long long>(w.q_begin) + token) * p.c.heads_q +
                                                w.head * p.c.group + row_head) * kHeadDim;
                float4* part = p.part_o + (static_cast<long long>(w.part) * Shared::kTiles + tile) * 32 * p.part_rows + r;
                const int from = two ? 0 : 2 * x, to = two ? 4 : 2 * x + 2;
#pragma unroll 1
                for (int c = from; c < to; ++c) {
                    uint32_t t[32];
                    if (two) {
                        tmem_ld_x32(o_tmem + x * 128 + c * 32, t);
                        tmem_wait_ld();
                    } else {
                        tmem_ld_x32(o_tmem + c * 32, t);
                        tmem_wait_ld();
                        if (w.blocks > 1) {
                            uint32_t t1[32];
                            tmem_ld_x32(o_tmem + 128 + c * 32, t1);
                            tmem_wait_ld();
#pragma unroll
                            for (int e = 0; e < 32; ++e) {
                                t[e] = __float_as_uint(fmaf(__uint_as_float(t1[e]), a1, __uint_as_float(t[e]) * a0));
                            }
                        }
                    }
                    if (!row_valid) continue;
                    if (not_finite) tree_add_not_finite(p, w, token, c * 32, t);
                    if (whole) {
                        uint4* dst = reinterpret_cast<uint4*>(o_row + c * 32);
#pragma unroll
                        for (int v = 0; v < 4; ++v) {
                            uint32_t o[4];
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                o[e] = pack_bf16x2(__uint_as_float(t[v * 8 + 2 * e]) * inv, __uint_as_float(t[v * 8 + 2 * e + 1]) * inv);
                            }
                            dst[v] = make_uint4(o[0], o[1], o[2], o[3]);
                        }
                    } else {
#pragma unroll
                        for (int v = 0; v < 8; ++v) {
                            part[(c * 8 + v) * p.part_rows] = make_float4(__uint_as_float(t[4 * v]), __uint_as_float(t[4 * v + 1]),
                                                                          __uint_as_float(t[4 * v + 2]), __uint_as_float(t[4 * v + 3]));
                        }
                    }
                }
                __syncwarp();
            }
            tc_fence_before_sync();
            if (!two) {
                // Neither warpgroup's next product may overwrite an O that the other still reads.
                mbar_arrive(smem_u32(&sh.both_read));
                ok = warp_wait(wctx, smem_u32(&sh.both_read), both_cnt & 1u, 17);
                ++both_cnt;
                if (!ok) break;
            }
            release();
        }
        PH_PRINT("tree softmax", 6);
    }

    // Common exit: every role arrives here (normally or after an abort).
    tc_fence_before_sync();
    __syncthreads();
    if (warp == kTreeQkWarp) {
        tc_fence_after_sync();
        tmem_dealloc(tmem_base, 512);
    }
}

// ---------------------------------------------------------------------------------------
// Adds up the pieces of the items that ends of runs cut, in slot order: O = sum_i w_i O_i / sum_i w_i l_i with
// w_i = 2^(m_i - max m).  CTA (i, strip) looks after the item that run i + 1 begins inside of, if it is the first to do so,
// and 32 rows of it.
// ---------------------------------------------------------------------------------------
constexpr int kTreeStrip = 32;

__global__ void __launch_bounds__(256)
tree_combine(const __grid_constant__ TreeParams p) {
    constexpr int kPitch = kHeadDim + 4;    // bf16; keeps the 8-byte column stores of 16 rows on distinct banks
    __shared__ __align__(8) __nv_bfloat16 out[kTreeStrip * kPitch];
    let_next_kernel_start();
    wait_for_previous_kernel();
    const int cta = blockIdx.x + 1;
    const int strips = (p.part_rows + kTreeStrip - 1) / kTreeStrip;
    const int tile = blockIdx.y / strips;
    const int row0 = blockIdx.y % strips * kTreeStrip;
    const TreeCut cut = p.cuts[cta];
    if (cut.run == 0 || cut.first < static_cast<long long>(cta - 1) * cut.run) return;   // none, or not the first run inside
    const int tok0 = cut.tok0 + tile * p.tile_tokens;
    const int rows = min(min(p.tile_tokens, cut.n - tok0) * p.c.group - row0, kTreeStrip);
    if (rows <= 0) return;
    const int pieces = static_cast<int>((cut.last - 1) / cut.run) - (cta - 1) + 1;
    // The first piece ends run cta - 1 (and may begin it); the others begin their runs.
    auto part_of = [&](int i) -> long long {
        const int second = i == 0 && cut.first > static_cast<long long>(cta - 1) * cut.run;
        return (2ll * (cta - 1 + i) + second) * p.part_tiles + tile;
    };
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    float m = -INFINITY, l = 0.f, norm = 0.f;
    if (lane < rows) {
#pragma unroll 4
        for (int i = 0; i < pieces; ++i) m = fmaxf(m, p.part_stat[part_of(i) * p.part_rows + row0 + lane].x);
    }
    // Each warp finds the row's weights by itself.
    auto weight_of = [&](const float2& st) { return st.x == m ? 1.f : fast_exp2((st.x - m) * p.scale_log2); };
    if (lane < rows) {
#pragma unroll 4
        for (int i = 0; i < pieces; ++i) {
            const float2 st = p.part_stat[part_of(i) * p.part_rows + row0 + lane];
            l = fmaf(st.y, weight_of(st), l);
        }
        norm = l == 0.f ? 0.f : 1.f / l;
        if (warp == 0) {
            const int r = row0 + lane, token = tok0 + r / p.c.group;
            p.lse[cut.seq * p.lse_seq_stride + (cut.head * p.c.group + r % p.c.group) * p.lse_head_stride +
                  (p.c.cu_seqlens_q == nullptr ? token : cut.q_begin + token)] =
                l == 0.f ? -INFINITY : (m * p.scale_log2 + kRescaleThreshold + fast_log2(l)) * kLn2;
        }
    }
    // Lane = row, four of the 32 column quads a warp.
    if (lane < rows) {
        float4 acc[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) acc[u] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 2
        for (int i = 0; i < pieces; ++i) {
            const float f = weight_of(p.part_stat[part_of(i) * p.part_rows + row0 + lane]) * norm;
            const float4* o = p.part_o + (part_of(i) * 32 + warp * 4) * p.part_rows + row0 + lane;
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const float4 v = __ldcs(o + u * p.part_rows);
                acc[u].x = fmaf(v.x, f, acc[u].x);
                acc[u].y = fmaf(v.y, f, acc[u].y);
                acc[u].z = fmaf(v.z, f, acc[u].z);
                acc[u].w = fmaf(v.w, f, acc[u].w);
            }
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            *reinterpret_cast<uint2*>(&out[lane * kPitch + (warp * 4 + u) * 4]) =
                make_uint2(pack_bf16x2(acc[u].x, acc[u].y), pack_bf16x2(acc[u].z, acc[u].w));
        }
    }
    __syncthreads();
    // A warp writes one whole 256-byte row per instruction.
    for (int rr = warp; rr < rows; rr += 8) {
        const int r = row0 + rr;
        const long long to = (static_cast<long long>(cut.q_begin) + tok0 + r / p.c.group) * p.c.heads_q +
                             cut.head * p.c.group + r % p.c.group;
        *reinterpret_cast<uint2*>(p.out + to * kHeadDim + lane * 4) = *reinterpret_cast<const uint2*>(&out[rr * kPitch + lane * 4]);
    }
}

template <bool kTwo>
int set_tree_smem() {
    B2A_CUDA_OK(cudaFuncSetAttribute(tree_attention<kTwo>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     static_cast<int>(tree_smem_bytes<kTwo>())));
    return B2A_OK;
}

struct TreeLayout {
    int ctas, tile_tokens, tiles, rows;   // rows of a tile; few rows: of an item, which is one tile
    bool few;
    size_t o, scratch;                    // of the pieces' results behind their sums, and of both
};

// What is kept after a call: header, status words and cuts.
constexpr size_t kTreeCutsAt = align_up(sizeof(WorkspaceHeader) + kFwdStatusWords * sizeof(unsigned int), 256);
constexpr size_t kTreeKept = align_up(kTreeCutsAt + kTreeMaxCtas * sizeof(TreeCut), 256);

TreeLayout tree_layout(int seqlen_q, int group, int sms) {
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

}  // namespace

}  // namespace b2a

extern "C" {

size_t b2a_tree_fwd_workspace_bytes(int32_t seqlen_q, int32_t heads_q, int32_t heads_k) {
    using namespace b2a;
    DeviceInfo dev{};
    if (seqlen_q < 1 || heads_k < 1 || heads_q < heads_k || heads_q % heads_k != 0 || heads_q / heads_k > kTileM ||
        current_device_info(&dev) != B2A_OK) {
        return 0;   // b2a_tree_fwd reports what is wrong
    }
    return kTreeKept + tree_layout(seqlen_q, heads_q / heads_k, dev.sm_count).scratch;
}

size_t b2a_tree_fwd_kept_workspace_bytes(void) { return b2a::kTreeKept; }

int b2a_tree_fwd(const b2a_tree_args* a, void* cuda_stream) {
    using namespace b2a;
    B2A_REQUIRE(a != nullptr, "args must not be NULL");
    B2A_REQUIRE(a->workspace != nullptr && (reinterpret_cast<uintptr_t>(a->workspace) & 0xF) == 0,
                "workspace must be a 16-byte aligned device pointer");
    const size_t behind = a->workspace_bytes > kTreeKept ? a->workspace_bytes - kTreeKept : 0;
    return b2a_tree_fwd_with_scratch(a, static_cast<uint8_t*>(a->workspace) + kTreeKept, behind, cuda_stream);
}

int b2a_tree_fwd_with_scratch(const b2a_tree_args* a, void* scratch, size_t scratch_bytes, void* cuda_stream) {
    using namespace b2a;
    B2A_REQUIRE(a != nullptr, "args must not be NULL");
    TreeParams p{};
    int rc = make_cache_queries(*a, true, &p.c);
    if (rc != B2A_OK) return rc;
    B2A_REQUIRE(a->out != nullptr && (reinterpret_cast<uintptr_t>(a->out) & 0xF) == 0, "out must be a 16-byte aligned device pointer");
    B2A_REQUIRE(a->workspace != nullptr && (reinterpret_cast<uintptr_t>(a->workspace) & 0xF) == 0,
                "workspace must be a 16-byte aligned device pointer");
    B2A_REQUIRE(scratch != nullptr && (reinterpret_cast<uintptr_t>(scratch) & 0xF) == 0,
                "scratch must be a 16-byte aligned device pointer");
    DeviceInfo dev{};
    rc = current_device_info(&dev);
    if (rc != B2A_OK) return rc;
    const TreeLayout t = tree_layout(a->seqlen_q, p.c.group, dev.sm_count);
    if (a->workspace_bytes < kTreeKept || scratch_bytes < t.scratch) {
        return fail(B2A_ERR_WORKSPACE_TOO_SMALL, "workspace has %zu bytes and %zu for the pieces, need %zu and %zu", a->workspace_bytes,
                    scratch_bytes, kTreeKept, t.scratch);
    }
    p.c.item_tokens = t.few ? t.tile_tokens : 2 * t.tile_tokens;
    p.c.min_run = 2;     // blocks (1, 2, 4 of them: a tree of 8 tokens over 700 slots, 32 heads over 8, 15.5, 14.9, 15.9 us)
    // A few blocks' time goes into an item's masks, sums and results, so that runs of equal numbers of blocks differ in how many
    // items end in them.  0, 2, 4, 6, 8 blocks (us): one token, 16 sequences of up to 8,001 slots, 58.5, 57.5, 57.2, 57.0, 57.3;
    // trees of up to 32 tokens 87.2, 83.5, 81.2, 80.6, 80.5; of 64, 64 over 8 heads, 179, 175, 172, 168, 173.
    p.c.item_extra = t.few ? 4 : 6;
    p.box_rows = slot_box_rows(p.c.cache);
    CUtensorMap map_q, map_k, map_v;
    const uint64_t q_sizes[2] = {static_cast<uint64_t>(a->total_q), static_cast<uint64_t>(a->heads_q)};
    rc = make_strided_map(&map_q, a->q, 3, q_sizes, a->q_stride, static_cast<uint32_t>(p.c.group), static_cast<uint32_t>(t.tile_tokens));
    if (rc == B2A_OK) rc = make_slot_map(&map_k, p.c.cache, true, p.box_rows);
    if (rc == B2A_OK) rc = make_slot_map(&map_v, p.c.cache, false, p.box_rows);
    if (rc == B2A_OK && t.tiles == 2) rc = once_per_device(dev.device, 6, set_tree_smem<true>);
    if (rc == B2A_OK && t.tiles == 1 && !t.few) rc = once_per_device(dev.device, 12, set_tree_smem<false>);
    if (rc != B2A_OK) return rc;

    uint8_t* ws = static_cast<uint8_t*>(a->workspace);
    p.out = static_cast<__nv_bfloat16*>(a->out);
    p.lse = a->lse;
    p.lse_head_stride = a->cu_seqlens_q == nullptr ? a->seqlen_q : a->total_q;
    p.lse_seq_stride = a->cu_seqlens_q == nullptr ? static_cast<long long>(a->heads_q) * a->seqlen_q : 0;
    p.tile_tokens = t.tile_tokens;
    p.scale_log2 = (a->softmax_scale > 0.f ? a->softmax_scale : 1.0f / std::sqrt(static_cast<float>(kHeadDim))) * kLog2e;
    p.status = reinterpret_cast<unsigned int*>(reinterpret_cast<WorkspaceHeader*>(ws) + 1);
    p.timeout_ns = wait_timeout_ns();
    p.cuts = reinterpret_cast<TreeCut*>(ws + kTreeCutsAt);
    p.part_stat = reinterpret_cast<float2*>(scratch);
    p.part_o = reinterpret_cast<float4*>(static_cast<uint8_t*>(scratch) + t.o);
    p.part_tiles = t.tiles;
    p.part_rows = t.rows;

    cudaStream_t stream = static_cast<cudaStream_t>(cuda_stream);
    if (t.few) return launch_tree_few(map_q, map_k, map_v, p, t.ctas, dev, stream);
    auto attention = t.tiles == 2 ? tree_attention<true> : tree_attention<false>;
    const size_t smem = t.tiles == 2 ? tree_smem_bytes<true>() : tree_smem_bytes<false>();
    auto combine = tree_combine;
    B2A_CUDA_OK(launch_early(attention, t.ctas, kTreeThreads, smem, stream, map_q, map_k, map_v, p));
    const int strips = t.tiles * ((t.rows + kTreeStrip - 1) / kTreeStrip);
    if (t.ctas > 1) B2A_CUDA_OK(launch_early(combine, dim3(t.ctas - 1, strips), 256, 0, stream, p));
    return B2A_OK;
}

}  // extern "C"
