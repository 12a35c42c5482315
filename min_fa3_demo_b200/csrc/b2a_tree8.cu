// Attention of drafted tokens, or of a prompt's next chunk, over a cache in 8 bits: O = softmax(scale Q K^T + mask) V.  Rows, items,
// their order, masks and tensor memory are those of b2a_tree.cu, the numbers those of b2a_cache8.cuh.
//
// Two tiles of 128 rows use each block in turn, as there: a thread takes its row's 128 scores at once, so that the S which both use is
// free again, and one warp turns V to f16 in the time that the two tiles' softmax needs.  (b2a_tree8_one.cu is for calls whose
// items have one tile.)  Q is turned into its two parts by the softmax warps, two rows a warp at a time, when a piece begins; a row's scale
// and K's meet in the factor of a score.
//
// Bound by what an SM does for a score rather than by memory: two products of K, one of V in f16, an exponential, and the sum with V's
// scale.  8 sequences of 64 drafted tokens, 64 heads over 8, up to 16,000 slots: 222 to 242 us (bf16: 189 to 208), up to 735 TFLOP/s; two
// chunks of 1,000 tokens, 32 heads over 8, behind up to 8,000: 338 us, 717 TFLOP/s.  No unit is near its limit (tensor pipe 38 %, special
// functions 39 %, issue slots 34 %; over bf16 49, 49, 32), and what the difference waits for is not found: that kernel uses one S for
// two tiles as well, and executes 57 million instructions for 81.
//
//   warp 0-3, 4-7   Q in two parts, then softmax, one thread a row
//   warp 8          Q K^T       warp 10   P V       warp 9   plan, loads of K, V and scales       warp 11   V to f16
#include "b2a_cache8.cuh"

#include <cfloat>
#include <cmath>

namespace b2a {

namespace {

constexpr int kTree8Threads = 384;
constexpr int kTree8Slots = 4;       // pieces in flight between the load warp and the others
constexpr int kTree8QkWarp = 8, kTree8LoadWarp = 9, kTree8PvWarp = 10, kTree8ConvertWarp = 11;

struct __align__(1024) Tree8Shared {
    static constexpr int kTiles = 2, kK = 3, kV = 2, kV16 = 2;
    uint8_t q[kTiles][2][kTile8Bytes];      // both parts
    uint8_t k[kK][kTile8Bytes];
    uint8_t v[kV][kTile8Bytes];
    uint8_t v16[kV16][kTileBytes];          // V in f16, two halves of 64 columns
    float q_scale[kTiles][kTileM];          // what a row of Q is multiplied by
    ScaleRing<1> scales;
    uint32_t seen[2][2][kTileM][4];   // warpgroup, turn, token: one bit for each slot of the block
    float2 stat[2][kTileM];           // row maximum and sum of the two warpgroups
    TreePiece piece[kTree8Slots];
    uint64_t q_full[2], q_empty[2];
    uint64_t k_full[kK], k_empty[kK];
    uint64_t v_full[kV], v_empty[kV];
    uint64_t v16_full[kV16], v16_empty[kV16];
    uint64_t s_full[2], s_empty, p_full[2], pv_done[2];
    uint64_t seen_full[2];
    uint64_t both_done, both_read;
    uint64_t piece_full[kTree8Slots], piece_empty[kTree8Slots];
    uint32_t not_finite[kTree8Slots]; // number, plus one, of the piece that met a drafted value that is NaN
    uint32_t missing;                 // the CTA has met a page that does not exist
    uint32_t tmem_base;
    uint32_t abort_flag;
};

constexpr size_t kTree8SmemBytes = sizeof(Tree8Shared) + 1024;
static_assert(kTree8SmemBytes <= 227 * 1024, "shared memory of a CTA");

// Whether a block goes to warpgroup x: both tiles take every block, one tile's warpgroups take turns.
__device__ __forceinline__ bool tree8_takes(bool two, int i, int x) { return two || (i & 1) == x; }

__global__ void __launch_bounds__(kTree8Threads, 1)
tree8_attention(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                const __grid_constant__ Tree8Params p8) {
    const TreeParams& p = p8.t;
    extern __shared__ uint8_t smem_raw[];
    using Shared = Tree8Shared;
    Shared& sh = *reinterpret_cast<Shared*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(smem_u32(&sh.q_full[i]), 8);             // warps; of two tiles each has four, which count twice
            mbar_init(smem_u32(&sh.q_empty[i]), 1);
            mbar_init(smem_u32(&sh.s_full[i]), 1);
            mbar_init(smem_u32(&sh.p_full[i]), kTileM);
            mbar_init(smem_u32(&sh.pv_done[i]), 1);
            mbar_init(smem_u32(&sh.seen_full[i]), kTileM);
        }
        mbar_init(smem_u32(&sh.s_empty), kTileM);
        sh.scales.init(8);                                  // warps, as for Q
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
        for (int i = 0; i < Shared::kV16; ++i) {
            mbar_init(smem_u32(&sh.v16_full[i]), 1);
            mbar_init(smem_u32(&sh.v16_empty[i]), 1);
        }
        for (int i = 0; i < kTree8Slots; ++i) {
            mbar_init(smem_u32(&sh.piece_full[i]), 1);
            mbar_init(smem_u32(&sh.piece_empty[i]), 3 + 8);   // MMA warps, converting and softmax warps
            sh.not_finite[i] = 0;
        }
        sh.abort_flag = 0;
        sh.missing = 0;
        fence_mbar_init();
        fence_proxy_async_smem();
    }
    if (warp == kTree8QkWarp) {
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
        if (warp == kTree8LoadWarp) {
            // ------------------------------------------------------------ plan, loads
            if (lane == 0) {
                tma_prefetch_desc(&map_k);
                tma_prefetch_desc(&map_v);
            }
            CacheWalk walk;
            walk.start(p.c, blockIdx.x, gridDim.x, lane);
            if (lane == 0) p.cuts[blockIdx.x] = tree_cut(p, walk);
            SlotLoader loader(p.box_rows);
            loader.bad = walk.bad;
            uint32_t k_it = 0;
            bool ok = true;
            PH_DECL(3)   // 0 other, 1 wait for K's stage, 2 issue K
            for (uint32_t it = 0; ok; ++it) {
                const uint32_t at = it % kTree8Slots;
                ok = warp_wait8(wctx, smem_u32(&sh.piece_empty[at]), ((it / kTree8Slots) & 1u) ^ 1u, 1);
                if (!ok) break;
                const TreePiece w = tree_piece(p, walk);
                if (lane == 0) {
                    sh.piece[at] = w;
                    mbar_arrive(smem_u32(&sh.piece_full[at]));
                }
                if (!w.valid) break;
                loader.look_up(p.c.cache, w.seq, w.j0, w.slots, lane);
                for (int i = 0; i < w.blocks && ok; ++i, ++k_it) {
                    SlotLoader now = loader;
                    if (i + 1 < w.blocks) loader.look_up(p.c.cache, w.seq, w.j0 + i + 1, w.slots, lane);
                    const int boxes = now.count(w.j0 + i, w.slots);
                    const uint32_t stage = k_it % Shared::kK;
                    PH_MARK(0);
                    ok = warp_wait8(wctx, smem_u32(&sh.k_empty[stage]), ((k_it / Shared::kK) & 1u) ^ 1u, 3);
                    if (!ok) break;
                    PH_MARK(1);
                    now.check(p.c.cache, boxes, lane, &sh.missing);
                    loader.bad |= now.bad;
                    ok = sh.scales.load(wctx, k_it, p.c.cache, p8.scales, now, w.j0 + i, w.slots, w.head, lane);
                    if (!ok) break;
                    load_slots8(now, &map_k, smem_u32(&sh.k[stage][0]), smem_u32(&sh.k_full[stage]), w.head, boxes, lane);
                    const uint32_t v_stage = k_it % Shared::kV;
                    ok = warp_wait8(wctx, smem_u32(&sh.v_empty[v_stage]), ((k_it / Shared::kV) & 1u) ^ 1u, 18);
                    if (!ok) break;
                    load_slots8(now, &map_v, smem_u32(&sh.v[v_stage][0]), smem_u32(&sh.v_full[v_stage]), w.head, boxes, lane);
                    PH_MARK(2);
                }
                if (!ok) break;
                walk.advance(p.c, w.blocks);
            }
            if (__any_sync(0xFFFFFFFFu, loader.bad) && lane == 0) set_status(wctx.status_word(), kStatusBadArg, 0x3Fu << 12);
            PH_PRINT("tree8 load", 3);
        } else if (warp == kTree8ConvertWarp) {
            tree8_convert_v<1, kTree8Slots, Shared::kV, Shared::kV16>(p, sh, wctx, lane, [](const TreePiece&, uint32_t) { return true; });
        } else if (warp == kTree8QkWarp || warp == kTree8PvWarp) {
            // ------------------------------------------------------------ MMA warps
            const bool qk = warp == kTree8QkWarp;
            constexpr uint32_t idesc_qk = make_idesc_first(kTileM, kTileN, 0, 0), idesc_pv = make_idesc_first(kTileM, kHeadDim, 0, 1);
            constexpr uint32_t kStageStep = kTile8Bytes >> 4;
            const uint32_t q_lo0 = desc_lo_kmajor(smem_u32(&sh.q[0][0][0]));
            const uint32_t k_lo0 = desc_lo_kmajor(smem_u32(&sh.k[0][0]));
            const uint32_t v_lo0 = desc_lo_mnmajor(smem_u32(&sh.v16[0][0]));
            uint32_t kv_it = 0, s_it = 0, par = 0;
            bool ok = true;
            PH_DECL(4)   // 0 other, 1 wait K (V), 2 wait S (P), 3 issue
            for (uint32_t it = 0; ok; ++it) {
                const uint32_t at = it % kTree8Slots;
                ok = warp_wait8(wctx, smem_u32(&sh.piece_full[at]), (it / kTree8Slots) & 1u, 5);
                if (!ok) break;
                const volatile TreePiece& w = sh.piece[at];
                const int valid = __shfl_sync(0xFFFFFFFFu, w.valid, 0);
                const int blocks = __shfl_sync(0xFFFFFFFFu, w.blocks, 0);
                const bool two = __shfl_sync(0xFFFFFFFFu, w.tokens[1], 0) > 0;
                if (lane == 0) mbar_arrive(smem_u32(&sh.piece_empty[at]));
                __syncwarp();
                if (!valid) break;
                for (int i = 0; i < blocks && ok; ++i, ++kv_it) {
                    const uint32_t stages = qk ? Shared::kK : Shared::kV16, stage = kv_it % stages, phase = (kv_it / stages) & 1u;
                    PH_MARK(0);
                    if (qk) {
                        ok = wait8(wctx, smem_u32(&sh.k_full[stage]), phase, 6);
                        if (!ok) break;
                        PH_MARK(1);
#pragma unroll
                        for (int x = 0; x < 2; ++x) {
                            if (!tree8_takes(two, i, x)) continue;
                            const int tile = two ? x : 0;
                            if (i == 0) {
                                ok = warp_wait8(wctx, smem_u32(&sh.q_full[tile]), (par >> tile) & 1u, 7);
                                if (!ok) break;
                                par ^= 1u << tile;
                            }
                            // The softmax warps have taken the S before this one out of tensor memory.
                            ok = wait8(wctx, smem_u32(&sh.s_empty), (s_it & 1u) ^ 1u, 8);
                            if (!ok) break;
                            PH_MARK(2);
                            ++s_it;
                            tc_fence_after_sync();
                            const uint32_t q_lo = q_lo0 + tile * 2 * kStageStep, k_lo = k_lo0 + stage * kStageStep;
                            umma8_ss_x4_w(tmem_base + kFwdColS, q_lo, k_lo, idesc_qk, 0u);
                            umma8_ss_x4_w(tmem_base + kFwdColS, q_lo + kStageStep, k_lo, idesc_qk, 1u);
                            tc_commit_w(smem_u32(&sh.s_full[x]));
                            if (i == blocks - 1) tc_commit_w(smem_u32(&sh.q_empty[tile]));
                            __syncwarp();
                            PH_MARK(3);
                        }
                        tc_commit_w(smem_u32(&sh.k_empty[stage]));
                    } else {
                        ok = wait8(wctx, smem_u32(&sh.v16_full[stage]), phase, 9);
                        if (!ok) break;
                        PH_MARK(1);
#pragma unroll
                        for (int x = 0; x < 2; ++x) {
                            if (!tree8_takes(two, i, x)) continue;
                            ok = wait8(wctx, smem_u32(&sh.p_full[x]), (par >> x) & 1u, 10);
                            if (!ok) break;
                            PH_MARK(2);
                            par ^= 1u << x;
                            tc_fence_after_sync();
                            umma_ts_x8_w(tmem_base + kFwdColO + x * 128u, tmem_base + kFwdColP + x * kFwdColPStep,
                                         v_lo0 + stage * (kTileBytes >> 4), idesc_pv, i > (two ? 0 : x) ? 1u : 0u);
                            tc_commit_w(smem_u32(&sh.pv_done[x]));
                            __syncwarp();
                            PH_MARK(3);
                        }
                        tc_commit_w(smem_u32(&sh.v16_empty[stage]));
                    }
                }
            }
            PH_PRINT("tree8 mma", 4);
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
        uint32_t s_cnt = 0, pv_cnt = 0, seen_cnt = 0, both_cnt = 0, kv_base = 0, q_par = 0;
        bool ok = true;
        PH_DECL(6)   // 0 other, 1 which slots are seen, 2 wait S, 3 take S, 4 V rows and mask, 5 softmax

        for (uint32_t it = 0; ok; ++it) {
            const uint32_t at = it % kTree8Slots;
            ok = warp_wait(wctx, smem_u32(&sh.piece_full[at]), (it / kTree8Slots) & 1u, 11);
            if (!ok) break;
            const TreePiece& w = sh.piece[at];
            auto release = [&]() {
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&sh.piece_empty[at]));
            };
            if (!w.valid) break;
            const bool two = w.tokens[1] > 0;
            const int tile = two ? x : 0;
            const int tokens = w.tokens[tile];
            const int rows = tokens * p.c.group;
            const bool row_valid = r < rows;
            const bool active = quarter * 32 < rows;      // the warp has a row at all
            const int token = w.tok0 + tile * p.tile_tokens + row_token;
            const bool masked = p.c.mask != nullptr;

            // Q in two parts: of two tiles a warpgroup has its own, of one tile a warp has 16 rows.
            {
                const int t0 = w.tok0 + tile * p.tile_tokens;
                const __nv_bfloat16* q = p8.q + (static_cast<long long>(w.q_begin) + t0) * p8.q_stride[0] +
                                         static_cast<long long>(w.head) * p.c.group * p8.q_stride[1] + (lane & 15) * 8;
                const int r0 = two ? quarter * 32 : warp * 16, r1 = min(rows, r0 + (two ? 32 : 16)), second = lane >> 4;
                auto ask = [&](int row) -> uint4 {
                    row = min(row, rows - 1);
                    const int t = row / p.c.group;
                    return *reinterpret_cast<const uint4*>(q + t * p8.q_stride[0] + (row - t * p.c.group) * p8.q_stride[1]);
                };
                uint4 next[2] = {ask(r0 + second), ask(r0 + 2 + second)};
                ok = warp_wait(wctx, smem_u32(&sh.q_empty[tile]), ((q_par >> tile) & 1u) ^ 1u, 2);
                if (!ok) break;
#pragma unroll 1
                for (int from = r0; from < r1; from += 4) {
                    const uint4 v[2] = {next[0], next[1]};
                    if (from + 4 < r1) {
                        next[0] = ask(from + 4 + second);
                        next[1] = ask(from + 6 + second);
                    }
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int row = from + 2 * e + second;
                        split_q_rows(v[e], row < r1, row, lane, &sh.q[tile][0][0], &sh.q[tile][1][0],
                                     &sh.q_scale[tile][row & (kTileM - 1)]);
                    }
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(smem_u32(&sh.q_full[tile]));
                    if (two) mbar_arrive(smem_u32(&sh.q_full[tile]));
                }
                ok = warp_wait(wctx, smem_u32(&sh.q_full[tile]), (q_par >> tile) & 1u, 19);
                if (!ok) break;
                q_par ^= two ? 3u : 1u;
            }
            const float q_scale = row_valid ? sh.q_scale[tile][r] * sl2 : 0.f;

            float m_used = -INFINITY;   // running reference maximum (log2 units, with V's scale)
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
                // Lane g < 8 has K's scale of slots [16 g, 16 g + 16) of the block, lane 8 + g V's.
                const uint32_t scale_slot = (kv_base + i) % kScaleSlots;
                ok = warp_wait(wctx, smem_u32(&sh.scales.full[scale_slot]), ((kv_base + i) / kScaleSlots) & 1u, 21);
                if (!ok) break;
                float scale = sh.scales.scale[scale_slot][(lane >> 3) & 1][lane & 7];
                if (lane >= 8) scale = fminf(fmaxf(scale, kScaleLeast), kScaleMost);
                const float scale_log2 = fast_log2(scale), scale_part = 1.f / scale;
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(smem_u32(&sh.scales.empty[scale_slot]));
                    if (!two) mbar_arrive(smem_u32(&sh.scales.empty[scale_slot]));
                }
                // What a score of 16 slots is multiplied by, and what is added: scores in log2 units, with V's scale.  Masked ones
                // are -inf, so the factor must not be 0.
                auto factor_of = [&](int g) { return fmaxf(q_scale * __shfl_sync(0xFFFFFFFFu, scale, g), FLT_MIN); };
                auto addend_of = [&](int g) { return __shfl_sync(0xFFFFFFFFu, scale_log2, 8 + g); };
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
                float bm = -INFINITY;
#pragma unroll
                for (int g = 0; g < 8; ++g) {
                    float m = fmaxf(s[g * 16], s[g * 16 + 1]);
#pragma unroll
                    for (int e = 2; e < 16; e += 2) m = max3(m, s[g * 16 + e], s[g * 16 + e + 1]);
                    bm = fmaxf(bm, fmaf(m, factor_of(g), addend_of(g)));
                }
                const float m_new = fmaxf(m_used, bm);
                if (begins) {
                    m_used = m_new;
                } else if (__any_sync(0xFFFFFFFFu, row_valid && m_new - m_used > kP8Most - kP8At)) {
                    // O is scaled only when the maximum has moved by a factor of 2^13: the division at the end uses the same
                    // one.  Rows of the tile that do not exist have no say: what lies there differs from call to call.
                    const float factor = m_new == -INFINITY ? 1.f : fast_exp2(m_used - m_new);
                    l *= factor;
                    m_used = m_new;
                    ok = wait_pv();
                    if (!ok) break;
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
                const float neg_m = m_used == -INFINITY ? 0.f : kP8At - m_used;
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    uint32_t t[32];
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        const float mul = factor_of(c * 4 + g), add = addend_of(c * 4 + g) + neg_m;
                        float2 acc = make_float2(0.f, 0.f);
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            const int at = c * 64 + g * 16 + e * 2;
                            const float2 x2 = fma2(make_float2(s[at], s[at + 1]), make_float2(mul, mul), make_float2(add, add));
                            const float2 p2 = make_float2(fast_exp2(x2.x), fast_exp2(x2.y));
                            acc = e == 0 ? p2 : add2(acc, p2);
                            t[g * 8 + e] = pack_half2(p2.x, p2.y);
                        }
                        l = fmaf(acc.x + acc.y, __shfl_sync(0xFFFFFFFFu, scale_part, 8 + c * 4 + g), l);
                    }
                    if (c == 0 && pv_pending) {
                        ok = wait_pv();
                        if (!ok) break;
                    }
                    tmem_st_x32(p_tmem + c * 32, t);
                }
                if (!ok) break;
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
                a0 = s0.x == m_used ? 1.f : fast_exp2(s0.x - m_used);
                a1 = s1.x == m_used ? 1.f : fast_exp2(s1.x - m_used);
                l = s0.y * a0 + s1.y * a1;
                if (w.blocks == 1) a1 = 0.f;
            }
            if (active) {
                const bool not_finite = *reinterpret_cast<volatile uint32_t*>(&sh.not_finite[at]) == it + 1;
                // A sum of 0: the row sees nothing (or only what is -inf).  NaN stays NaN.
                const float inv = l == 0.f ? 0.f : 1.f / l;
                const bool whole = w.part < 0;
                if (row_valid && (two || x == 0)) {
                    if (whole) {
                        const float lse = l == 0.f ? -INFINITY : (m_used - kP8At + fast_log2(l)) * kLn2;
                        const int head = w.head * p.c.group + row_head;
                        p.lse[w.seq * p.lse_seq_stride + head * p.lse_head_stride +
                              (p.c.cu_seqlens_q == nullptr ? token : w.q_begin + token)] = lse;
                    } else {
                        p.part_stat[(static_cast<long long>(w.part) * Shared::kTiles + tile) * p.part_rows + r] =
                            make_float2(m_used - kP8At - kRescaleThreshold, l);      // tree_combine's reference
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
                    if (not_finite) tree8_add_not_finite(p, w, token, c * 32, t);
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
        PH_PRINT("tree8 softmax", 6);
    }

    // Common exit: every role arrives here (normally or after an abort).
    tc_fence_before_sync();
    __syncthreads();
    if (warp == kTree8QkWarp) {
        tc_fence_after_sync();
        tmem_dealloc(tmem_base, 512);
    }
}

int set_tree8_smem() {
    B2A_CUDA_OK(cudaFuncSetAttribute(tree8_attention, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kTree8SmemBytes)));
    return B2A_OK;
}

}  // namespace

}  // namespace b2a

extern "C" {

int b2a_tree8_fwd(const b2a_tree_args* a, const b2a_cache_scales* scales, void* scratch, size_t scratch_bytes, void* cuda_stream) {
    using namespace b2a;
    B2A_REQUIRE(a != nullptr && scales != nullptr, "args and scales must not be NULL");
    Tree8Params p8{};
    TreeParams& p = p8.t;
    int rc = make_cache_queries(*a, true, &p.c);
    if (rc == B2A_OK) rc = make_cache_scales(*scales, a->cache, &p8.scales);
    if (rc != B2A_OK) return rc;
    for (int i = 0; i < 2; ++i) {
        // Of one token or head it is never stepped, and a caller may say anything.
        p8.q_stride[i] = (i == 0 ? a->total_q : a->heads_q) == 1 ? 0 : a->q_stride[i];
        B2A_REQUIRE(p8.q_stride[i] >= 0 && p8.q_stride[i] % 8 == 0, "strides of q must be multiples of 8 elements");
    }
    p8.q = static_cast<const __nv_bfloat16*>(a->q);
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
    p.c.min_run = 2;      // blocks of a CTA, at least: 1, 2, 4, 8 take 20.5, 20.3, 22.5, 26.6 us for a tree of 8 over 700 slots
    // What an item costs besides its blocks, in blocks, for the cuts between CTAs.  4 and 6, 16 sequences of a token over up to 8,001
    // slots: 44.8, 44.5 us; 6 and 9, of up to 32 tokens with one tile: 80.3, 82.9, of 64 with two, 8 sequences of up to 16,000: 222.9, 220.2.
    p.c.item_extra = t.tiles == 2 ? 9 : 6;
    p.box_rows = slot_box_rows(p.c.cache);
    CUtensorMap map_k, map_v;
    rc = make_slot_map8(&map_k, p.c.cache, true, p.box_rows);
    if (rc == B2A_OK) rc = make_slot_map8(&map_v, p.c.cache, false, p.box_rows);
    if (rc == B2A_OK && t.tiles == 2) rc = once_per_device(dev.device, 15, set_tree8_smem);
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
    if (t.few) return launch_tree8_few(map_k, map_v, p8, t.ctas, dev, stream);
    if (t.tiles == 1) {
        rc = launch_tree8_one(map_k, map_v, p8, t.ctas, dev, stream);
        if (rc != B2A_OK) return rc;
    } else {
        auto attention = tree8_attention;
        B2A_CUDA_OK(launch_early(attention, t.ctas, kTree8Threads, kTree8SmemBytes, stream, map_k, map_v, p8));
    }
    if (t.ctas == 1) return B2A_OK;
    TreeParams parts = p;
    parts.scale_log2 = 1.f;      // the pieces' references are in log2 units already
    return launch_tree_combine(parts, t.ctas, stream);
}

}  // extern "C"
