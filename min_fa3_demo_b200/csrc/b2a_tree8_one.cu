// Attention over a cache in 8 bits of calls whose items have one tile of rows, more than 32 and at most 128: larger trees.  As
// b2a_tree8.cu, except for what follows from the time that a block has: the two warpgroups take turns at the blocks, so each block
// has to be done in half the time that one of two tiles has.
//
// Four warps turn V to f16.  What is left of the registers is 184 a thread, so a thread takes its row's scores in halves of 64, and each
// warpgroup has an S of its own, which it may hold meanwhile: P goes to where S's first half was, and the next K Q^T of a warpgroup
// waits for its P V.  The reference need not be the maximum, so it stays where the first half put it unless the second lies more
// than 2^13 above it.  Trees of up to 32 tokens, 32 heads over 8, 16 sequences of up to 8,000 slots: 153 MB in 81 us, as of two
// tiles 100; of 64 tokens, 64 heads over 8, which has two tiles, 262 us so and 228 as in b2a_tree8.cu.
//
//   warp 0-3, 4-7   Q in two parts, then softmax, one thread a row
//   warp 8          Q K^T       warp 10   P V       warp 9   plan, loads of K and scales       warp 11   loads of V
//   warp 12-15      V to f16
//
// Tensor memory (512 columns): S of the warpgroups [0,128) [128,256), O [256,384) [384,512).
#include "b2a_cache8.cuh"

#include <cfloat>
#include <cmath>

namespace b2a {

namespace {

constexpr int kOne8Threads = 512;
constexpr int kOne8Slots = 4;       // pieces in flight between the load warp and the others
constexpr int kOne8QkWarp = 8, kOne8LoadWarp = 9, kOne8PvWarp = 10, kOne8VWarp = 11, kOne8ConvertWarp = 12;

struct __align__(1024) One8Shared {
    static constexpr int kK = 4, kV = 3, kV16 = 2;
    uint8_t q[2][kTile8Bytes];              // both parts
    uint8_t k[kK][kTile8Bytes];
    uint8_t v[kV][kTile8Bytes];
    uint8_t v16[kV16][kTileBytes];          // V in f16, two halves of 64 columns
    float q_scale[kTileM];                  // what a row of Q is multiplied by
    ScaleRing<1> scales;
    uint32_t seen[2][2][kTileM][4];   // warpgroup, turn, token: one bit for each slot of the block
    float2 stat[2][kTileM];           // row maximum and sum of the two warpgroups
    TreePiece piece[kOne8Slots];
    uint64_t q_full, q_empty;
    uint64_t k_full[kK], k_empty[kK];
    uint64_t v_full[kV], v_empty[kV];
    uint64_t v16_full[kV16], v16_empty[kV16];
    uint64_t s_full[2], p_full[2], pv_done[2];
    uint64_t seen_full[2];
    uint64_t both_done, both_read;
    uint64_t piece_full[kOne8Slots], piece_empty[kOne8Slots];
    uint32_t not_finite[kOne8Slots]; // number, plus one, of the piece that met a drafted value that is NaN
    uint32_t missing;                 // the CTA has met a page that does not exist
    uint32_t tmem_base;
    uint32_t abort_flag;
};

constexpr size_t kOne8SmemBytes = sizeof(One8Shared) + 1024;
static_assert(kOne8SmemBytes <= 227 * 1024, "shared memory of a CTA");

__global__ void __launch_bounds__(kOne8Threads, 1)
tree8_attention_one(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                const __grid_constant__ Tree8Params p8) {
    const TreeParams& p = p8.t;
    extern __shared__ uint8_t smem_raw[];
    using Shared = One8Shared;
    Shared& sh = *reinterpret_cast<Shared*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(smem_u32(&sh.s_full[i]), 1);
            mbar_init(smem_u32(&sh.p_full[i]), kTileM);
            mbar_init(smem_u32(&sh.pv_done[i]), 1);
            mbar_init(smem_u32(&sh.seen_full[i]), kTileM);
        }
        sh.scales.init(4);
        mbar_init(smem_u32(&sh.q_full), 8);             // warps
        mbar_init(smem_u32(&sh.q_empty), 1);
        mbar_init(smem_u32(&sh.both_done), 2 * kTileM);
        mbar_init(smem_u32(&sh.both_read), 2 * kTileM);
        for (int i = 0; i < Shared::kK; ++i) {
            mbar_init(smem_u32(&sh.k_full[i]), 1);
            mbar_init(smem_u32(&sh.k_empty[i]), 1);
        }
        for (int i = 0; i < Shared::kV; ++i) {
            mbar_init(smem_u32(&sh.v_full[i]), 1);
            mbar_init(smem_u32(&sh.v_empty[i]), 4);
        }
        for (int i = 0; i < Shared::kV16; ++i) {
            mbar_init(smem_u32(&sh.v16_full[i]), 4);
            mbar_init(smem_u32(&sh.v16_empty[i]), 1);
        }
        for (int i = 0; i < kOne8Slots; ++i) {
            mbar_init(smem_u32(&sh.piece_full[i]), 1);
            mbar_init(smem_u32(&sh.piece_empty[i]), 3 + 4 + 8);   // MMA warps, V's load warp, converting and softmax warps
            sh.not_finite[i] = 0;
        }
        sh.abort_flag = 0;
        sh.missing = 0;
        fence_mbar_init();
        fence_proxy_async_smem();
    }
    if (warp == kOne8QkWarp) {
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
        if (warp == kOne8LoadWarp) {
            // ------------------------------------------------------------ plan, loads of K and scales
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
                const uint32_t at = it % kOne8Slots;
                ok = warp_wait8(wctx, smem_u32(&sh.piece_empty[at]), ((it / kOne8Slots) & 1u) ^ 1u, 1);
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
                    PH_MARK(2);
                }
                if (!ok) break;
                walk.advance(p.c, w.blocks);
            }
            if (__any_sync(0xFFFFFFFFu, loader.bad) && lane == 0) set_status(wctx.status_word(), kStatusBadArg, 0x3Fu << 12);
            PH_PRINT("one8 load", 3);
        } else if (warp == kOne8VWarp) {
            tree8_load_v<kOne8Slots, Shared::kV>(p, sh, &map_v, wctx, lane);
        } else if (warp >= kOne8ConvertWarp) {
            tree8_convert_v<4, kOne8Slots, Shared::kV, Shared::kV16>(p, sh, wctx, threadIdx.x - 32 * kOne8ConvertWarp,
                                                                      [](const TreePiece&, uint32_t) { return true; });
        } else if (warp == kOne8QkWarp || warp == kOne8PvWarp) {
            // ------------------------------------------------------------ MMA warps
            const bool qk = warp == kOne8QkWarp;
            constexpr uint32_t idesc_qk = make_idesc_first(kTileM, kTileN, 0, 0), idesc_pv = make_idesc_first(kTileM, kHeadDim, 0, 1);
            constexpr uint32_t kStageStep = kTile8Bytes >> 4;
            const uint32_t q_lo0 = desc_lo_kmajor(smem_u32(&sh.q[0][0]));
            const uint32_t k_lo0 = desc_lo_kmajor(smem_u32(&sh.k[0][0]));
            const uint32_t v_lo0 = desc_lo_mnmajor(smem_u32(&sh.v16[0][0]));
            uint32_t kv_it = 0, par = 0;       // bit x of par: phase of warpgroup x's P V (qk), P
            bool ok = true;
            PH_DECL(4)   // 0 other, 1 wait K (V), 2 wait S (P), 3 issue
            for (uint32_t it = 0; ok; ++it) {
                const uint32_t at = it % kOne8Slots;
                ok = warp_wait8(wctx, smem_u32(&sh.piece_full[at]), (it / kOne8Slots) & 1u, 5);
                if (!ok) break;
                const volatile TreePiece& w = sh.piece[at];
                const int valid = __shfl_sync(0xFFFFFFFFu, w.valid, 0);
                const int blocks = __shfl_sync(0xFFFFFFFFu, w.blocks, 0);
                if (lane == 0) mbar_arrive(smem_u32(&sh.piece_empty[at]));
                __syncwarp();
                if (!valid) break;
                for (int i = 0; i < blocks && ok; ++i, ++kv_it) {
                    const uint32_t stages = qk ? Shared::kK : Shared::kV16, stage = kv_it % stages, phase = (kv_it / stages) & 1u;
                    const uint32_t x = i & 1;
                    PH_MARK(0);
                    if (qk) {
                        ok = wait8(wctx, smem_u32(&sh.k_full[stage]), phase, 6);
                        if (!ok) break;
                        PH_MARK(1);
                        if (i == 0) {
                            ok = warp_wait8(wctx, smem_u32(&sh.q_full), it & 1u, 7);
                            if (!ok) break;
                        }
                        // P takes S's place, so the product with it has to be done.
                        ok = wait8(wctx, smem_u32(&sh.pv_done[x]), ((par >> x) & 1u) ^ 1u, 8);
                        if (!ok) break;
                        par ^= 1u << x;
                        PH_MARK(2);
                        tc_fence_after_sync();
                        const uint32_t k_lo = k_lo0 + stage * kStageStep;
                        umma8_ss_x4_w(tmem_base + x * 128u, q_lo0, k_lo, idesc_qk, 0u);
                        umma8_ss_x4_w(tmem_base + x * 128u, q_lo0 + kStageStep, k_lo, idesc_qk, 1u);
                        tc_commit_w(smem_u32(&sh.s_full[x]));
                        tc_commit_w(smem_u32(&sh.k_empty[stage]));
                        if (i == blocks - 1) tc_commit_w(smem_u32(&sh.q_empty));
                    } else {
                        ok = wait8(wctx, smem_u32(&sh.v16_full[stage]), phase, 9);
                        if (!ok) break;
                        PH_MARK(1);
                        ok = wait8(wctx, smem_u32(&sh.p_full[x]), (par >> x) & 1u, 10);
                        if (!ok) break;
                        par ^= 1u << x;
                        PH_MARK(2);
                        tc_fence_after_sync();
                        umma_ts_x8_w(tmem_base + kFwdColO + x * 128u, tmem_base + x * 128u, v_lo0 + stage * (kTileBytes >> 4), idesc_pv,
                                     i > static_cast<int>(x) ? 1u : 0u);
                        tc_commit_w(smem_u32(&sh.pv_done[x]));
                        tc_commit_w(smem_u32(&sh.v16_empty[stage]));
                    }
                    __syncwarp();
                    PH_MARK(3);
                }
            }
            PH_PRINT("one8 mma", 4);
        }
    } else {
        // ---------------------------------------------------------------- softmax warpgroups
        reg_alloc<184>();
        const int x = warp >> 2;
        const int quarter = warp & 3;
        const int r = quarter * 32 + lane;
        const uint32_t lane_base = static_cast<uint32_t>(quarter * 32) << 16;
        const uint32_t s_tmem = tmem_base + lane_base + static_cast<uint32_t>(x) * 128u;
        const uint32_t p_tmem = s_tmem;      // both halves of P in the columns of S's first half, read by then
        const uint32_t o_tmem = tmem_base + lane_base + kFwdColO;
        const float sl2 = p.scale_log2;
        const int row_token = r / p.c.group;           // of the tile
        const int row_head = r - row_token * p.c.group;
        uint32_t s_cnt = 0, pv_cnt = 0, seen_cnt = 0, both_cnt = 0, kv_base = 0;
        bool ok = true;
        PH_DECL(6)   // 0 other, 1 which slots are seen, 2 wait S, 3 take S, 4 V rows and mask, 5 softmax

        for (uint32_t it = 0; ok; ++it) {
            const uint32_t at = it % kOne8Slots;
            ok = warp_wait(wctx, smem_u32(&sh.piece_full[at]), (it / kOne8Slots) & 1u, 11);
            if (!ok) break;
            const TreePiece& w = sh.piece[at];
            auto release = [&]() {
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&sh.piece_empty[at]));
            };
            if (!w.valid) break;
            const int tokens = w.tokens[0];
            const int rows = tokens * p.c.group;
            const bool row_valid = r < rows;
            const bool active = quarter * 32 < rows;      // the warp has a row at all
            const int token = w.tok0 + row_token;
            const bool masked = p.c.mask != nullptr;

            // Q in two parts, 16 rows a warp.
            {
                const __nv_bfloat16* q = p8.q + (static_cast<long long>(w.q_begin) + w.tok0) * p8.q_stride[0] +
                                         static_cast<long long>(w.head) * p.c.group * p8.q_stride[1] + (lane & 15) * 8;
                const int r0 = warp * 16, r1 = min(rows, r0 + 16), second = lane >> 4;
                auto ask = [&](int row) -> uint4 {
                    row = min(row, rows - 1);
                    const int t = row / p.c.group;
                    return *reinterpret_cast<const uint4*>(q + t * p8.q_stride[0] + (row - t * p.c.group) * p8.q_stride[1]);
                };
                uint4 next[2] = {ask(r0 + second), ask(r0 + 2 + second)};
                ok = warp_wait(wctx, smem_u32(&sh.q_empty), (it & 1u) ^ 1u, 2);
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
                        split_q_rows(v[e], row < r1, row, lane, &sh.q[0][0], &sh.q[1][0], &sh.q_scale[row & (kTileM - 1)]);
                    }
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&sh.q_full));
                ok = warp_wait(wctx, smem_u32(&sh.q_full), it & 1u, 19);
                if (!ok) break;
            }
            const float q_scale = row_valid ? sh.q_scale[r] * sl2 : 0.f;

            float m_used = -INFINITY;   // running reference maximum (log2 units, with V's scale)
            float l = 0.f;              // running row sum relative to m_used
            for (int i = x; i < w.blocks; i += 2) {
                const int base = (w.j0 + i) * kSlotBlock;
                const bool tail = base + kSlotBlock > w.len;   // drafted tokens, or no slots any more
                uint32_t* seen = nullptr;
                PH_MARK(0);
                if (tail && masked) {
                    // Which slots of the block each token sees: a warp's lanes are 32 slots.  Eight tokens' bytes at a time.
                    const int slot = base + quarter * 32 + lane, u = slot - w.len;
                    const bool ask = slot < w.slots && u >= 0 && u < w.n, always = u < 0 && slot < w.slots;
                    const unsigned char* byte = tree_mask_row(p, w, w.tok0) + (ask ? u : 0);
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
                // Lane g < 8 has K's scale of slots [16 g, 16 g + 16) of the block, lane 8 + g V's.
                const uint32_t scale_slot = (kv_base + i) % kScaleSlots;
                ok = warp_wait(wctx, smem_u32(&sh.scales.full[scale_slot]), ((kv_base + i) / kScaleSlots) & 1u, 21);
                if (!ok) break;
                float scale = sh.scales.scale[scale_slot][(lane >> 3) & 1][lane & 7];
                if (lane >= 8) scale = fminf(fmaxf(scale, kScaleLeast), kScaleMost);
                const float scale_log2 = fast_log2(scale), scale_part = 1.f / scale;
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&sh.scales.empty[scale_slot]));
                // What a score of 16 slots is multiplied by, and what is added: scores in log2 units, with V's scale.  Masked ones are -inf, so
                // the factor must not be 0.
                auto factor_of = [&](int g) { return fmaxf(q_scale * __shfl_sync(0xFFFFFFFFu, scale, g), FLT_MIN); };
                auto addend_of = [&](int g) { return __shfl_sync(0xFFFFFFFFu, scale_log2, 8 + g); };
                const bool begins = i == static_cast<int>(x);
                bool pv_pending = !begins;
                auto wait_pv = [&]() -> bool {
                    if (!mbar_wait(wctx, smem_u32(&sh.pv_done[x]), pv_cnt & 1u, 15)) return false;
                    ++pv_cnt;
                    tc_fence_after_sync();
                    pv_pending = false;
                    return true;
                };

                if (tail && masked) {
                    ok = warp_wait(wctx, smem_u32(&sh.seen_full[x]), seen_cnt & 1u, 13);
                    if (!ok) break;
                    ++seen_cnt;
                }
                if (!active) {
                    // None of the warp's rows exists; it keeps step, and its P and O are never looked at.
                    if (pv_pending) {
                        ok = wait_pv();
                        if (!ok) break;
                    }
                    mbar_arrive(smem_u32(&sh.p_full[x]));
                    continue;
                }
                const bool missing = __any_sync(0xFFFFFFFFu, *reinterpret_cast<volatile uint32_t*>(&sh.missing) != 0u);
                PH_MARK(3);
                // Half of the block at a time, so that a thread has 64 scores and not 128: the reference need not be the maximum, and it
                // may stay where the first half put it unless the second lies more than 2^13 above it.
#pragma unroll 1
                for (int h = 0; h < 2; ++h) {
                    float s[64];
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        uint32_t t[32];
                        tmem_ld_x32(s_tmem + h * 64 + c * 32, t);
#pragma unroll
                        for (int e = 0; e < 32; ++e) s[c * 32 + e] = __uint_as_float(t[e]);
                    }
                    tmem_wait_ld();
                    if (__builtin_expect(tail || missing, 0)) {
                        // One bit per visible slot of 32 (missing: asked once for the warp, as the flag may go up, for a block still to
                        // come, between two lanes' looks).
                        const int lim = min(w.slots, w.len + token + 1) - base;
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            const int at = h * 64 + c * 32;
                            uint32_t bits = 0xFFFFFFFFu;
                            if (tail && masked) {
                                bits = seen[min(row_token, tokens - 1) * 4 + h * 2 + c];
                            } else if (tail) {
                                const int vis = min(max(lim - at, 0), 32);
                                bits = vis == 32 ? 0xFFFFFFFFu : (1u << vis) - 1u;
                            }
                            if (missing) bits &= __ballot_sync(0xFFFFFFFFu, p.c.cache.has(w.seq, base + at + lane));
#pragma unroll
                            for (int e = 0; e < 32; ++e) {
                                if (!((bits >> e) & 1u)) s[c * 32 + e] = -INFINITY;
                            }
                        }
                    }
                    float bm = -INFINITY;
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        float m = fmaxf(s[g * 16], s[g * 16 + 1]);
#pragma unroll
                        for (int e = 2; e < 16; e += 2) m = max3(m, s[g * 16 + e], s[g * 16 + e + 1]);
                        bm = fmaxf(bm, fmaf(m, factor_of(h * 4 + g), addend_of(h * 4 + g)));
                    }
                    const float m_new = fmaxf(m_used, bm);
                    if (begins && h == 0) {
                        m_used = m_new;
                    } else if (__builtin_expect(__any_sync(0xFFFFFFFFu, row_valid && m_new - m_used > kP8Most - kP8At), 0)) {
                        // What there is relative to the old reference is scaled: the sum, O, and P of the first half.  The division at the
                        // end uses the same one.  Rows that do not exist have no say: what lies there differs from
                        // call to call.
                        const float factor = m_new == -INFINITY ? 1.f : fast_exp2(m_used - m_new);
                        l *= factor;
                        m_used = m_new;
                        if (pv_pending) {
                            ok = wait_pv();
                            if (!ok) break;
                        }
#pragma unroll 1
                        for (int c = 0; c < 16 && !begins; ++c) {
                            uint32_t t[8];
                            few_ld<8>(o_tmem + x * 128 + c * 8, t);
                            tmem_wait_ld();
#pragma unroll
                            for (int e = 0; e < 8; ++e) t[e] = __float_as_uint(__uint_as_float(t[e]) * factor);
                            tmem_st_x8(o_tmem + x * 128 + c * 8, t);
                        }
                        if (h == 1) tmem_wait_st();
#pragma unroll 1
                        for (int c = 0; c < 4 && h == 1; ++c) {
                            uint32_t t[8];
                            few_ld<8>(p_tmem + c * 8, t);
                            tmem_wait_ld();
#pragma unroll
                            for (int e = 0; e < 8; ++e) {
                                const float2 two = half2_to_float2(t[e]);
                                t[e] = pack_half2(two.x * factor, two.y * factor);
                            }
                            tmem_st_x8(p_tmem + c * 8, t);
                        }
                    }
                    const float neg_m = m_used == -INFINITY ? 0.f : kP8At - m_used;
                    uint32_t t[32];
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        const float mul = factor_of(h * 4 + g), add = addend_of(h * 4 + g) + neg_m;
                        float2 acc = make_float2(0.f, 0.f);
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            const int at = g * 16 + e * 2;
                            const float2 x2 = fma2(make_float2(s[at], s[at + 1]), make_float2(mul, mul), make_float2(add, add));
                            const float2 p2 = make_float2(fast_exp2(x2.x), fast_exp2(x2.y));
                            acc = e == 0 ? p2 : add2(acc, p2);
                            t[g * 8 + e] = pack_half2(p2.x, p2.y);
                        }
                        l = fmaf(acc.x + acc.y, __shfl_sync(0xFFFFFFFFu, scale_part, 8 + h * 4 + g), l);
                    }
                    if (pv_pending) {
                        ok = wait_pv();
                        if (!ok) break;
                    }
                    tmem_st_x32(p_tmem + h * 32, t);
                }
                if (!ok) break;
                tmem_wait_st();
                tc_fence_before_sync();
                mbar_arrive(smem_u32(&sh.p_full[x]));
                PH_MARK(5);
            }
            if (!ok) break;
            kv_base += w.blocks;
            if (w.blocks > x) {
                ok = mbar_wait(wctx, smem_u32(&sh.pv_done[x]), pv_cnt & 1u, 15);
                if (!ok) break;
                ++pv_cnt;
                tc_fence_after_sync();
            }

            // The two warpgroups' parts, O = a0 O0 + a1 O1; each does half of the columns.
            sh.stat[x][r] = make_float2(m_used, l);
            tc_fence_before_sync();
            mbar_arrive(smem_u32(&sh.both_done));
            ok = warp_wait(wctx, smem_u32(&sh.both_done), both_cnt & 1u, 16);
            if (!ok) break;
            tc_fence_after_sync();
            const float2 s0 = sh.stat[0][r], s1 = sh.stat[1][r];
            m_used = fmaxf(s0.x, s1.x);
            const float a0 = s0.x == m_used ? 1.f : fast_exp2(s0.x - m_used), a1 = s1.x == m_used ? 1.f : fast_exp2(s1.x - m_used);
            l = s0.y * a0 + s1.y * a1;
            if (active) {
                const bool not_finite = *reinterpret_cast<volatile uint32_t*>(&sh.not_finite[at]) == it + 1;
                // A sum of 0: the row sees nothing (or only what is -inf).  NaN stays NaN.
                const float inv = l == 0.f ? 0.f : 1.f / l;
                const bool whole = w.part < 0;
                if (row_valid && x == 0) {
                    if (whole) {
                        const float lse = l == 0.f ? -INFINITY : (m_used - kP8At + fast_log2(l)) * kLn2;
                        const int head = w.head * p.c.group + row_head;
                        p.lse[w.seq * p.lse_seq_stride + head * p.lse_head_stride +
                              (p.c.cu_seqlens_q == nullptr ? token : w.q_begin + token)] = lse;
                    } else {
                        p.part_stat[static_cast<long long>(w.part) * p.part_rows + r] =
                            make_float2(m_used - kP8At - kRescaleThreshold, l);      // tree_combine's reference
                    }
                }
                __nv_bfloat16* o_row = p.out + ((static_cast<long long>(w.q_begin) + token) * p.c.heads_q +
                                                w.head * p.c.group + row_head) * kHeadDim;
                float4* part = p.part_o + static_cast<long long>(w.part) * 32 * p.part_rows + r;
#pragma unroll 1
                for (int c = 2 * x; c < 2 * x + 2; ++c) {
                    uint32_t t[32];
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
            // Neither warpgroup's next product may overwrite an O that the other still reads.
            mbar_arrive(smem_u32(&sh.both_read));
            ok = warp_wait(wctx, smem_u32(&sh.both_read), both_cnt & 1u, 17);
            ++both_cnt;
            if (!ok) break;
            release();
        }
        PH_PRINT("one8 softmax", 6);
    }

    // Common exit: every role arrives here (normally or after an abort).
    tc_fence_before_sync();
    __syncthreads();
    if (warp == kOne8QkWarp) {
        tc_fence_after_sync();
        tmem_dealloc(tmem_base, 512);
    }
}

int set_one8_smem() {
    B2A_CUDA_OK(cudaFuncSetAttribute(tree8_attention_one, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kOne8SmemBytes)));
    return B2A_OK;
}

}  // namespace

int launch_tree8_one(const CUtensorMap& map_k, const CUtensorMap& map_v, const Tree8Params& p, int ctas, const DeviceInfo& dev,
                     cudaStream_t stream) {
    const int rc = once_per_device(dev.device, 16, set_one8_smem);
    if (rc != B2A_OK) return rc;
    auto attention = tree8_attention_one;
    B2A_CUDA_OK(launch_early(attention, ctas, kOne8Threads, kOne8SmemBytes, stream, map_k, map_v, p));
    return B2A_OK;
}

}  // namespace b2a
