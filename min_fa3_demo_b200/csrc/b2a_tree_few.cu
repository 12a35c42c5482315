// Attention of drafted tokens over a cache for items of at most 32 rows (tokens times query heads of a K/V head): plain
// decoding, and small trees.  The mathematics, the work's order and the masks are those of b2a_tree.cu; the products are made the
// other way round.
//
// S^T = K Q^T has a lane of tensor memory for each slot and a column for each row, so that all 128 threads of a warpgroup share
// the softmax of a few rows, where a thread for each row would leave most of them idle and one warp with 128 exponentials a
// row and block.  P^T goes to shared memory in bf16, and O^T += V^T P^T has a lane for each dimension and a column for each row.
// Both products are 128 x N x 128 with N = 16 or 32.
//
// Softmax across threads: a row's probabilities are taken relative to a reference in shared memory which all slots of a block
// have to share.  It need not be the maximum: P in bf16 and the sums in fp32 have the exponents of fp32, so any bound will
// do that lies no more than 2^32 above some score (V down to 2^-90 then keeps its products normal).  A piece begins with that
// much above its first slot's, and a block asks once whether any score is larger (one barrier of the warpgroup); only then
// are the maxima over the threads looked for.  No probability is above 1, so no product with a finite V overflows.  Each
// thread adds up its own slots' probabilities; the sums meet at the end of the piece.
//
// The two warpgroups take turns at the blocks, each with a reference, a sum and an O^T of its own.  A block needs some 1,000 clk
// from K to the end of its product with V, and up to six stages of 32 KiB are on their way: bound by memory.
// One token, 32 heads over 8, 16 sequences of 16,384 slots: 1.07 GB in 171 us, 6.3 TB/s; of up to 8,001 slots: 293 MB in 57 us,
// 5.1 TB/s.
//
//   warp 0-3, 4-7   softmax
//   warp 8          K Q^T       warp 10   V^T P^T       warp 9   plan, loads of Q and K       warp 11   loads of V
#include "b2a_tree.cuh"

namespace b2a {

namespace {

constexpr int kFewThreads = 384;
constexpr int kFewSlots = 4;
constexpr int kFewQkWarp = 8, kFewLoadWarp = 9, kFewPvWarp = 10, kFewVWarp = 11;
constexpr float kFewAbove = 32.f;     // log2 units: how far above the score that it was taken from a reference lies

template <int N>
struct __align__(1024) FewShared {
    // More rows leave room for fewer blocks.
    static constexpr int kQ = N == 16 ? 2 : 1, kK = 3, kV = 3;
    uint8_t q[kQ][N * 256];           // two halves of [N rows][128 bytes]
    uint8_t p[2][N * 256];            // P^T of the warpgroups, likewise
    uint8_t k[kK][kTileBytes];
    uint8_t v[kV][kTileBytes];
    float minus_ref[2][N];            // -reference of each row (log2 units); 0: none yet; -inf: there is no such row
    uint32_t none[2][N];              // the row has no reference yet
    long long lse_at[N];              // of each row of an item, from its first: where its lse lies,
    int out_at[N];                    // and which row of out it is
    float top[2][4][N];               // of each warp: maxima, then sums
    float2 stat[2][N];                // reference and sum of the two warpgroups
    uint32_t token_rows[N];           // the rows of a token
    TreePiece piece[kFewSlots];
    uint64_t q_full[kQ], q_empty[kQ];
    uint64_t k_full[kK], k_empty[kK];
    uint64_t v_full[kV], v_empty[kV];
    uint64_t s_full[2], s_empty[2], p_full[2], pv_done[2], meet[2];
    uint64_t both_done, both_read;
    uint64_t piece_full[kFewSlots], piece_empty[kFewSlots];
    uint32_t moves[2][2];             // of each warpgroup, in turn: number of the last block that had to move a reference
    uint32_t not_finite;
    uint32_t missing;                 // the CTA has met a page that does not exist
    uint32_t tmem_base;
    uint32_t abort_flag;
};

template <int N>
constexpr size_t few_smem_bytes() { return sizeof(FewShared<N>) + 1024; }
static_assert(few_smem_bytes<16>() <= 227 * 1024 && few_smem_bytes<32>() <= 227 * 1024, "");

// N columns of tensor memory.
template <int N>
__device__ __forceinline__ void few_ld(uint32_t taddr, uint32_t (&r)[N]) {
    if constexpr (N == 8) {
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
    if constexpr (N == 16) {
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] += __shfl_xor_sync(0xFFFFFFFFu, v[i], 16);
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

// The eight k-steps of a 128 x N x 128 product, B with two halves of N rows of 128 bytes.
template <int N, bool kAMnMajor>
__device__ __forceinline__ void few_product(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t accumulate) {
    constexpr uint32_t idesc = make_idesc_bf16(kTileM, N, kAMnMajor ? 1 : 0, 0);
#pragma unroll
    for (int ks = 0; ks < 8; ++ks) {
        const uint32_t a_step = kAMnMajor ? kstep_mnmajor(ks) : kstep_kmajor(ks);
        const uint32_t b_step = static_cast<uint32_t>((ks >> 2) * (N * 128 >> 4) + (ks & 3) * 2);
        umma_ss_lo_w(d, a_lo + a_step, b_lo + b_step, idesc, ks > 0 ? 1u : accumulate);
    }
}

template <int N>
__global__ void __launch_bounds__(kFewThreads, 1)
tree_attention_few(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                   const __grid_constant__ CUtensorMap map_v, const __grid_constant__ TreeParams p) {
    using Shared = FewShared<N>;
    extern __shared__ uint8_t smem_raw[];
    Shared& sh = *reinterpret_cast<Shared*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    constexpr uint32_t kTmem = N * 4;                 // S^T of the warpgroups [0, 2 N), O^T [2 N, 4 N)

    if (threadIdx.x == 0) {
        for (int i = 0; i < Shared::kQ; ++i) {
            mbar_init(smem_u32(&sh.q_full[i]), 1);
            mbar_init(smem_u32(&sh.q_empty[i]), 1);
        }
        for (int i = 0; i < Shared::kK; ++i) {
            mbar_init(smem_u32(&sh.k_full[i]), 1);
            mbar_init(smem_u32(&sh.k_empty[i]), 1);
        }
        for (int i = 0; i < Shared::kV; ++i) {
            mbar_init(smem_u32(&sh.v_full[i]), 1);
            mbar_init(smem_u32(&sh.v_empty[i]), 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(smem_u32(&sh.s_full[i]), 1);
            mbar_init(smem_u32(&sh.s_empty[i]), 4);
            mbar_init(smem_u32(&sh.p_full[i]), 4);
            mbar_init(smem_u32(&sh.pv_done[i]), 1);
            mbar_init(smem_u32(&sh.meet[i]), 4);
            sh.moves[i][0] = sh.moves[i][1] = 0;
        }
        mbar_init(smem_u32(&sh.both_done), 8);
        mbar_init(smem_u32(&sh.both_read), 8);
        for (int i = 0; i < kFewSlots; ++i) {
            mbar_init(smem_u32(&sh.piece_full[i]), 1);
            mbar_init(smem_u32(&sh.piece_empty[i]), 3 + 8);
        }
        sh.abort_flag = 0;
        sh.not_finite = 0;
        sh.missing = 0;
        fence_mbar_init();
        fence_proxy_async_smem();
    }
    // Rows of Q that no load ever writes.
    for (int i = threadIdx.x; i < Shared::kQ * N * 16; i += kFewThreads) reinterpret_cast<uint4*>(&sh.q[0][0])[i] = make_uint4(0u, 0u, 0u, 0u);
    if (threadIdx.x < N) {
        const int first = threadIdx.x * p.c.group, last = first + p.c.group;
        const uint32_t to = last >= 32 ? ~0u : (1u << last) - 1, from = first >= 32 ? ~0u : (1u << first) - 1;
        sh.token_rows[threadIdx.x] = to & ~from;
        const int token = threadIdx.x / p.c.group, head = threadIdx.x - token * p.c.group;
        sh.lse_at[threadIdx.x] = head * p.lse_head_stride + token;
        sh.out_at[threadIdx.x] = token * p.c.heads_q + head;
    }
    fence_proxy_async_smem();
    if (warp == kFewQkWarp) {
        tmem_alloc(smem_u32(&sh.tmem_base), kTmem);
        tmem_relinquish();
        tc_fence_before_sync();
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

    if (warp == kFewLoadWarp) {
        // ---------------------------------------------------------------- plan, loads of Q and K
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
        uint32_t k_it = 0;
        bool ok = true;
        PH_DECL(3)   // 0 other, 1 wait for K's stage, 2 issue K
        for (uint32_t it = 0; ok; ++it) {
            const uint32_t at = it % kFewSlots;
            ok = warp_wait(wctx, smem_u32(&sh.piece_empty[at]), ((it / kFewSlots) & 1u) ^ 1u, 1);
            if (!ok) break;
            const TreePiece w = tree_piece(p, walk);
            if (lane == 0) {
                sh.piece[at] = w;
                mbar_arrive(smem_u32(&sh.piece_full[at]));
            }
            if (!w.valid) break;
            loader.look_up(p.c.cache, w.seq, w.j0, w.slots, lane);
            const uint32_t buf = it % Shared::kQ;
            ok = warp_wait(wctx, smem_u32(&sh.q_empty[buf]), ((it / Shared::kQ) & 1u) ^ 1u, 2);
            if (!ok) break;
            if (lane == 0) {
                const uint32_t bar = smem_u32(&sh.q_full[buf]), dst = smem_u32(&sh.q[buf][0]);
                mbar_arrive_expect_tx(bar, static_cast<uint32_t>(p.tile_tokens * p.c.group) * 256u);
                tma_load_3d(dst, &map_q, bar, 0, w.head * p.c.group, w.q_begin);
                tma_load_3d(dst + N * 128, &map_q, bar, 64, w.head * p.c.group, w.q_begin);
            }
            __syncwarp();
            for (int i = 0; i < w.blocks; ++i, ++k_it) {
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
            }
            if (!ok) break;
            walk.advance(p.c, w.blocks);
        }
        if (__any_sync(0xFFFFFFFFu, loader.bad) && lane == 0) set_status(wctx.status_word(), kStatusBadArg, 0x3Fu << 12);
        PH_PRINT("few load", 3);
    } else if (warp == kFewVWarp) {
        tree_load_v<kFewSlots, Shared::kV>(p, sh, &map_v, wctx, lane);
    } else if (warp == kFewQkWarp || warp == kFewPvWarp) {
        // ---------------------------------------------------------------- products
        const bool qk = warp == kFewQkWarp;
        const uint32_t q_lo0 = desc_lo_kmajor(smem_u32(&sh.q[0][0])), p_lo0 = desc_lo_kmajor(smem_u32(&sh.p[0][0]));
        const uint32_t k_lo0 = desc_lo_kmajor(smem_u32(&sh.k[0][0])), v_lo0 = desc_lo_mnmajor(smem_u32(&sh.v[0][0]));
        uint32_t kv_it = 0;
        uint32_t par = 0;       // bit x: phase of warpgroup x's S^T (P^T)
        bool ok = true;
        PH_DECL(4)   // 0 other, 1 wait K (V), 2 wait S (P), 3 issue
        for (uint32_t it = 0; ok; ++it) {
            const uint32_t at = it % kFewSlots;
            ok = warp_wait(wctx, smem_u32(&sh.piece_full[at]), (it / kFewSlots) & 1u, 5);
            if (!ok) break;
            const volatile TreePiece& w = sh.piece[at];
            const int valid = __shfl_sync(0xFFFFFFFFu, w.valid, 0);
            const int blocks = __shfl_sync(0xFFFFFFFFu, w.blocks, 0);
            if (lane == 0) mbar_arrive(smem_u32(&sh.piece_empty[at]));
            __syncwarp();
            if (!valid) break;
            const uint32_t buf = it % Shared::kQ;
            if (qk) {
                ok = warp_wait(wctx, smem_u32(&sh.q_full[buf]), (it / Shared::kQ) & 1u, 7);
                if (!ok) break;
            }
            for (int i = 0; i < blocks; ++i, ++kv_it) {
                const uint32_t x = i & 1;
                PH_MARK(0);
                if (qk) {
                    const uint32_t stage = kv_it % Shared::kK;
                    ok = warp_wait(wctx, smem_u32(&sh.k_full[stage]), (kv_it / Shared::kK) & 1u, 6);
                    if (!ok) break;
                    PH_MARK(1);
                    ok = warp_wait(wctx, smem_u32(&sh.s_empty[x]), ((par >> x) & 1u) ^ 1u, 8);
                    if (!ok) break;
                    par ^= 1u << x;
                    PH_MARK(2);
                    tc_fence_after_sync();
                    few_product<N, false>(tmem_base + x * N, k_lo0 + stage * (kTileBytes >> 4), q_lo0 + buf * (N * 256 >> 4), 0u);
                    tc_commit_w(smem_u32(&sh.s_full[x]));
                    tc_commit_w(smem_u32(&sh.k_empty[stage]));
                    if (i == blocks - 1) tc_commit_w(smem_u32(&sh.q_empty[buf]));
                } else {
                    const uint32_t stage = kv_it % Shared::kV;
                    ok = warp_wait(wctx, smem_u32(&sh.v_full[stage]), (kv_it / Shared::kV) & 1u, 9);
                    if (!ok) break;
                    PH_MARK(1);
                    ok = warp_wait(wctx, smem_u32(&sh.p_full[x]), (par >> x) & 1u, 10);
                    if (!ok) break;
                    par ^= 1u << x;
                    PH_MARK(2);
                    tc_fence_after_sync();
                    few_product<N, true>(tmem_base + (2 + x) * N, v_lo0 + stage * (kTileBytes >> 4), p_lo0 + x * (N * 256 >> 4),
                                         i > static_cast<int>(x) ? 1u : 0u);
                    tc_commit_w(smem_u32(&sh.pv_done[x]));
                    tc_commit_w(smem_u32(&sh.v_empty[stage]));
                }
                __syncwarp();
                PH_MARK(3);
            }
        }
        PH_PRINT("few mma", 4);
    } else {
        // ---------------------------------------------------------------- softmax
        const int x = warp >> 2, quarter = warp & 3, r = quarter * 32 + lane;      // r: slot of the block, dimension of O^T
        const uint32_t lane_base = static_cast<uint32_t>(quarter * 32) << 16;
        const uint32_t s_tmem = tmem_base + lane_base + x * N, o_tmem = tmem_base + lane_base + 2 * N;
        const float sl2 = p.scale_log2;
        // Where this slot's probabilities lie in P^T: 128-byte rows, 16-byte chunks exchanged by the row's number.
        uint32_t p_at[8];
#pragma unroll
        for (int c = 0; c < 8; ++c) {
            p_at[c] = smem_u32(&sh.p[x][(r >> 6) * (N * 128) + c * 128 + ((((r & 63) >> 3) ^ c) << 4) + (r & 7) * 2]);
        }
        uint32_t s_cnt = 0, pv_cnt = 0, meet_cnt = 0, both_cnt = 0, v_base = 0, block_cnt = 0;
        bool ok = true;
        auto meet = [&]() -> bool {      // of the warpgroup
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&sh.meet[x]));
            return warp_wait(wctx, smem_u32(&sh.meet[x]), meet_cnt++ & 1u, 13);
        };
        PH_DECL(6)   // 0 other, 1 wait S, 2 take S, 3 V rows and mask, 4 reference, 5 P

        for (uint32_t it = 0; ok; ++it) {
            const uint32_t at = it % kFewSlots;
            ok = warp_wait(wctx, smem_u32(&sh.piece_full[at]), (it / kFewSlots) & 1u, 11);
            if (!ok) break;
            const TreePiece& w = sh.piece[at];
            if (!w.valid) break;
            const int rows = w.n * p.c.group;
            float sum[N];
#pragma unroll
            for (int c = 0; c < N; ++c) sum[c] = 0.f;
            bool open = false;           // a row has no reference yet

            for (int i = x; i < w.blocks; i += 2) {
                const int slot = (w.j0 + i) * kSlotBlock + r;
                const bool tail = (w.j0 + i + 1) * kSlotBlock > w.len;     // drafted tokens, or no slots any more
                bool pv_pending = i > x;
                auto wait_pv = [&]() -> bool {
                    if (!pv_pending) return true;
                    if (!warp_wait(wctx, smem_u32(&sh.pv_done[x]), pv_cnt & 1u, 15)) return false;
                    ++pv_cnt;
                    tc_fence_after_sync();
                    pv_pending = false;
                    return true;
                };
                // Rows that see this slot: all of them if it lies before the drafted tokens.
                uint32_t see = ~0u;
                if (tail && slot >= w.len) {
                    const int u = slot - w.len;
                    see = 0;
                    if (slot < w.slots && p.c.mask == nullptr) {
                        see = u * p.c.group >= 32 ? 0u : ~0u << (u * p.c.group);
                    } else if (slot < w.slots && u < w.n) {
                        const unsigned char* byte = tree_mask_row(p, w, 0) + u;
#pragma unroll 8
                        for (int t = 0; t < w.n; ++t) {
                            if (byte[t * p.c.mask_stride[1]] != 0) see |= sh.token_rows[t];
                        }
                    }
                }
                PH_MARK(0);
                ok = warp_wait(wctx, smem_u32(&sh.s_full[x]), s_cnt & 1u, 12);
                if (!ok) break;
                ++s_cnt;
                ++block_cnt;
                PH_MARK(1);
                tc_fence_after_sync();
                // One answer for the warp: the flag may go up, for a block still to come, between two lanes' looks.
                const bool missing = __any_sync(0xFFFFFFFFu, *reinterpret_cast<volatile uint32_t*>(&sh.missing) != 0u);
                uint32_t s[N];
                few_ld<N>(s_tmem, s);
                tmem_wait_ld();
                tc_fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&sh.s_empty[x]));
                PH_MARK(2);
                if (tail) {
                    // As in b2a_tree.cu: a barrier tells the last phase from the one before it, so the V that lay in this
                    // stage before has to have come, which the warpgroup's last product proves.
                    ok = wait_pv();
                    if (!ok) break;
                    const uint32_t stage = (v_base + i) % Shared::kV;
                    ok = warp_wait(wctx, smem_u32(&sh.v_full[stage]), ((v_base + i) / Shared::kV) & 1u, 14);
                    if (!ok) break;
                    if (slot >= w.slots || (slot >= w.len && (w.n > 1 || p.c.mask != nullptr))) {
                        if (tree_clean_row(&sh.v[stage][r * 128], r, slot >= w.slots)) {
                            *reinterpret_cast<volatile uint32_t*>(&sh.not_finite) = it + 1;
                        }
                    }
                    fence_proxy_async_smem();
                }
                if (missing && !p.c.cache.has(w.seq, slot)) see = 0;
                if ((tail || missing) && __any_sync(0xFFFFFFFFu, see != ~0u)) {
#pragma unroll
                    for (int c = 0; c < N; ++c) {
                        if (!((see >> c) & 1u)) s[c] = 0xFF800000u;    // -inf
                    }
                }
                PH_MARK(3);

                const float4* minus_ref = reinterpret_cast<const float4*>(&sh.minus_ref[x][0]);
                if (i == x) {
                    // A piece's first references are the scores of the block's first slot, if all rows see it.
                    if (r == 0) {
#pragma unroll
                        for (int c = 0; c < N; ++c) {
                            const float y = __uint_as_float(s[c]) * sl2;
                            const bool none = !(fabsf(y) < INFINITY);
                            sh.minus_ref[x][c] = c >= rows ? -INFINITY : none ? 0.f : -y - kFewAbove;
                            sh.none[x][c] = none;
                            open |= none && c < rows;
                        }
                        if (open) *reinterpret_cast<volatile uint32_t*>(&sh.moves[x][block_cnt & 1u]) = block_cnt;
                    }
                    ok = meet();
                    if (!ok) break;
                }
                float top = -INFINITY;
#pragma unroll
                for (int c = 0; c < N; c += 4) {
                    const float4 m = minus_ref[c / 4];
                    top = fmaxf(top, fmaxf(fmaxf(fmaf(__uint_as_float(s[c]), sl2, m.x), fmaf(__uint_as_float(s[c + 1]), sl2, m.y)),
                                           fmaxf(fmaf(__uint_as_float(s[c + 2]), sl2, m.z), fmaf(__uint_as_float(s[c + 3]), sl2, m.w))));
                }
                if (__any_sync(0xFFFFFFFFu, open || top > 0.f) && lane == 0) {
                    *reinterpret_cast<volatile uint32_t*>(&sh.moves[x][block_cnt & 1u]) = block_cnt;
                }
                ok = meet();
                if (!ok) break;
                if (__builtin_expect(*reinterpret_cast<volatile uint32_t*>(&sh.moves[x][block_cnt & 1u]) == block_cnt, 0)) {
                    // The rows' maxima over the block: ordered as integers, for which a warp has a reduction.
#pragma unroll
                    for (int c = 0; c < N; ++c) {
                        const float y = __uint_as_float(s[c]) * sl2;
                        const int bits = y == y ? __float_as_int(y) : static_cast<int>(0xFF800000u);
                        const int key = __reduce_max_sync(0xFFFFFFFFu, bits ^ ((bits >> 31) & 0x7FFFFFFF));
                        if (lane == 0) sh.top[x][quarter][c] = __int_as_float(key ^ ((key >> 31) & 0x7FFFFFFF));
                    }
                    ok = wait_pv();
                    if (!ok) break;
                    ok = meet();
                    if (!ok) break;
                    open = false;
                    // In turn, so that no thread has more than a few factors at a time.
#pragma unroll
                    for (int c0 = 0; c0 < N; c0 += 8) {
                        float factor[8];
                        uint32_t o[8];
                        if (i > x) {
                            few_ld<8>(o_tmem + x * N + c0, o);
                            tmem_wait_ld();
                        }
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            const int c = c0 + e;
                            const float m = fmaxf(fmaxf(sh.top[x][0][c], sh.top[x][1][c]), fmaxf(sh.top[x][2][c], sh.top[x][3][c]));
                            const bool none = sh.none[x][c] != 0u;           // then sum and O are 0
                            factor[e] = !none && m + sh.minus_ref[x][c] > 0.f ? fast_exp2(-sh.minus_ref[x][c] - m - kFewAbove) : 1.f;
                            open |= c < rows && none && m == -INFINITY;
                            sum[c] *= factor[e];
                        }
                        if (i > x) {
#pragma unroll
                            for (int e = 0; e < 8; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * factor[e]);
                            asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                                         ::"r"(o_tmem + x * N + c0), "r"(o[0]), "r"(o[1]), "r"(o[2]), "r"(o[3]), "r"(o[4]), "r"(o[5]),
                                           "r"(o[6]), "r"(o[7])
                                         : "memory");
                        }
                    }
                    if (i > x) tmem_wait_st();
                    ok = meet();                 // all have read the old references
                    if (!ok) break;
                    if (r < rows) {
                        const float m = fmaxf(fmaxf(sh.top[x][0][r], sh.top[x][1][r]), fmaxf(sh.top[x][2][r], sh.top[x][3][r]));
                        if (sh.none[x][r] != 0u ? m != -INFINITY : m + sh.minus_ref[x][r] > 0.f) {
                            sh.minus_ref[x][r] = -m - kFewAbove;
                            sh.none[x][r] = 0u;
                        }
                    }
                    ok = meet();
                    if (!ok) break;
                }
                PH_MARK(4);
                ok = wait_pv();                  // P^T of the block before has been read
                if (!ok) break;
#pragma unroll
                for (int c = 0; c < N; c += 4) {
                    const float4 m4 = minus_ref[c / 4];
                    const float m[4] = {m4.x, m4.y, m4.z, m4.w};
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float prob = fast_exp2(fmaf(__uint_as_float(s[c + e]), sl2, m[e]));
                        sum[c + e] += prob;
                        // Rounded to bf16 for the product: 2^-9 of a term on average, as much as the rounding of out.
                        asm volatile("st.shared.b16 [%0], %1;" ::"r"(p_at[(c + e) & 7] + ((c + e) >> 3) * 1024),
                                     "h"(__bfloat16_as_ushort(__float2bfloat16_rn(prob))) : "memory");
                    }
                }
                fence_proxy_async_smem();
                tc_fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&sh.p_full[x]));
                PH_MARK(5);
            }
            if (!ok) break;
            v_base += w.blocks;
            if (w.blocks > x) {
                ok = warp_wait(wctx, smem_u32(&sh.pv_done[x]), pv_cnt & 1u, 15);
                if (!ok) break;
                ++pv_cnt;
                tc_fence_after_sync();
            }

            // The warpgroup's sums, and then both warpgroups' parts: O = a0 O0 + a1 O1, half of the rows each.
            few_column_sums<N>(sum, lane);
            ok = meet();                         // nobody still reads maxima
            if (!ok) break;
            if (lane < N) sh.top[x][quarter][lane] = sum[0];
            ok = meet();
            if (!ok) break;
            if (r < N) {
                const float ref = w.blocks <= x || sh.none[x][r] != 0u ? -INFINITY : -sh.minus_ref[x][r];
                sh.stat[x][r] = make_float2(ref, (sh.top[x][0][r] + sh.top[x][1][r]) + (sh.top[x][2][r] + sh.top[x][3][r]));
            }
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&sh.both_done));
            ok = warp_wait(wctx, smem_u32(&sh.both_done), both_cnt & 1u, 16);
            if (!ok) break;
            tc_fence_after_sync();
            const bool not_finite = *reinterpret_cast<volatile uint32_t*>(&sh.not_finite) == it + 1;
            const bool whole = w.part < 0;
            for (int c0 = x * (N / 2); c0 < min((x + 1) * (N / 2), rows); c0 += 8) {
                uint32_t o0[8], o1[8];
                few_ld<8>(o_tmem + c0, o0);
                if (w.blocks > 1) few_ld<8>(o_tmem + N + c0, o1);
                tmem_wait_ld();
                float o[8], ref[8], l[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float2 s0 = sh.stat[0][c0 + e], s1 = sh.stat[1][c0 + e];
                    ref[e] = fmaxf(s0.x, s1.x);
                    const float a0 = s0.x == ref[e] ? 1.f : fast_exp2(s0.x - ref[e]);
                    const float a1 = s1.x == ref[e] ? 1.f : fast_exp2(s1.x - ref[e]);
                    l[e] = s0.y * a0 + s1.y * a1;
                    o[e] = __uint_as_float(o0[e]) * a0;
                    if (w.blocks > 1) o[e] = fmaf(__uint_as_float(o1[e]), a1, o[e]);
                }
                if (not_finite) {
                    // Values of drafted tokens that are not finite, added to the rows that see them.
                    const int from = max(0, w.j0 * kSlotBlock - w.len), to = min(w.n, (w.j0 + w.blocks) * kSlotBlock - w.len);
                    for (int u = from; u < to; ++u) {
                        const long long slot = static_cast<long long>(w.len) + u;
                        int row;
                        const int page = slot < w.slots ? p.c.cache.page_of(w.seq, slot, &row) : -1;
                        if (page < 0) continue;
                        const uint32_t bits = __bfloat16_as_ushort(p.c.cache.v[p.c.cache.at(p.c.cache.v_stride, page, row, w.head) + r]);
                        if (!bf16_not_finite(bits)) continue;
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            if (c0 + e < rows && tree_sees(p, w, (c0 + e) / p.c.group, u)) o[e] += __uint_as_float(bits << 16);
                        }
                    }
                }
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int row = c0 + e;
                    if (row >= rows) continue;
                    if (whole) {
                        const long long to = static_cast<long long>(w.q_begin) * p.c.heads_q + w.head * p.c.group + sh.out_at[row];
                        // A sum of 0: the row sees nothing (or only what is -inf).  NaN stays NaN.
                        const float inv = l[e] == 0.f ? 0.f : 1.f / l[e];
                        p.out[to * kHeadDim + r] = __float2bfloat16_rn(o[e] * inv);
                        if (r == 0) {
                            p.lse[w.seq * p.lse_seq_stride + w.head * p.c.group * p.lse_head_stride +
                                  (p.c.cu_seqlens_q == nullptr ? 0 : w.q_begin) + sh.lse_at[row]] =
                                l[e] == 0.f ? -INFINITY : (ref[e] + fast_log2(l[e])) * kLn2;
                        }
                    } else {
                        const long long to = static_cast<long long>(w.part) * p.part_rows + row;
                        reinterpret_cast<float*>(p.part_o)[to * kHeadDim + r] = o[e];
                        if (r == 0) p.part_stat[to] = make_float2(ref[e], l[e]);
                    }
                }
            }
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&sh.both_read));
            ok = warp_wait(wctx, smem_u32(&sh.both_read), both_cnt & 1u, 17);
            ++both_cnt;
            if (!ok) break;
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&sh.piece_empty[at]));
        }
        PH_PRINT("few softmax", 6);
    }

    tc_fence_before_sync();
    __syncthreads();
    if (warp == kFewQkWarp) {
        tc_fence_after_sync();
        tmem_dealloc(tmem_base, kTmem);
    }
}

// As tree_combine: adds up the pieces of the item that run blockIdx.x + 1 begins inside of, if it is the first to do so.  A warp a row.
__global__ void __launch_bounds__(256)
tree_combine_few(const __grid_constant__ TreeParams p) {
    let_next_kernel_start();
    wait_for_previous_kernel();
    const int cta = blockIdx.x + 1, lane = threadIdx.x & 31;
    const TreeCut cut = p.cuts[cta];
    if (cut.run == 0 || cut.first < static_cast<long long>(cta - 1) * cut.run) return;
    const int row = blockIdx.y * 8 + (threadIdx.x >> 5);
    if (row >= cut.n * p.c.group) return;
    const int pieces = static_cast<int>((cut.last - 1) / cut.run) - (cta - 1) + 1;
    auto part_of = [&](int i) -> long long {
        const int second = i == 0 && cut.first > static_cast<long long>(cta - 1) * cut.run;
        return (2ll * (cta - 1 + i) + second) * p.part_rows + row;
    };
    float m = -INFINITY;
#pragma unroll 4
    for (int i = 0; i < pieces; ++i) m = fmaxf(m, p.part_stat[part_of(i)].x);
    float l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int i = 0; i < pieces; ++i) {
        const float2 st = p.part_stat[part_of(i)];
        const float4 v = p.part_o[part_of(i) * 32 + lane];
        const float f = st.x == m ? 1.f : fast_exp2(st.x - m);
        l = fmaf(st.y, f, l);
        o = make_float4(fmaf(v.x, f, o.x), fmaf(v.y, f, o.y), fmaf(v.z, f, o.z), fmaf(v.w, f, o.w));
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const int token = row / p.c.group, head = cut.head * p.c.group + row - token * p.c.group;
    const long long to = (static_cast<long long>(cut.q_begin) + token) * p.c.heads_q + head;
    *reinterpret_cast<uint2*>(p.out + to * kHeadDim + lane * 4) =
        make_uint2(pack_bf16x2(o.x * inv, o.y * inv), pack_bf16x2(o.z * inv, o.w * inv));
    if (lane == 0) {
        p.lse[cut.seq * p.lse_seq_stride + head * p.lse_head_stride + (p.c.cu_seqlens_q == nullptr ? token : cut.q_begin + token)] =
            l == 0.f ? -INFINITY : (m + fast_log2(l)) * kLn2;
    }
}

template <int N>
int set_few_smem() {
    B2A_CUDA_OK(cudaFuncSetAttribute(tree_attention_few<N>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     static_cast<int>(few_smem_bytes<N>())));
    return B2A_OK;
}

template <int N>
int launch_few(const CUtensorMap& map_q, const CUtensorMap& map_k, const CUtensorMap& map_v, const TreeParams& p, int ctas,
               cudaStream_t stream) {
    auto attention = tree_attention_few<N>;
    B2A_CUDA_OK(launch_early(attention, ctas, kFewThreads, few_smem_bytes<N>(), stream, map_q, map_k, map_v, p));
    return B2A_OK;
}

}  // namespace

int launch_tree_few(const CUtensorMap& map_q, const CUtensorMap& map_k, const CUtensorMap& map_v, const TreeParams& p, int ctas,
                    const DeviceInfo& dev, cudaStream_t stream) {
    int rc;
    if (p.part_rows <= 16) {
        rc = once_per_device(dev.device, 8, set_few_smem<16>);
        if (rc == B2A_OK) rc = launch_few<16>(map_q, map_k, map_v, p, ctas, stream);
    } else {
        rc = once_per_device(dev.device, 9, set_few_smem<32>);
        if (rc == B2A_OK) rc = launch_few<32>(map_q, map_k, map_v, p, ctas, stream);
    }
    if (rc != B2A_OK || ctas == 1) return rc;
    auto combine = tree_combine_few;
    B2A_CUDA_OK(launch_early(combine, dim3(ctas - 1, (p.part_rows + 7) / 8), 256, 0, stream, p));
    return B2A_OK;
}

}  // namespace b2a
