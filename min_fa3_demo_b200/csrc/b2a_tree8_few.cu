// Attention of drafted tokens over a cache in 8 bits for items of at most 32 rows (tokens times query heads of a K/V head): plain
// decoding, and small trees.  The work's order and the masks are those of b2a_tree_few.cu, the numbers those of b2a_cache8.cuh.
//
// S^T = K Q^T has a lane of tensor memory for each slot and a column for each row, O^T += V^T P^T a lane for each dimension: K
// and V (in f16) are the A operands, the two 8-bit parts of Q and P in f16 the B operands.
//
// A step is two blocks, 256 slots: K of 32 KiB, as much as a block of a bf16 cache, so that the warps that load and multiply do as
// little for a byte as there.  A thread has two slots, and so two scales of K and two of V.  The products have at least 16
// columns, but only as many as there may be rows go through the softmax: 8, 16, or, in steps of one block, 32.
//
// Softmax across threads, as in b2a_tree_few.cu: a row's reference is a score, the first slot's of a piece, and moves to a maximum
// that is looked for when a score lies more than 2^13 above it (f16 has fewer exponents than bf16, so not 2^32 below); whether
// one does costs a barrier of the warpgroup a step.  The two warpgroups take turns at the steps, each with a reference, a sum and an O^T
// of its own.
//
// Bound by memory: 16 sequences of one token, 32 heads over 8, up to 8,001 slots, 173 MB in 43 us; one of 131,072 slots, 269 MB in 60.
// Longer ones go at 6.3 TB/s behind 17 us that do not depend on the length: the first loads and products of a CTA, its pieces'
// results, and the launch that joins them.
//
//   warp 0-3, 4-7   softmax
//   warp 8          K Q^T       warp 10   V^T P^T       warp 9   plan, loads of K and scales       warp 11   loads of V
//   warp 12-15      Q in two parts, V to f16
#include "b2a_cache8.cuh"

#include <cuda_fp16.h>

namespace b2a {

namespace {

constexpr int kFew8Threads = 512;
constexpr int kFew8Slots = 4;       // pieces in flight
constexpr int kFew8QkWarp = 8, kFew8LoadWarp = 9, kFew8PvWarp = 10, kFew8VWarp = 11, kFew8ConvertWarp = 12;

// R: rows, of which there may be fewer.
template <int R>
struct __align__(1024) Few8Shared {
    static constexpr int N = R < 16 ? 16 : R;      // columns of the products
    static constexpr int B = R == 32 ? 1 : 2;      // blocks of a step
    static constexpr int kQ = 2, kK = 4 / B, kV = R == 32 ? 3 : 4, kV16 = 2;
    static constexpr uint32_t kTmem = 128;         // S^T of the warpgroups, N columns a block, then O^T
    static_assert(2 * B * N + 2 * N <= kTmem, "tensor memory");
    uint8_t q[kQ][2][N * 128];        // both parts
    uint8_t p[2][B][N * 256];         // P^T of the warpgroups in f16, a block as two halves of [N rows][128 bytes]
    uint8_t k[kK][B * kTile8Bytes];
    uint8_t v[kV][kTile8Bytes];
    uint8_t v16[kV16][kTileBytes];    // V in f16, two halves of 64 columns
    float q_scale[kQ][N];             // what a row of Q is multiplied by
    ScaleRing<B> scales;
    float minus_ref[2][N];            // -reference of each row (log2 units); 0: none yet; -inf: there is no such row
    uint32_t none[2][N];              // the row has no reference yet
    long long lse_at[N];              // of each row of an item, from its first: where its lse lies,
    long long q_at[N];                // where its query lies,
    int out_at[N];                    // and which row of out it is
    float top[2][4][N];               // of each warp: maxima, then sums
    float2 stat[2][N];                // reference and sum of the two warpgroups
    uint32_t token_rows[N];           // the rows of a token
    TreePiece piece[kFew8Slots];
    uint64_t q_full[kQ], q_empty[kQ];
    uint64_t k_full[kK], k_empty[kK];
    uint64_t v_full[kV], v_empty[kV];
    uint64_t v16_full[kV16], v16_empty[kV16];
    uint64_t s_full[2], s_empty[2], p_full[2], pv_done[2], meet[2];
    uint64_t both_done, both_read;
    uint64_t piece_full[kFew8Slots], piece_empty[kFew8Slots];
    uint32_t moves[2][2];             // of each warpgroup, in turn: number of the last step that had to move a reference
    uint32_t not_finite[kFew8Slots];  // number, plus one, of the piece that met a drafted value that is NaN
    uint32_t missing;                 // the CTA has met a page that does not exist
    uint32_t tmem_base;
    uint32_t abort_flag;
};

template <int R>
constexpr size_t few8_smem_bytes() {
    static_assert(sizeof(Few8Shared<R>) + 1024 <= 227 * 1024, "shared memory of a CTA");
    return sizeof(Few8Shared<R>) + 1024;
}

__device__ __forceinline__ float v_scale_of(float scale) { return fminf(fmaxf(scale, kScaleLeast), kScaleMost); }

// Rows that see a slot, a bit each.  Little of it is needed often.
static __device__ __noinline__ uint32_t few8_seen(const TreeParams& p, const TreePiece& w, const uint32_t* token_rows, int slot) {
    if (slot >= w.slots || !p.c.cache.has(w.seq, slot)) return 0u;
    const int u = slot - w.len;
    if (u < 0) return ~0u;
    if (p.c.mask == nullptr) return u * p.c.group >= 32 ? 0u : ~0u << (u * p.c.group);
    uint32_t see = 0;
    const unsigned char* byte = tree_mask_row(p, w, 0) + u;
#pragma unroll 4
    for (int t = 0; t < w.n; ++t) {
        if (byte[t * p.c.mask_stride[1]] != 0) see |= token_rows[t];
    }
    return see;
}

// Whether a row's token sees a drafted token of the piece whose value of dimension `dim` is NaN.
static __device__ __noinline__ bool few8_sees_nan(const TreeParams& p, const TreePiece& w, int token, int dim) {
    const int from = max(0, w.j0 * kSlotBlock - w.len), to = min(w.n, (w.j0 + w.blocks) * kSlotBlock - w.len);
    for (int u = from; u < to; ++u) {
        const long long slot = static_cast<long long>(w.len) + u;
        int row;
        const int page = slot < w.slots ? p.c.cache.page_of(w.seq, slot, &row) : -1;
        if (page < 0 || !tree_sees(p, w, token, u)) continue;
        const uint8_t* v = reinterpret_cast<const uint8_t*>(p.c.cache.v) + p.c.cache.at(p.c.cache.v_stride, page, row, w.head);
        if (e4m3_not_finite(v[dim])) return true;
    }
    return false;
}

// Of four rows' values those of pair e: of a step of two blocks a row's value for both slots, of one block two rows'.
template <int B>
__device__ __forceinline__ float2 few8_rows(const float4& v, int e) {
    if constexpr (B == 2) {
        const float x = e == 0 ? v.x : e == 1 ? v.y : e == 2 ? v.z : v.w;
        return make_float2(x, x);
    } else {
        return e == 0 ? make_float2(v.x, v.y) : make_float2(v.z, v.w);
    }
}

template <int R>
__global__ void __launch_bounds__(kFew8Threads, 1)
tree8_attention_few(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                    const __grid_constant__ Tree8Params p8) {
    using Shared = Few8Shared<R>;
    constexpr int N = Shared::N, B = Shared::B;
    const TreeParams& p = p8.t;
    extern __shared__ uint8_t smem_raw[];
    Shared& sh = *reinterpret_cast<Shared*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int i = 0; i < Shared::kQ; ++i) {
            mbar_init(smem_u32(&sh.q_full[i]), 4);
            mbar_init(smem_u32(&sh.q_empty[i]), 1 + 8);      // the products, and the warps that read q_scale
        }
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
        for (int i = 0; i < 2; ++i) {
            mbar_init(smem_u32(&sh.s_full[i]), 1);
            mbar_init(smem_u32(&sh.s_empty[i]), 4);
            mbar_init(smem_u32(&sh.p_full[i]), 4);
            mbar_init(smem_u32(&sh.pv_done[i]), 1);
            mbar_init(smem_u32(&sh.meet[i]), 4);
            sh.moves[i][0] = sh.moves[i][1] = 0;
        }
        sh.scales.init(4);
        mbar_init(smem_u32(&sh.both_done), 8);
        mbar_init(smem_u32(&sh.both_read), 8);
        for (int i = 0; i < kFew8Slots; ++i) {
            mbar_init(smem_u32(&sh.piece_full[i]), 1);
            mbar_init(smem_u32(&sh.piece_empty[i]), 3 + 4 + 8);     // MMA warps, V's load warp, converting and softmax warps
            sh.not_finite[i] = 0;
        }
        sh.abort_flag = 0;
        sh.missing = 0;
        fence_mbar_init();
    }
    // Rows of Q that are never written, and their scales.
    for (int i = threadIdx.x; i < Shared::kQ * 2 * N * 8; i += kFew8Threads) {
        reinterpret_cast<uint4*>(&sh.q[0][0][0])[i] = make_uint4(0u, 0u, 0u, 0u);
    }
    if (threadIdx.x < N) {
        const int first = threadIdx.x * p.c.group, last = first + p.c.group;
        const uint32_t to = last >= 32 ? ~0u : (1u << last) - 1, from = first >= 32 ? ~0u : (1u << first) - 1;
        sh.token_rows[threadIdx.x] = to & ~from;
        const int token = threadIdx.x / p.c.group, head = threadIdx.x - token * p.c.group;
        sh.lse_at[threadIdx.x] = head * p.lse_head_stride + token;
        sh.q_at[threadIdx.x] = token * p8.q_stride[0] + head * p8.q_stride[1];
        sh.out_at[threadIdx.x] = token * p.c.heads_q + head;
        for (int i = 0; i < Shared::kQ; ++i) sh.q_scale[i][threadIdx.x] = 1.f;
    }
    fence_proxy_async_smem();
    if (warp == kFew8QkWarp) {
        tmem_alloc(smem_u32(&sh.tmem_base), Shared::kTmem);
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

    if (warp == kFew8LoadWarp) {
        // ---------------------------------------------------------------- plan, loads of K
        if (lane == 0) {
            tma_prefetch_desc(&map_k);
            tma_prefetch_desc(&map_v);
        }
        CacheWalk walk;
        walk.start(p.c, blockIdx.x, gridDim.x, lane);
        if (lane == 0) p.cuts[blockIdx.x] = tree_cut(p, walk);
        SlotLoader loader(p.box_rows, B);
        loader.bad = walk.bad;
        uint32_t k_it = 0;
        bool ok = true;
        PH_DECL(3)   // 0 other, 1 wait for K's stage, 2 issue K
        for (uint32_t it = 0; ok; ++it) {
            const uint32_t at = it % kFew8Slots;
            ok = warp_wait8(wctx, smem_u32(&sh.piece_empty[at]), ((it / kFew8Slots) & 1u) ^ 1u, 1);
            if (!ok) break;
            const TreePiece w = tree_piece(p, walk);
            if (lane == 0) {
                sh.piece[at] = w;
                mbar_arrive(smem_u32(&sh.piece_full[at]));
            }
            if (!w.valid) break;
            const int slots = min(w.slots, (w.j0 + w.blocks) * kSlotBlock);
            loader.look_up(p.c.cache, w.seq, w.j0, slots, lane);
            for (int i = 0; i < w.blocks; i += B, ++k_it) {
                SlotLoader now = loader;
                if (i + B < w.blocks) loader.look_up(p.c.cache, w.seq, w.j0 + i + B, slots, lane);
                const int boxes = now.count(w.j0 + i, slots);
                const uint32_t stage = k_it % Shared::kK;
                PH_MARK(0);
                ok = warp_wait8(wctx, smem_u32(&sh.k_empty[stage]), ((k_it / Shared::kK) & 1u) ^ 1u, 3);
                if (!ok) break;
                PH_MARK(1);
                now.check(p.c.cache, boxes, lane, &sh.missing);
                loader.bad |= now.bad;
                load_slots8(now, &map_k, smem_u32(&sh.k[stage][0]), smem_u32(&sh.k_full[stage]), w.head, boxes, lane);
                ok = sh.scales.load(wctx, k_it, p.c.cache, p8.scales, now, w.j0 + i, slots, w.head, lane);
                if (!ok) break;
                PH_MARK(2);
            }
            if (!ok) break;
            walk.advance(p.c, w.blocks);
        }
        if (__any_sync(0xFFFFFFFFu, loader.bad) && lane == 0) set_status(wctx.status_word(), kStatusBadArg, 0x3Fu << 12);
        PH_PRINT("few8 load", 3);
    } else if (warp == kFew8VWarp) {
        tree8_load_v<kFew8Slots, Shared::kV>(p, sh, &map_v, wctx, lane);
    } else if (warp >= kFew8ConvertWarp) {
        // ---------------------------------------------------------------- Q in two parts, and then V to f16
        const int mine = warp - kFew8ConvertWarp;
        tree8_convert_v<4, kFew8Slots, Shared::kV, Shared::kV16>(p, sh, wctx, mine * 32 + lane, [&](const TreePiece& w, uint32_t it) {
            const int rows = w.n * p.c.group;
            const uint32_t buf = it % Shared::kQ;
            const __nv_bfloat16* q = p8.q + w.q_begin * p8.q_stride[0] + static_cast<long long>(w.head) * p.c.group * p8.q_stride[1] +
                                     (lane & 15) * 8;
            auto ask = [&](int row) { return *reinterpret_cast<const uint4*>(q + sh.q_at[min(row, rows - 1)]); };
            int row = 2 * mine + (lane >> 4);
            uint4 x{};
            if (2 * mine < rows) x = ask(row);
            // A warp without rows waits as well: it could be as far as the next piece that uses this buffer, and what it then adds to
            // q_full would stand for a warp that is still waiting for its rows of this one.
            if (!warp_wait8(wctx, smem_u32(&sh.q_empty[buf]), ((it / Shared::kQ) & 1u) ^ 1u, 2)) return false;
#pragma unroll 1
            for (; row - (lane >> 4) < rows; row += 8) {
                split_q_rows(x, row < rows, row, lane, &sh.q[buf][0][0], &sh.q[buf][1][0], &sh.q_scale[buf][row]);
                if (row - (lane >> 4) + 8 < rows) x = ask(row + 8);
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&sh.q_full[buf]));
            return true;
        });
    } else if (warp == kFew8QkWarp || warp == kFew8PvWarp) {
        // ---------------------------------------------------------------- products
        const bool qk = warp == kFew8QkWarp;
        constexpr uint32_t idesc_qk = make_idesc_first(kTileM, N, 0, 0), idesc_pv = make_idesc_first(kTileM, N, 1, 0);
        constexpr uint32_t kPart = N * 128 >> 4, kStage = kTile8Bytes >> 4;
        const uint32_t q_lo0 = desc_lo_kmajor(smem_u32(&sh.q[0][0][0])), p_lo0 = desc_lo_kmajor(smem_u32(&sh.p[0][0][0]));
        const uint32_t k_lo0 = desc_lo_kmajor(smem_u32(&sh.k[0][0])), v_lo0 = desc_lo_mnmajor(smem_u32(&sh.v16[0][0]));
        uint32_t step = 0, v_it = 0;
        uint32_t par = 0;       // bit x: phase of warpgroup x's S^T (P^T)
        bool ok = true;
        PH_DECL(4)   // 0 other, 1 wait K (V), 2 wait S (P), 3 issue
        for (uint32_t it = 0; ok; ++it) {
            const uint32_t at = it % kFew8Slots;
            ok = warp_wait8(wctx, smem_u32(&sh.piece_full[at]), (it / kFew8Slots) & 1u, 5);
            if (!ok) break;
            const volatile TreePiece& w = sh.piece[at];
            const int valid = __shfl_sync(0xFFFFFFFFu, w.valid, 0);
            const int blocks = __shfl_sync(0xFFFFFFFFu, w.blocks, 0);
            if (lane == 0) mbar_arrive(smem_u32(&sh.piece_empty[at]));
            __syncwarp();
            if (!valid) break;
            const uint32_t buf = it % Shared::kQ;
            if (qk) {
                ok = warp_wait8(wctx, smem_u32(&sh.q_full[buf]), (it / Shared::kQ) & 1u, 7);
                if (!ok) break;
            }
            for (int i = 0; i < blocks; i += B, ++step) {
                const uint32_t x = (i / B) & 1;
                const int here = min(B, blocks - i);
                PH_MARK(0);
                if (qk) {
                    const uint32_t stage = step % Shared::kK;
                    ok = warp_wait8(wctx, smem_u32(&sh.k_full[stage]), (step / Shared::kK) & 1u, 6);
                    if (!ok) break;
                    PH_MARK(1);
                    ok = warp_wait8(wctx, smem_u32(&sh.s_empty[x]), ((par >> x) & 1u) ^ 1u, 8);
                    if (!ok) break;
                    par ^= 1u << x;
                    PH_MARK(2);
                    tc_fence_after_sync();
                    const uint32_t q_lo = q_lo0 + buf * 2 * kPart;
                    for (int h = 0; h < here; ++h) {
                        const uint32_t k_lo = k_lo0 + (stage * B + h) * kStage, to = tmem_base + (x * B + h) * N;
                        umma8_ss_x4_w(to, k_lo, q_lo, idesc_qk, 0u);
                        umma8_ss_x4_w(to, k_lo, q_lo + kPart, idesc_qk, 1u);
                    }
                    tc_commit_w(smem_u32(&sh.s_full[x]));
                    tc_commit_w(smem_u32(&sh.k_empty[stage]));
                    if (i + B >= blocks) tc_commit_w(smem_u32(&sh.q_empty[buf]));
                } else {
                    ok = warp_wait8(wctx, smem_u32(&sh.p_full[x]), (par >> x) & 1u, 10);
                    if (!ok) break;
                    par ^= 1u << x;
                    PH_MARK(2);
                    for (int h = 0; h < here; ++h, ++v_it) {
                        const uint32_t tile = v_it % Shared::kV16;
                        ok = warp_wait8(wctx, smem_u32(&sh.v16_full[tile]), (v_it / Shared::kV16) & 1u, 9);
                        if (!ok) break;
                        PH_MARK(1);
                        tc_fence_after_sync();
                        umma_ss_nk_x8_w<N>(tmem_base + (2 * B + x) * N, v_lo0 + tile * (kTileBytes >> 4),
                                           p_lo0 + (x * B + h) * (N * 256 >> 4), idesc_pv, i + h >= 2 * B || h > 0 ? 1u : 0u);
                        tc_commit_w(smem_u32(&sh.v16_empty[tile]));
                    }
                    if (!ok) break;
                    tc_commit_w(smem_u32(&sh.pv_done[x]));
                }
                __syncwarp();
                PH_MARK(3);
            }
        }
        PH_PRINT("few8 mma", 4);
    } else {
        // ---------------------------------------------------------------- softmax
        const int x = warp >> 2, quarter = warp & 3, r = quarter * 32 + lane;      // r: slot of the block, dimension of O^T
        const uint32_t lane_base = static_cast<uint32_t>(quarter * 32) << 16;
        const uint32_t s_tmem = tmem_base + lane_base + x * B * N, o_tmem = tmem_base + lane_base + 2 * B * N;
        const float sl2 = p.scale_log2;
        // Where a slot's probabilities lie in P^T: 128-byte rows, 16-byte chunks exchanged by the row's number.
        uint32_t p_at[8];
#pragma unroll
        for (int c = 0; c < 8; ++c) {
            p_at[c] = smem_u32(&sh.p[x][0][(r >> 6) * (N * 128) + c * 128 + ((((r & 63) >> 3) ^ c) << 4) + (r & 7) * 2]);
        }
        uint32_t s_cnt = 0, pv_cnt = 0, meet_cnt = 0, both_cnt = 0, k_base = 0, step_cnt = 0;
        bool ok = true;
        auto meet = [&]() -> bool {      // of the warpgroup
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&sh.meet[x]));
            return warp_wait8(wctx, smem_u32(&sh.meet[x]), meet_cnt++ & 1u, 13);
        };
        PH_DECL(10)   // 0 other, 1 wait S, 2 take S, 3 mask, 4 reference, 5 P, 6 wait for Q, 7 move references, 8 results, 9 wait for P V

        for (uint32_t it = 0; ok; ++it) {
            const uint32_t at = it % kFew8Slots;
            ok = warp_wait8(wctx, smem_u32(&sh.piece_full[at]), (it / kFew8Slots) & 1u, 11);
            if (!ok) break;
            const TreePiece& w = sh.piece[at];
            if (!w.valid) break;
            const int rows = w.n * p.c.group;
            const uint32_t buf = it % Shared::kQ;
            PH_MARK(0);
            ok = warp_wait8(wctx, smem_u32(&sh.q_full[buf]), (it / Shared::kQ) & 1u, 19);
            if (!ok) break;
            PH_MARK(6);
            const float4* q_scale = reinterpret_cast<const float4*>(&sh.q_scale[buf][0]);
            float sum[R];
#pragma unroll
            for (int c = 0; c < R; ++c) sum[c] = 0.f;
            bool open = false;           // a row has no reference yet

            for (int i = x * B; i < w.blocks; i += 2 * B) {
                const bool first = i < 2 * B;
                bool pv_pending = !first;
                auto wait_pv = [&]() -> bool {
                    if (!pv_pending) return true;
                    if (!warp_wait8(wctx, smem_u32(&sh.pv_done[x]), pv_cnt & 1u, 15)) return false;
                    ++pv_cnt;
                    tc_fence_after_sync();
                    pv_pending = false;
                    return true;
                };
                const uint32_t step = k_base + i / B, scale_slot = step % kScaleSlots;
                PH_MARK(0);
                ok = warp_wait8(wctx, smem_u32(&sh.s_full[x]), s_cnt & 1u, 12);
                if (!ok) break;
                ++s_cnt;
                ++step_cnt;
                PH_MARK(1);
                tc_fence_after_sync();
                // Scores in log2 units, with V's scale, in pairs: of rows c, c + 1, ... for slots r and 128 + r, or of rows c, c + 1
                // and c + 2, c + 3 for slot r.
                constexpr int kFour = 2 * B;       // pairs of four rows
                float2 y[R / 4 * kFour];
                {
                    uint32_t raw[B][R];
#pragma unroll
                    for (int h = 0; h < B; ++h) few_ld<R>(s_tmem + h * N, raw[h]);
                    ok = warp_wait8(wctx, smem_u32(&sh.scales.full[scale_slot]), (step / kScaleSlots) & 1u, 21);
                    if (!ok) break;
                    tmem_wait_ld();
                    tc_fence_before_sync();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(smem_u32(&sh.s_empty[x]));
                    const float* k_scale = &sh.scales.scale[scale_slot][0][r >> 4];
                    const float* v_scale = &sh.scales.scale[scale_slot][1][r >> 4];
                    const float2 k2 = make_float2(k_scale[0] * sl2, k_scale[(B - 1) * 8] * sl2);
                    const float2 v2 = make_float2(fast_log2(v_scale_of(v_scale[0])), fast_log2(v_scale_of(v_scale[(B - 1) * 8])));
#pragma unroll
                    for (int c = 0; c < R; c += 4) {
                        const float4 q4 = q_scale[c / 4];
#pragma unroll
                        for (int e = 0; e < kFour; ++e) {
                            const float2 s = B == 2 ? make_float2(__uint_as_float(raw[0][c + e]), __uint_as_float(raw[B - 1][c + e]))
                                                    : make_float2(__uint_as_float(raw[0][c + 2 * (e & 1)]), __uint_as_float(raw[0][c + 2 * (e & 1) + 1]));
                            y[c / 4 * kFour + e] = fma2(mul2(s, k2), few8_rows<B>(q4, e), v2);
                        }
                    }
                }
                PH_MARK(2);
                // Drafted tokens, or no slots any more; pages that do not exist (one answer for the warp: the flag may go up, for
                // a step still to come, between two lanes' looks).
                const bool tail = (w.j0 + i + B) * kSlotBlock > w.len;
                const bool missing = __any_sync(0xFFFFFFFFu, *reinterpret_cast<volatile uint32_t*>(&sh.missing) != 0u);
                if (__builtin_expect(tail || i + B > w.blocks || missing, 0)) {
                    uint32_t see[B];
#pragma unroll
                    for (int h = 0; h < B; ++h) {
                        see[h] = i + h < w.blocks ? few8_seen(p, w, sh.token_rows, (w.j0 + i + h) * kSlotBlock + r) : 0u;
                    }
#pragma unroll
                    for (int t = 0; t < R / 4 * kFour; ++t) {
                        if (!((see[0] >> (B == 2 ? t : 2 * t)) & 1u)) y[t].x = -INFINITY;
                        if (!((see[B - 1] >> (B == 2 ? t : 2 * t + 1)) & 1u)) y[t].y = -INFINITY;
                    }
                }
                PH_MARK(3);

                const float4* minus_ref = reinterpret_cast<const float4*>(&sh.minus_ref[x][0]);
                if (first) {
                    // A piece's first references are the scores of the block's first slot, if all rows see it.
                    if (r == 0) {
#pragma unroll
                        for (int c = 0; c < R; ++c) {
                            const float score = B == 2 ? y[c].x : c & 1 ? y[c / 2].y : y[c / 2].x;
                            const bool none = !(fabsf(score) < INFINITY);
                            sh.minus_ref[x][c] = c >= rows ? -INFINITY : none ? 0.f : kP8At - score;
                            sh.none[x][c] = none;
                            open |= none && c < rows;
                        }
                        if (open) *reinterpret_cast<volatile uint32_t*>(&sh.moves[x][step_cnt & 1u]) = step_cnt;
                    }
                    ok = meet();
                    if (!ok) break;
                }
                float top = -INFINITY;
#pragma unroll
                for (int c = 0; c < R; c += 4) {
                    const float4 m4 = minus_ref[c / 4];
#pragma unroll
                    for (int e = 0; e < kFour; ++e) {
                        const float2 up = add2(y[c / 4 * kFour + e], few8_rows<B>(m4, e));
                        top = max3(top, up.x, up.y);
                    }
                }
                if (__any_sync(0xFFFFFFFFu, open || top > kP8Most) && lane == 0) {
                    *reinterpret_cast<volatile uint32_t*>(&sh.moves[x][step_cnt & 1u]) = step_cnt;
                }
                ok = meet();
                if (!ok) break;
                PH_MARK(4);
                if (__builtin_expect(*reinterpret_cast<volatile uint32_t*>(&sh.moves[x][step_cnt & 1u]) == step_cnt, 0)) {
                    // The rows' maxima over the block: ordered as integers, for which a warp has a reduction.
#pragma unroll
                    for (int c = 0; c < R; ++c) {
                        const float score = B == 2 ? fmaxf(y[c].x, y[c].y) : c & 1 ? y[c / 2].y : y[c / 2].x;
                        const int bits = __float_as_int(fmaxf(score, -INFINITY));      // NaN has no say
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
                    for (int c0 = 0; c0 < R; c0 += 8) {
                        float factor[8];
                        uint32_t o[8];
                        if (!first) {
                            few_ld<8>(o_tmem + x * N + c0, o);
                            tmem_wait_ld();
                        }
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            const int c = c0 + e;
                            factor[e] = 1.f;
                            if (c >= R) continue;
                            const float m = fmaxf(fmaxf(sh.top[x][0][c], sh.top[x][1][c]), fmaxf(sh.top[x][2][c], sh.top[x][3][c]));
                            const bool none = sh.none[x][c] != 0u;           // then sum and O are 0
                            if (!none && m + sh.minus_ref[x][c] > kP8Most) factor[e] = fast_exp2(kP8At - m - sh.minus_ref[x][c]);
                            open |= c < rows && none && m == -INFINITY;
                            sum[c] *= factor[e];
                        }
                        if (!first) {
#pragma unroll
                            for (int e = 0; e < 8; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * factor[e]);
                            tmem_st_x8(o_tmem + x * N + c0, o);
                        }
                    }
                    if (!first) tmem_wait_st();
                    ok = meet();                 // all have read the old references
                    if (!ok) break;
                    if (r < rows) {
                        const float m = fmaxf(fmaxf(sh.top[x][0][r], sh.top[x][1][r]), fmaxf(sh.top[x][2][r], sh.top[x][3][r]));
                        if (sh.none[x][r] != 0u ? m != -INFINITY : m + sh.minus_ref[x][r] > kP8Most) {
                            sh.minus_ref[x][r] = kP8At - m;
                            sh.none[x][r] = 0u;
                        }
                    }
                    ok = meet();
                    if (!ok) break;
                }
                PH_MARK(7);
                ok = wait_pv();                  // P^T of the step before has been read
                if (!ok) break;
                PH_MARK(9);
                const float* v_scale = &sh.scales.scale[scale_slot][1][r >> 4];
                const float2 part = make_float2(1.f / v_scale_of(v_scale[0]), 1.f / v_scale_of(v_scale[(B - 1) * 8]));
#pragma unroll
                for (int c = 0; c < R; c += 4) {
                    const float4 m4 = minus_ref[c / 4];
#pragma unroll
                    for (int e = 0; e < kFour; ++e) {
                        const float2 up = add2(y[c / 4 * kFour + e], few8_rows<B>(m4, e));
                        const float2 prob = make_float2(fast_exp2(up.x), fast_exp2(up.y));
                        const int row = B == 2 ? c + e : c + 2 * (e & 1), other = B == 2 ? row : row + 1;
                        if constexpr (B == 2) {
                            sum[row] = fmaf(prob.x, part.x, fmaf(prob.y, part.y, sum[row]));
                        } else {
                            sum[row] = fmaf(prob.x, part.x, sum[row]);
                            sum[other] = fmaf(prob.y, part.y, sum[other]);
                        }
                        const uint32_t to = p_at[row & 7] + (row >> 3) * 1024;
                        const uint32_t to_other = p_at[other & 7] + (other >> 3) * 1024 + (B - 1) * N * 256;
                        asm volatile("{\n\t.reg .b16 l, u;\n\tmov.b32 {l, u}, %2;\n\tst.shared.b16 [%0], l;\n\tst.shared.b16 [%1], u;\n\t}"
                                     ::"r"(to), "r"(to_other), "r"(pack_half2(prob.x, prob.y)) : "memory");
                    }
                }
                fence_proxy_async_smem();
                tc_fence_before_sync();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(smem_u32(&sh.p_full[x]));
                    mbar_arrive(smem_u32(&sh.scales.empty[scale_slot]));
                }
                PH_MARK(5);
            }
            if (!ok) break;
            k_base += (w.blocks + B - 1) / B;
            if (w.blocks > x * B) {
                ok = warp_wait8(wctx, smem_u32(&sh.pv_done[x]), pv_cnt & 1u, 15);
                if (!ok) break;
                ++pv_cnt;
                tc_fence_after_sync();
            }

            // The warpgroup's sums, and then both warpgroups' parts: O = a0 O0 + a1 O1, eight rows at a time.
            few_column_sums<R>(sum, lane);
            ok = meet();                         // nobody still reads maxima
            if (!ok) break;
            if (lane < R) sh.top[x][quarter][lane] = sum[0];
            ok = meet();
            if (!ok) break;
            if (r < R) {
                const float ref = w.blocks <= x * B || sh.none[x][r] != 0u ? -INFINITY : -sh.minus_ref[x][r];
                sh.stat[x][r] = make_float2(ref, (sh.top[x][0][r] + sh.top[x][1][r]) + (sh.top[x][2][r] + sh.top[x][3][r]));
            }
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(smem_u32(&sh.q_empty[buf]));
                mbar_arrive(smem_u32(&sh.both_done));
            }
            ok = warp_wait8(wctx, smem_u32(&sh.both_done), both_cnt & 1u, 16);
            if (!ok) break;
            tc_fence_after_sync();
            const bool not_finite = *reinterpret_cast<volatile uint32_t*>(&sh.not_finite[at]) == it + 1;
            const bool whole = w.part < 0;
            const bool second = w.blocks > B;
            // A thread a row for what it needs once; the sums' places take the two parts' factors.
            if (r < rows) {
                const float2 s0 = sh.stat[0][r], s1 = sh.stat[1][r];
                const float ref = fmaxf(s0.x, s1.x);
                float a0 = s0.x == ref ? 1.f : fast_exp2(s0.x - ref);
                float a1 = s1.x == ref ? 1.f : fast_exp2(s1.x - ref);
                const float l = s0.y * a0 + s1.y * a1;
                if (whole) {
                    // A sum of 0: the row sees nothing (or only what is -inf).  NaN stays NaN.  The sum of weights, each at
                    // most 2^15 over a scale, is far below the 2^126 that the fast division wants.
                    const float inv = l == 0.f ? 0.f : __fdividef(1.f, l);
                    a0 *= inv;
                    a1 *= inv;
                    if (x == 0) {
                        p.lse[w.seq * p.lse_seq_stride + w.head * p.c.group * p.lse_head_stride +
                              (p.c.cu_seqlens_q == nullptr ? 0 : w.q_begin) + sh.lse_at[r]] =
                            l == 0.f ? -INFINITY : (ref + fast_log2(l)) * kLn2;
                    }
                } else if (x == 0) {
                    p.part_stat[static_cast<long long>(w.part) * p.part_rows + r] = make_float2(ref, l);
                }
                sh.top[x][0][r] = a0;
                sh.top[x][1][r] = a1;
            }
            ok = meet();
            if (!ok) break;
            // Four rows at a time: this runs once a piece, and all its code comes from L2.
            __nv_bfloat16* const out = p.out + (static_cast<long long>(w.q_begin) * p.c.heads_q + w.head * p.c.group) * kHeadDim + r;
            float* const part = reinterpret_cast<float*>(p.part_o) + static_cast<long long>(w.part) * p.part_rows * kHeadDim + r;
#pragma unroll 1
            for (int c0 = 4 * x; c0 < rows; c0 += 8) {
                uint32_t o0[4], o1[4] = {0u, 0u, 0u, 0u};
                few_ld<4>(o_tmem + c0, o0);
                if (second) few_ld<4>(o_tmem + N + c0, o1);
                tmem_wait_ld();
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int row = c0 + e;
                    if (row >= rows) break;
                    float o = __uint_as_float(o0[e]) * sh.top[x][0][row];
                    if (second) o = fmaf(__uint_as_float(o1[e]), sh.top[x][1][row], o);
                    if (not_finite && few8_sees_nan(p, w, row / p.c.group, r)) o = NAN;
                    if (whole) {
                        out[static_cast<long long>(sh.out_at[row]) * kHeadDim] = __float2bfloat16_rn(o);
                    } else {
                        part[row * kHeadDim] = o;
                    }
                }
            }
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&sh.both_read));
            ok = warp_wait8(wctx, smem_u32(&sh.both_read), both_cnt & 1u, 17);
            ++both_cnt;
            if (!ok) break;
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&sh.piece_empty[at]));
            PH_MARK(8);
        }
        PH_PRINT("few8 softmax", 10);
    }

    tc_fence_before_sync();
    __syncthreads();
    if (warp == kFew8QkWarp) {
        tc_fence_after_sync();
        tmem_dealloc(tmem_base, Shared::kTmem);
    }
}

template <int R>
int set_few8_smem() {
    B2A_CUDA_OK(cudaFuncSetAttribute(tree8_attention_few<R>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     static_cast<int>(few8_smem_bytes<R>())));
    return B2A_OK;
}

template <int R>
int launch_few8(const CUtensorMap& map_k, const CUtensorMap& map_v, const Tree8Params& p, int ctas, const DeviceInfo& dev, int slot,
                cudaStream_t stream) {
    const int rc = once_per_device(dev.device, slot, set_few8_smem<R>);
    if (rc != B2A_OK) return rc;
    auto attention = tree8_attention_few<R>;
    B2A_CUDA_OK(launch_early(attention, ctas, kFew8Threads, few8_smem_bytes<R>(), stream, map_k, map_v, p));
    return B2A_OK;
}

}  // namespace

int launch_tree8_few(const CUtensorMap& map_k, const CUtensorMap& map_v, const Tree8Params& p, int ctas, const DeviceInfo& dev,
                     cudaStream_t stream) {
    const int rows = p.t.part_rows;
    // 4 rows, 16 sequences of up to 8,001 slots, with 8, 16 and 32: 43.7, 51.0, 75.3 us; one of 131,072: 59.8, 65.1, 97.8.
    const int rc = rows <= 8    ? launch_few8<8>(map_k, map_v, p, ctas, dev, 14, stream)
                   : rows <= 16 ? launch_few8<16>(map_k, map_v, p, ctas, dev, 21, stream)
                                : launch_few8<32>(map_k, map_v, p, ctas, dev, 22, stream);
    return rc != B2A_OK || ctas == 1 ? rc : launch_tree_combine_few(p.t, ctas, stream);
}

}  // namespace b2a
