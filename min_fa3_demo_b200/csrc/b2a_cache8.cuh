// A cache of e4m3 values with a scale for each block of slots and K/V head, as the kernels see it, and products with it.
//
// K Q^T is a product of 8-bit operands: K's tiles go from global memory to shared memory by TMA and from there into the product, and are
// never converted.  Q has to have 8 bits too, and e4m3 has only four significant ones, so Q is the sum of two such
// numbers, which take part one after the other in the same accumulator: a bf16 rounded to e4m3 leaves a signed rest of four
// bits, which e4m3 holds exactly.  A row is scaled so that its largest value lies in [2^7, 2^8); rests of values below 2^-2 are rounded
// to a multiple of 2^-9, so they are off by 2^-10 at most, 2^-17 of that value.  Twice the products at twice the rate of bf16.
//
// P V is a product of f16: e4m3 is exact in f16, and warps of their own convert V's tiles (16 KiB in, 32 KiB out, an instruction for
// two values): four, or one where two tiles of rows give it the time.  P in f16 is off by 2^-11 of itself, or by 2^-25 where it is
// small, 2^-27 of a row's largest or less.  P as a sum of two 8-bit numbers, as Q is, needs no conversion of V but six instructions for
// two probabilities instead of one, which the softmax has no time for (trees of 64 tokens, 64 heads over 8, 8 sequences of up to
// 16,000 slots: 344 us).
//
// Scales never meet the values: K's multiplies a score, V's is an addend of the exponent, by which P takes it into the
// product, and what goes into the row's sum is divided by it again.
#pragma once

#include "b2a_tree.cuh"

namespace b2a {

constexpr uint32_t kTile8Bytes = kTileM * kHeadDim;      // 16 KiB: 128 slots of 128 bytes
// V's scales are taken within these bounds, so that sums of probabilities divided by them stay in range.
constexpr float kScaleLeast = 5.421010862427522e-20f, kScaleMost = 18446744073709551616.f;      // 2^-64, 2^64

// Strides in elements.
struct CacheScales {
    float* k;
    float* v;
    long long k_stride[3];       // page, block, head
    long long v_stride[3];
    int shift;                   // log2 of a block's slots
    __device__ __forceinline__ long long at(const long long (&stride)[3], int page, int row, int head) const {
        return page * stride[0] + (row >> shift) * stride[1] + head * stride[2];
    }
};

inline int make_cache_scales(const b2a_cache_scales& s, const b2a_cache& c, CacheScales* out) {
    B2A_REQUIRE(s.k != nullptr && s.v != nullptr, "the scales of the cache must not be NULL");
    B2A_REQUIRE(s.block == 16 || s.block == 32 || s.block == 64 || s.block == 128, "a scale must have 16, 32, 64 or 128 slots, got %d",
                s.block);
    B2A_REQUIRE(c.block_table == nullptr || c.page_size % s.block == 0,
                "page_size must be a multiple of a scale's slots, got %d and %d", c.page_size, s.block);
    for (int i = 0; i < 3; ++i) {
        B2A_REQUIRE(s.k_stride[i] >= 0 && s.v_stride[i] >= 0, "strides of the scales must not be negative");
        B2A_REQUIRE(c.k_stride[i] % 16 == 0 && c.v_stride[i] % 16 == 0, "strides of a cache in 8 bits must be multiples of 16 elements");
        out->k_stride[i] = s.k_stride[i];
        out->v_stride[i] = s.v_stride[i];
    }
    out->k = s.k;
    out->v = s.v;
    out->shift = 0;
    while ((1 << out->shift) < s.block) ++out->shift;
    return B2A_OK;
}

inline int make_slot_map8(CUtensorMap* map, const CacheView& c, bool keys, int box_rows) {
    const uint64_t sizes[3] = {static_cast<uint64_t>(c.pages), static_cast<uint64_t>(c.page_size), static_cast<uint64_t>(c.heads)};
    const long long* st = keys ? c.k_stride : c.v_stride;
    const int64_t strides[3] = {st[0], st[1], st[2]};
    return make_strided_map8(map, keys ? c.k : c.v, 4, sizes, strides, 1, static_cast<uint32_t>(box_rows));
}

// As SlotLoader::load, rows of 128 bytes.
__device__ __forceinline__ void load_slots8(const SlotLoader& at, const CUtensorMap* map, uint32_t dst, uint32_t bar, int head, int n,
                                            int lane) {
    if (lane == 0) mbar_arrive_expect_tx(bar, static_cast<uint32_t>(n << at.shift) * 128u);
    __syncwarp();
    if (lane < n) tma_load_4d(dst + static_cast<uint32_t>(lane << at.shift) * 128u, map, bar, 0, head, at.row, at.page);
    __syncwarp();
}

// mbar_wait with little code at each wait: the roles of these kernels run different code at the same time, and with mbar_wait's loop
// everywhere it is more than the instruction cache holds (one token, 16 sequences of up to 8,001 slots: a third of the
// requests missed, and the kernel took twice the time).  The loop that looks at the clock is a function, which a caller
// with many live registers should hardly ever need to call.
static __device__ __noinline__ bool wait8_longer(uint32_t abort_smem, unsigned int* status, uint32_t timeout_ns, uint32_t bar, uint32_t parity,
                                                 uint32_t tag) {
    return mbar_wait(WaitCtx{abort_smem, status, timeout_ns, 1u}, bar, parity, tag);
}

constexpr int kWait8Polls = 1024;

__device__ __forceinline__ bool wait8(const WaitCtx& ctx, uint32_t bar, uint32_t parity, uint32_t tag) {
#pragma unroll 1
    for (int i = 0; i < kWait8Polls; ++i) {
        if (mbar_try_wait(bar, parity)) return true;
    }
    return wait8_longer(ctx.abort_smem, ctx.status, ctx.timeout_ns, bar, parity, tag);
}

// As warp_wait: one answer for all lanes.
__device__ __forceinline__ bool warp_wait8(const WaitCtx& ctx, uint32_t bar, uint32_t parity, uint32_t tag) {
#pragma unroll 1
    for (int i = 0; i < kWait8Polls; ++i) {
        if (__all_sync(0xFFFFFFFFu, mbar_try_wait(bar, parity))) return true;
    }
    return __all_sync(0xFFFFFFFFu, wait8_longer(ctx.abort_smem, ctx.status, ctx.timeout_ns, bar, parity, tag));
}

// The scales of the steps under way, kBlocks blocks each: one of K and one of V for 16 slots.  The warp that loads K asks for them, as it
// has the pages at hand, and copies them without waiting; the softmax warps take them from shared memory, where they
// cost no registers while they are on their way.
constexpr int kScaleSlots = 8;

template <int kBlocks>
struct ScaleRing {
    float scale[kScaleSlots][2][8 * kBlocks];
    uint64_t full[kScaleSlots], empty[kScaleSlots];

    // consumers: arrivals that give a slot back.
    __device__ __forceinline__ void init(int consumers) {
        for (int i = 0; i < kScaleSlots; ++i) {
            mbar_init(smem_u32(&full[i]), 32);
            mbar_init(smem_u32(&empty[i]), consumers);
        }
    }
    // By a warp, of the blocks from `block` on, which `at` has looked up.  What does not exist is zero, and masked.
    __device__ __forceinline__ bool load(const WaitCtx& wctx, uint32_t it, const CacheView& c, const CacheScales& s, const SlotLoader& at,
                                         int block, int slots, int head, int lane) {
        constexpr int kGroups = 8 * kBlocks;
        const uint32_t slot = it % kScaleSlots;
        const int group = lane % kGroups, box = (group * 16) >> at.shift;
        const bool keys = lane < kGroups;
        const int page = __shfl_sync(0xFFFFFFFFu, at.page, box);
        const int row = __shfl_sync(0xFFFFFFFFu, at.row, box) + ((group * 16) & ((1 << at.shift) - 1));
        if (!warp_wait8(wctx, smem_u32(&empty[slot]), ((it / kScaleSlots) & 1u) ^ 1u, 20)) return false;
        if (lane < 2 * kGroups) {
            const bool there = block * kSlotBlock + group * 16 < slots && static_cast<unsigned>(page) < static_cast<unsigned>(c.pages);
            const float* from = keys ? s.k : s.v;
            if (there) from += s.at(keys ? s.k_stride : s.v_stride, page, row, head);
            const uint32_t to = smem_u32(&scale[slot][keys ? 0 : 1][group]);
            asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to), "l"(from), "r"(there ? 4 : 0) : "memory");
        }
        asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(&full[slot])) : "memory");
        __syncwarp();
        return true;
    }
};

// ---------------------------------------------------------------------------------------
// Numbers as sums of two of 8 bits
// ---------------------------------------------------------------------------------------
// The first of a pair in the low byte.
__device__ __forceinline__ uint32_t pack_e4m3x2(float lo, float hi) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}

__device__ __forceinline__ uint32_t e4m3x2_to_half2(uint32_t two) {
    uint32_t r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(static_cast<uint16_t>(two)));
    return r;
}

__device__ __forceinline__ void e4m3x4_to_half4(uint32_t four, uint32_t& lo, uint32_t& hi) {
    asm("{\n\t.reg .b16 l, u;\n\tmov.b32 {l, u}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, u;\n\t}"
        : "=r"(lo), "=r"(hi)
        : "r"(four));
}

__device__ __forceinline__ float2 half2_to_float2(uint32_t h) {
    float2 f;
    asm("{\n\t.reg .b16 l, u;\n\tmov.b32 {l, u}, %2;\n\tcvt.f32.f16 %0, l;\n\tcvt.f32.f16 %1, u;\n\t}" : "=f"(f.x), "=f"(f.y) : "r"(h));
    return f;
}

__device__ __forceinline__ float2 e4m3x2_to_float2(uint32_t two) { return half2_to_float2(e4m3x2_to_half2(two)); }

__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

// Rows of Q by a warp into [rows][128 bytes] of both parts, 16-byte chunks exchanged by the row's number: half a warp a row, a lane has
// the eight dimensions from (lane & 15) * 8 on.  What a row has been divided by goes to `scale`.  `there`: the lane's row exists (the
// whole warp calls).  In f16, which holds the eight bits of a bf16 and the difference of the two.
__device__ __forceinline__ void split_q_rows(const uint4& q, bool there, int row, int lane, uint8_t* first, uint8_t* rest, float* scale) {
    const uint32_t words[4] = {q.x, q.y, q.z, q.w};
    uint32_t most = 0;      // two magnitudes
#pragma unroll
    for (int i = 0; i < 4; ++i) most = __vmaxu2(most, words[i] & 0x7FFF7FFFu);
#pragma unroll
    for (int d = 8; d > 0; d >>= 1) most = __vmaxu2(most, __shfl_xor_sync(0xFFFFFFFFu, most, d));
    most = max(most & 0xFFFFu, most >> 16);
    // Exponent field e of the largest value: times 2^(134 - e).  A row of zeros keeps its own.  A row with infinities or NaN, whose
    // scores with anything are NaN as well, becomes NaN whole.
    const int up = most == 0u ? 0 : min(134 - static_cast<int>(most >> 7), 126);
    const float mul = most >= 0x7F80u ? NAN : __int_as_float((127 + up) << 23);
    uint32_t a[2], b[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        uint32_t part[2], left[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const uint32_t w = words[2 * i + e];
            const uint32_t x = pack_half2(__uint_as_float(w << 16) * mul, __uint_as_float(w & 0xFFFF0000u) * mul);
            uint16_t u, v;
            uint32_t d;
            asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(u) : "r"(x));
            asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(x), "r"(e4m3x2_to_half2(u)));
            asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(v) : "r"(d));
            part[e] = u;
            left[e] = v;
        }
        a[i] = part[0] | part[1] << 16;
        b[i] = left[0] | left[1] << 16;
    }
    if (there) {
        const int at = row * 128 + ((((lane & 15) >> 1) ^ (row & 7)) << 4) + (lane & 1) * 8;
        *reinterpret_cast<uint2*>(first + at) = make_uint2(a[0], a[1]);
        *reinterpret_cast<uint2*>(rest + at) = make_uint2(b[0], b[1]);
        if ((lane & 15) == 0) *scale = __int_as_float((127 - up) << 23);
    }
}

// ---------------------------------------------------------------------------------------
// Products of 8-bit operands
// ---------------------------------------------------------------------------------------
// Instruction descriptor with D in f32 and both operands in the kind's first format: e4m3 (kind::f8f6f4) or f16 (kind::f16).
__host__ __device__ constexpr uint32_t make_idesc_first(int m, int n, int a_mn_major, int b_mn_major) {
    return (1u << 4) | (static_cast<uint32_t>(a_mn_major) << 15) | (static_cast<uint32_t>(b_mn_major) << 16) |
           (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}

// The four k-steps of a product over 128, 32 bytes each along the rows of A and B, as umma_ss_kk_x8_w.
__device__ __forceinline__ void umma8_ss_x4_w(uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t"
        ".reg .pred p, pe, pt;\n\t"
        ".reg .b64 da, db;\n\t"
        ".reg .b32 ra, rb;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "setp.eq.b32 pt, 0, 0;\n\t"
        "elect.sync _|pe, 0xFFFFFFFF;\n\t"
        "mov.b64 da, {%1, %5};\n\t"
        "mov.b64 db, {%2, %5};\n\t"
        "@pe tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], da, db, %3, p;\n\t"
        "add.u32 ra, %1, 2;\n\t"
        "add.u32 rb, %2, 2;\n\t"
        "mov.b64 da, {ra, %5};\n\t"
        "mov.b64 db, {rb, %5};\n\t"
        "@pe tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], da, db, %3, pt;\n\t"
        "add.u32 ra, ra, 2;\n\t"
        "add.u32 rb, rb, 2;\n\t"
        "mov.b64 da, {ra, %5};\n\t"
        "mov.b64 db, {rb, %5};\n\t"
        "@pe tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], da, db, %3, pt;\n\t"
        "add.u32 ra, ra, 2;\n\t"
        "add.u32 rb, rb, 2;\n\t"
        "mov.b64 da, {ra, %5};\n\t"
        "mov.b64 db, {rb, %5};\n\t"
        "@pe tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], da, db, %3, pt;\n\t"
        "}\n"
        ::"r"(d_tmem), "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(accumulate), "r"(kDescHiSw128)
        : "memory");
}

// The eight k-steps of a product of f16 over 128, A across two halves of 64 columns, B with two halves of N rows of 128 bytes.
template <int N>
__device__ __forceinline__ void umma_ss_nk_x8_w(uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t"
        ".reg .pred p, pe, pt;\n\t"
        ".reg .b64 da, db;\n\t"
        ".reg .b32 ra, rb;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "setp.eq.b32 pt, 0, 0;\n\t"
        "elect.sync _|pe, 0xFFFFFFFF;\n\t"
        "mov.b64 da, {%1, %5};\n\t"
        "mov.b64 db, {%2, %5};\n\t"
        "@pe tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n\t"
        "add.u32 ra, %1, 128;\n\t"
        "add.u32 rb, %2, 2;\n\t"
        "mov.b64 da, {ra, %5};\n\t"
        "mov.b64 db, {rb, %5};\n\t"
        "@pe tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, pt;\n\t"
        "add.u32 ra, %1, 256;\n\t"
        "add.u32 rb, %2, 4;\n\t"
        "mov.b64 da, {ra, %5};\n\t"
        "mov.b64 db, {rb, %5};\n\t"
        "@pe tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, pt;\n\t"
        "add.u32 ra, %1, 384;\n\t"
        "add.u32 rb, %2, 6;\n\t"
        "mov.b64 da, {ra, %5};\n\t"
        "mov.b64 db, {rb, %5};\n\t"
        "@pe tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, pt;\n\t"
        "add.u32 ra, %1, 512;\n\t"
        "add.u32 rb, %2, %6;\n\t"
        "mov.b64 da, {ra, %5};\n\t"
        "mov.b64 db, {rb, %5};\n\t"
        "@pe tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, pt;\n\t"
        "add.u32 ra, %1, 640;\n\t"
        "add.u32 rb, rb, 2;\n\t"
        "mov.b64 da, {ra, %5};\n\t"
        "mov.b64 db, {rb, %5};\n\t"
        "@pe tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, pt;\n\t"
        "add.u32 ra, %1, 768;\n\t"
        "add.u32 rb, rb, 2;\n\t"
        "mov.b64 da, {ra, %5};\n\t"
        "mov.b64 db, {rb, %5};\n\t"
        "@pe tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, pt;\n\t"
        "add.u32 ra, %1, 896;\n\t"
        "add.u32 rb, rb, 2;\n\t"
        "mov.b64 da, {ra, %5};\n\t"
        "mov.b64 db, {rb, %5};\n\t"
        "@pe tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, pt;\n\t"
        "}\n"
        ::"r"(d_tmem), "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(accumulate), "r"(kDescHiSw128), "n"(N * 128 >> 4)
        : "memory");
}

// ---------------------------------------------------------------------------------------
// What the kernels of b2a_tree8_fwd share
// ---------------------------------------------------------------------------------------
struct Tree8Params {
    TreeParams t;
    CacheScales scales;
    const __nv_bfloat16* q;
    long long q_stride[2];       // token, head
};

// Probabilities, with V's scale, are at most 2^15; a new reference puts the score that it is taken from at 2^2, so that it moves only when
// the maximum has grown by a factor of 2^13.
constexpr float kP8Most = 15.f, kP8At = 2.f;

__device__ __forceinline__ bool e4m3_not_finite(uint32_t byte) { return (byte & 0x7Fu) == 0x7Fu; }

__device__ __forceinline__ uint4 ld_shared_v4(uint32_t at) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
    return v;
}

__device__ __forceinline__ void st_shared_v4(uint32_t at, const uint4& v) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

// As tree_clean_row, for a row of 128 bytes, whose only values that are not finite are NaN.  Little code, as few rows need it.
static __device__ __noinline__ bool tree8_clean_row(uint8_t* row, int r, bool behind) {
    // A magnitude of 0x7F plus one carries into its byte's sign bit, and no other does.
    auto ones = [](uint32_t w) { return ((w & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u; };
    uint32_t any = 0;
#pragma unroll 1
    for (int c = 0; c < 8; ++c) {
        // Another chunk first in each row, so that rows of 128 bytes do not meet in the same banks.
        uint4* chunk = reinterpret_cast<uint4*>(row + ((c + r) & 7) * 16);
        uint4 v = behind ? make_uint4(0u, 0u, 0u, 0u) : *chunk;
        const uint4 n = make_uint4(ones(v.x), ones(v.y), ones(v.z), ones(v.w));
        any |= n.x | n.y | n.z | n.w;
        v = make_uint4(v.x & ~((n.x >> 7) * 0xFFu), v.y & ~((n.y >> 7) * 0xFFu), v.z & ~((n.z >> 7) * 0xFFu), v.w & ~((n.w >> 7) * 0xFFu));
        if (behind || (n.x | n.y | n.z | n.w) != 0u) *chunk = v;
    }
    return any != 0u;
}

// V's tiles from e4m3 to f16 by kWarps warps, r being the thread's number among them, a row at a time.  What a product must not see
// is left out on the way: rows behind the last slot, and of drafted tokens NaN, since 0 * NaN is NaN (e4m3 has no infinities); that
// there was one is noted for the piece.
// begin(piece, number): what there is to do before a piece's blocks.
template <int kWarps, int kSlots, int kStages, int kTiles, typename Shared, typename Begin>
__device__ __forceinline__ void tree8_convert_v(const TreeParams& p, Shared& sh, const WaitCtx& wctx, int r, Begin begin) {
    uint32_t v_it = 0;
    bool ok = true;
    PH_DECL(4)   // 0 other, 1 wait for V, 2 wait for a tile, 3 convert
    for (uint32_t it = 0; ok; ++it) {
        const uint32_t at = it % kSlots;
        ok = warp_wait8(wctx, smem_u32(&sh.piece_full[at]), (it / kSlots) & 1u, 22);
        if (!ok) break;
        const TreePiece& piece = sh.piece[at];
        const int valid = piece.valid, j0 = piece.j0, slots = piece.slots, blocks = piece.blocks;
        const int len = piece.n > 1 || p.c.mask != nullptr ? piece.len : slots;      // from here on tokens that not all rows see
        ok = !valid || begin(piece, it);
        __syncwarp();
        if ((r & 31) == 0) mbar_arrive(smem_u32(&sh.piece_empty[at]));
        if (!valid || !ok) break;
        for (int i = 0; i < blocks; ++i, ++v_it) {
            const uint32_t stage = v_it % kStages, tile = v_it % kTiles;
            PH_MARK(0);
            ok = warp_wait8(wctx, smem_u32(&sh.v_full[stage]), (v_it / kStages) & 1u, 23);
            if (!ok) break;
            PH_MARK(1);
            ok = warp_wait8(wctx, smem_u32(&sh.v16_empty[tile]), ((v_it / kTiles) & 1u) ^ 1u, 24);
            if (!ok) break;
            PH_MARK(2);
#pragma unroll 1
            for (int row = r; row < kSlotBlock; row += 32 * kWarps) {
                const int slot = (j0 + i) * kSlotBlock + row;
                if (slot >= len && tree8_clean_row(&sh.v[stage][row * 128], row, slot >= slots)) {
                    *reinterpret_cast<volatile uint32_t*>(&sh.not_finite[at]) = it + 1;
                }
                // 16 values: chunks 2 c and 2 c + 1 of 8, which lie in a half of 64 columns.  Rows begin at multiples of 128 bytes, so chunks
                // are exchanged by an exclusive or of the address.
                const uint32_t from = smem_u32(&sh.v[stage][row * 128]) + (row & 7) * 16;
                const uint32_t to = smem_u32(&sh.v16[tile][row * 128]) + (row & 7) * 16;
#pragma unroll 1
                for (int half = 0; half < 2; ++half) {
#pragma unroll
                    for (int c = 0; c < 4; c += 2) {
                        uint4 v[2];
#pragma unroll
                        for (int e = 0; e < 2; ++e) v[e] = ld_shared_v4((from ^ (half * 64)) ^ ((c + e) * 16));
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            uint4 x, y;
                            e4m3x4_to_half4(v[e].x, x.x, x.y);
                            e4m3x4_to_half4(v[e].y, x.z, x.w);
                            e4m3x4_to_half4(v[e].z, y.x, y.y);
                            e4m3x4_to_half4(v[e].w, y.z, y.w);
                            const uint32_t there = to + half * kHalfTileBytes;
                            st_shared_v4(there ^ ((c + e) * 32), x);
                            st_shared_v4(there ^ ((c + e) * 32 + 16), y);
                        }
                    }
                }
            }
            fence_proxy_async_smem();
            __syncwarp();
            if ((r & 31) == 0) {
                mbar_arrive(smem_u32(&sh.v_empty[stage]));
                mbar_arrive(smem_u32(&sh.v16_full[tile]));
            }
            PH_MARK(3);
        }
    }
    PH_PRINT("tree8 convert", 4);
}

// Loads of V by one warp, as tree_load_v.
template <int kSlots, int kStages, typename Shared>
__device__ __forceinline__ void tree8_load_v(const TreeParams& p, Shared& sh, const CUtensorMap* map, const WaitCtx& wctx, int lane) {
    SlotLoader loader(p.box_rows);
    uint32_t v_it = 0;
    bool ok = true;
    for (uint32_t it = 0; ok; ++it) {
        const uint32_t at = it % kSlots;
        ok = warp_wait8(wctx, smem_u32(&sh.piece_full[at]), (it / kSlots) & 1u, 4);
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
            ok = warp_wait8(wctx, smem_u32(&sh.v_empty[stage]), ((v_it / kStages) & 1u) ^ 1u, 18);
            if (!ok) break;
            load_slots8(now, map, smem_u32(&sh.v[stage][0]), smem_u32(&sh.v_full[stage]), w.head, boxes, lane);
        }
    }
}

// Values of drafted tokens that are NaN, given to a row that sees them: columns [column, column + 32) of O.
__device__ __forceinline__ void tree8_add_not_finite(const TreeParams& p, const TreePiece& w, int token, int column, uint32_t (&t)[32]) {
    const int from = max(0, w.j0 * kSlotBlock - w.len), to = min(w.n, (w.j0 + w.blocks) * kSlotBlock - w.len);
#pragma unroll 1
    for (int u = from; u < to; ++u) {
        const long long slot = static_cast<long long>(w.len) + u;
        if (slot >= w.slots || !tree_sees(p, w, token, u)) continue;
        int row;
        const int page = p.c.cache.page_of(w.seq, slot, &row);
        if (page < 0) continue;
        const uint8_t* v = reinterpret_cast<const uint8_t*>(p.c.cache.v) + p.c.cache.at(p.c.cache.v_stride, page, row, w.head) + column;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint4 chunk = reinterpret_cast<const uint4*>(v)[i];
            const uint32_t words[4] = {chunk.x, chunk.y, chunk.z, chunk.w};
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                if (e4m3_not_finite(words[e >> 2] >> (e & 3) * 8)) t[i * 16 + e] = 0x7FFFFFFFu;
            }
        }
    }
}

// b2a_tree8_one.cu: calls of more rows an item, but no more than a tile's 128; b2a_tree8_few.cu: of at most kFewRows, which is as
// many as it takes.  Us of the latter and the former, 8 K/V heads, sequences x slots:
//              1 x 16,384     64 x 2,048      16 x 16,384     4 x 400        32 x 1,000
//    4 rows    19.5  30.4     66.4  128.1     104.8  198.8    13.0  16.8     29.1  42.9
//    9         21.2  32.0     78.0  132.0     107.6  199.8    14.4  17.7     33.3  44.3
//   16         21.6  33.0     78.6  135.1     108.3  201.3    14.7  18.3     33.7  46.8
//   17         24.7  33.8    111.9  136.7     160.1  201.6    16.5  18.4     40.4  47.3
//   24         25.0  33.4    113.4  136.1     160.9  201.5    16.8  18.6     41.1  47.3
//   32         26.0  34.0    115.6  136.4     162.0  202.1    17.0  19.0     42.9  47.9
int launch_tree8_one(const CUtensorMap& map_k, const CUtensorMap& map_v, const Tree8Params& p, int ctas, const DeviceInfo& dev,
                     cudaStream_t stream);
int launch_tree8_few(const CUtensorMap& map_k, const CUtensorMap& map_v, const Tree8Params& p, int ctas, const DeviceInfo& dev,
                     cudaStream_t stream);

}  // namespace b2a
