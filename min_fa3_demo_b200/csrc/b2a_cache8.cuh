// A cache of e4m3 values with a scale for each block of slots and K/V head, as the kernels see it, and products with it.
//
// The tensor cores multiply 8-bit operands as they lie in memory, so K and V are never converted: a tile goes from global memory
// to shared memory by TMA and from there into the product.  What is multiplied by them has to have 8 bits too, and e4m3 has only
// four significant bits.  So Q and P are sums of two such numbers, of which each takes part in the product with the same
// accumulator: the value rounded to e4m3, and what is left over.
//   Q: bf16 has eight significant bits; the first four, rounded, leave a signed rest of four, which e4m3 holds exactly.  A row is
//      scaled so that its largest value lies in [2^7, 2^8); rests below 2^-9 lose bits, which is 2^-18 of that value.
//   P: the rest is rounded to e5m2, whose exponents reach to 2^-16: P is off by 2^-7 of itself at most, 0.0013 in the mean
//      square (bf16: 2^-8 and 0.0016), and by 2^-17 where it is small, 2^-22 of a row's largest or less.
// Twice the products at twice the rate of bf16.  Scales never meet the values: K's multiplies a score, V's is an addend of the
// exponent, by which P takes it into the product, and the row's sum is divided by it again.
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
    B2A_REQUIRE(s.block >= 16 && (s.block & (s.block - 1)) == 0, "slots of a scale must be a power of two, 16 or more, got %d", s.block);
    B2A_REQUIRE(c.block_table == nullptr || c.page_size % s.block == 0, "page_size must be a multiple of a scale's slots, got %d and %d",
                c.page_size, s.block);
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
__device__ __forceinline__ void load_slots8(const SlotLoader& at, const CUtensorMap* map, uint32_t dst, uint32_t bar, int head, int n, int lane) {
    if (lane == 0) mbar_arrive_expect_tx(bar, static_cast<uint32_t>(n << at.shift) * 128u);
    __syncwarp();
    if (lane < n) tma_load_4d(dst + static_cast<uint32_t>(lane << at.shift) * 128u, map, bar, 0, head, at.row, at.page);
    __syncwarp();
}

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

__device__ __forceinline__ float2 half2_to_float2(uint32_t h) {
    float2 f;
    asm("{\n\t.reg .b16 l, u;\n\tmov.b32 {l, u}, %2;\n\tcvt.f32.f16 %0, l;\n\tcvt.f32.f16 %1, u;\n\t}" : "=f"(f.x), "=f"(f.y) : "r"(h));
    return f;
}

__device__ __forceinline__ float2 e4m3x2_to_float2(uint32_t two) { return half2_to_float2(e4m3x2_to_half2(two)); }

// Two probabilities of at most 2^8: e4m3, and e5m2 of the rest.  f16 has 11 bits, so the difference is that of p rounded
// to them, which is what is left of it after the two.
__device__ __forceinline__ void split_p(float p0, float p1, uint32_t& first, uint32_t& rest) {
    uint32_t p;
    uint16_t r;
    first = pack_e4m3x2(p0, p1);
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(p) : "f"(p1), "f"(p0));
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(p) : "r"(p), "r"(e4m3x2_to_half2(first)));
    asm("cvt.rn.satfinite.e5m2x2.f16x2 %0, %1;" : "=h"(r) : "r"(p));
    rest = r;
}

// Rows of Q by a warp into [rows][128 bytes] of both parts, 16-byte chunks exchanged by the row's number: a lane has four
// dimensions.  What a row has been divided by goes to `scale`.
__device__ __forceinline__ void split_q_row(uint2 q, int row, int lane, uint8_t* first, uint8_t* rest, float* scale) {
    const uint32_t abs0 = q.x & 0x7FFF7FFFu, abs1 = q.y & 0x7FFF7FFFu;
    auto finite = [](uint32_t bits) { return bits < 0x7F80u ? bits : 0u; };
    const uint32_t most = __reduce_max_sync(0xFFFFFFFFu, max(max(finite(abs0 & 0xFFFFu), finite(abs0 >> 16)),
                                                             max(finite(abs1 & 0xFFFFu), finite(abs1 >> 16))));
    // Exponent field e of the largest value: times 2^(134 - e).  A row of zeros keeps its own.
    const int up = most == 0u ? 0 : min(134 - static_cast<int>(most >> 7), 126);
    const float mul = __int_as_float((127 + up) << 23);
    float x[4] = {__uint_as_float(q.x << 16), __uint_as_float(q.x & 0xFFFF0000u), __uint_as_float(q.y << 16), __uint_as_float(q.y & 0xFFFF0000u)};
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = fabsf(x[i]) < INFINITY ? x[i] * mul : NAN;      // an infinity has no part to leave over
    const uint32_t a = pack_e4m3x2(x[0], x[1]), b = pack_e4m3x2(x[2], x[3]);
    const float2 fa = e4m3x2_to_float2(a), fb = e4m3x2_to_float2(b);
    const int at = row * 128 + (((lane >> 2) ^ (row & 7)) << 4) + (lane & 3) * 4;
    *reinterpret_cast<uint32_t*>(first + at) = a | b << 16;
    *reinterpret_cast<uint32_t*>(rest + at) = pack_e4m3x2(x[0] - fa.x, x[1] - fa.y) | pack_e4m3x2(x[2] - fb.x, x[3] - fb.y) << 16;
    if (lane == 0) *scale = __int_as_float((127 - up) << 23);
}

// ---------------------------------------------------------------------------------------
// Products of 8-bit operands
// ---------------------------------------------------------------------------------------
// Instruction descriptor: D in f32, A and B in e4m3 (0) or e5m2 (1).
__host__ __device__ constexpr uint32_t make_idesc_8(int m, int n, int a_mn_major, int b_mn_major, int a_e5m2, int b_e5m2) {
    return (1u << 4) | (static_cast<uint32_t>(a_e5m2) << 7) | (static_cast<uint32_t>(b_e5m2) << 10) |
           (static_cast<uint32_t>(a_mn_major) << 15) | (static_cast<uint32_t>(b_mn_major) << 16) | (static_cast<uint32_t>(n >> 3) << 17) |
           (static_cast<uint32_t>(m >> 4) << 24);
}

// Steps of 32 elements of the contraction: 32 bytes of a row where it runs along the rows, 32 rows where it runs across them.
// A tile of 128 columns is one swizzle atom wide, so an operand across has no second one for a leading offset to lead to.
constexpr int kStep8Along = 32 >> 4, kStep8Across = 32 * 128 >> 4;

// The four k-steps of a product over 128, as umma_ss_kk_x8_w.
template <int kAStep, int kBStep>
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
        "add.u32 ra, %1, %6;\n\t"
        "add.u32 rb, %2, %7;\n\t"
        "mov.b64 da, {ra, %5};\n\t"
        "mov.b64 db, {rb, %5};\n\t"
        "@pe tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], da, db, %3, pt;\n\t"
        "add.u32 ra, ra, %6;\n\t"
        "add.u32 rb, rb, %7;\n\t"
        "mov.b64 da, {ra, %5};\n\t"
        "mov.b64 db, {rb, %5};\n\t"
        "@pe tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], da, db, %3, pt;\n\t"
        "add.u32 ra, ra, %6;\n\t"
        "add.u32 rb, rb, %7;\n\t"
        "mov.b64 da, {ra, %5};\n\t"
        "mov.b64 db, {rb, %5};\n\t"
        "@pe tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], da, db, %3, pt;\n\t"
        "}\n"
        ::"r"(d_tmem), "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(accumulate), "r"(kDescHiSw128), "n"(kAStep), "n"(kBStep)
        : "memory");
}

// A from tensor memory, four elements a column.
template <int kBStep>
__device__ __forceinline__ void umma8_ts_x4_w(uint32_t d_tmem, uint32_t a_tmem, uint32_t b_lo, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t"
        ".reg .pred p, pe, pt;\n\t"
        ".reg .b64 db;\n\t"
        ".reg .b32 ra, rb;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "setp.eq.b32 pt, 0, 0;\n\t"
        "elect.sync _|pe, 0xFFFFFFFF;\n\t"
        "mov.b64 db, {%2, %5};\n\t"
        "@pe tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], [%1], db, %3, p;\n\t"
        "add.u32 ra, %1, 8;\n\t"
        "add.u32 rb, %2, %6;\n\t"
        "mov.b64 db, {rb, %5};\n\t"
        "@pe tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], [ra], db, %3, pt;\n\t"
        "add.u32 ra, ra, 8;\n\t"
        "add.u32 rb, rb, %6;\n\t"
        "mov.b64 db, {rb, %5};\n\t"
        "@pe tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], [ra], db, %3, pt;\n\t"
        "add.u32 ra, ra, 8;\n\t"
        "add.u32 rb, rb, %6;\n\t"
        "mov.b64 db, {rb, %5};\n\t"
        "@pe tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], [ra], db, %3, pt;\n\t"
        "}\n"
        ::"r"(d_tmem), "r"(a_tmem), "r"(b_lo), "r"(idesc), "r"(accumulate), "r"(kDescHiSw128), "n"(kBStep)
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

// Probabilities are at most 2^8 for the product; a new reference puts the largest one at 2^5, so that it moves only when the
// maximum has grown by a factor of eight.
constexpr float kP8Most = 8.f, kP8At = 5.f;

__device__ __forceinline__ bool e4m3_not_finite(uint32_t byte) { return (byte & 0x7Fu) == 0x7Fu; }

// As tree_clean_row, for a row of 128 bytes: e4m3 has no infinities.
__device__ __forceinline__ bool tree8_clean_row(uint8_t* row, int r, bool behind) {
    auto chunk = [&](int c) { return reinterpret_cast<uint4*>(row + ((c + r) & 7) * 16); };
    if (behind) {
#pragma unroll
        for (int c = 0; c < 8; ++c) *chunk(c) = make_uint4(0u, 0u, 0u, 0u);
        return false;
    }
    // A magnitude of 0x7F plus one carries into its byte's sign bit, and no other does.
    auto ones = [](uint32_t w) { return ((w & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u; };
    uint32_t any = 0;
#pragma unroll
    for (int c = 0; c < 8; ++c) {
        const uint4 v = *chunk(c);
        any |= ones(v.x) | ones(v.y) | ones(v.z) | ones(v.w);
    }
    if (any == 0u) return false;
#pragma unroll 1
    for (int c = 0; c < 8; ++c) {
        const uint4 v = *chunk(c);
        auto without = [&](uint32_t w) { return w & ~((ones(w) >> 7) * 0xFFu); };
        *chunk(c) = make_uint4(without(v.x), without(v.y), without(v.z), without(v.w));
    }
    return true;
}

// Loads of V by one warp, as tree_load_v.
template <int kSlots, int kStages, typename Shared>
__device__ __forceinline__ void tree8_load_v(const TreeParams& p, Shared& sh, const CUtensorMap* map, const WaitCtx& wctx, int lane) {
    SlotLoader loader(p.box_rows);
    uint32_t v_it = 0;
    bool ok = true;
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
            ok = warp_wait(wctx, smem_u32(&sh.v_empty[stage]), ((v_it / kStages) & 1u) ^ 1u, 18);
            if (!ok) break;
            load_slots8(now, map, smem_u32(&sh.v[stage][0]), smem_u32(&sh.v_full[stage]), w.head, boxes, lane);
        }
    }
}

// b2a_tree8_few.cu: calls of at most kFewRows rows an item.
int launch_tree8_few(const CUtensorMap& map_k, const CUtensorMap& map_v, const Tree8Params& p, int ctas, const DeviceInfo& dev,
                     cudaStream_t stream);

}  // namespace b2a
