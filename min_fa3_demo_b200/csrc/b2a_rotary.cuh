// Rotary positions as the kernels see them: a token's angles, a head's pairs turned by them, and where a new token goes.
#pragma once

#include "b2a_cache.cuh"

#include <cmath>

namespace b2a {

constexpr int kRotaryThreads = 256;

struct RotaryParams {
    const __nv_bfloat16* src[3];     // q, k, v
    long long stride[3][3];          // sequence, token, head
    int heads[3];
    __nv_bfloat16* dst[2];           // contiguous q and, without a cache, k
    const void* positions;
    long long positions_stride[3];   // axis, sequence, token
    int positions_64;
    int seqlen;                      // of fixed-length batches
    int total;
    int batch;
    int pairs;
    int adjacent;
    float sign;
    float magnitude;
    // Cache writes only:
    CacheView cache;
    const int* cache_lens;
    const int* cu_seqlens;
    WorkspaceHeader* header;
    unsigned long long turn[64];
    unsigned char axis[64];
};

struct TokenPlace {
    int seq;
    int number;          // within its sequence
    long long k_at;      // element of the cache's row; -1: the token has no place
    long long v_at;
    int valid;
};

// Sequence and number of a packed token by one warp: how many sequences end at or before it.
__device__ __forceinline__ TokenPlace find_token(const RotaryParams& p, int token, int lane) {
    TokenPlace at{};
    at.valid = token < p.total;
    if (!at.valid) return at;
    if (p.cu_seqlens == nullptr) {
        at.seq = token / p.seqlen;
        at.number = token - at.seq * p.seqlen;
        return at;
    }
    // Of more than 64, first which 32nd of them it is in.
    int ended = 0;
    if (p.batch > 64) {
        const int part = (p.batch + 31) / 32, last = (lane + 1) * part;
        ended = part * __popc(__ballot_sync(0xFFFFFFFFu, last <= p.batch && p.cu_seqlens[min(last, p.batch)] <= token));
    }
    for (int b = ended; b < p.batch; b += 32) {
        const bool before = b + lane < p.batch && p.cu_seqlens[b + lane + 1] <= token;
        const int n = __popc(__ballot_sync(0xFFFFFFFFu, before));
        ended += n;
        if (n < 32) break;
    }
    at.seq = ended;
    at.valid = ended < p.batch;
    if (at.valid) {
        at.number = token - p.cu_seqlens[ended];
        at.valid = at.number >= 0;
    }
    return at;
}

__device__ __forceinline__ float2 bf16x2_to_float2(uint32_t x) {
    return make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xFFFF0000u));
}

__device__ __forceinline__ long long position_of(const RotaryParams& p, int axis, int seq, int number) {
    const long long at = axis * p.positions_stride[0] + seq * p.positions_stride[1] + number * p.positions_stride[2];
    return p.positions_64 ? static_cast<const long long*>(p.positions)[at] : static_cast<const int*>(p.positions)[at];
}

// Cosine and sine of a pair's angle, times the magnitude.
__device__ __forceinline__ float2 angle_of(const RotaryParams& p, unsigned long long turn, long long position) {
    const unsigned long long turns = static_cast<unsigned long long>(position) * turn;
    float s, c;
    sincospif(static_cast<float>(static_cast<int>(turns >> 32)) * 4.656612873077393e-10f, &s, &c);   // 2^-31
    return make_float2(c * p.magnitude, s * p.sign * p.magnitude);
}

__device__ __forceinline__ float2 pair_angle(const RotaryParams& p, int pair, int seq, int number) {
    return angle_of(p, p.turn[pair], position_of(p, p.axis[pair], seq, number));
}

// Every sequence's new slots and pages exist?  CTA 0 of a cache write finds out and writes the whole header, so that no
// launch has to clear it; the others only leave out what has no place.  A lane a sequence; where one has more than two new pages, those
// of the warp's 32 sequences one behind the other, a lane a page, whoever they belong to: a long prompt among many single tokens.
// One K/V head in pages of 8, us as it was with a warp a sequence up to 64 of them and a thread a sequence beyond, and now: one token of
// 64 sequences 7.2, 3.4; of 4,096 12.9, 11.7; 32,768 tokens of one of 64 40.9, 24.3; of one of 65 511, 24.4.
__device__ __forceinline__ void check_append(const RotaryParams& p) {
    constexpr int kWarps = kRotaryThreads / 32;
    __shared__ int bad;
    if (threadIdx.x == 0) bad = 0;
    __syncthreads();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    bool wrong = false;
    int first = 0, begin = 0, end = 0;
    auto ask = [&](int b) {
        if (b >= p.batch) return;
        first = p.cache_lens[b];
        begin = p.cu_seqlens == nullptr ? 0 : p.cu_seqlens[b];
        end = p.cu_seqlens == nullptr ? p.seqlen : p.cu_seqlens[b + 1];
    };
    auto gone = [&](int b, int entry) {
        const int page = p.cache.block_table[b * p.cache.table_stride + entry];
        return page < 0 || page >= p.cache.pages;
    };
    ask(lane * kWarps + warp);
#pragma unroll 1
    for (int b0 = 0; b0 < p.batch; b0 += kRotaryThreads) {
        const int b = b0 + lane * kWarps + warp;
        int entry = 0, pages = 0;        // of the sequence's row of the block table
        if (b < p.batch) {
            const long long last = first + (static_cast<long long>(end) - begin);
            if (begin < 0 || end < begin || (p.cu_seqlens != nullptr && end > p.total) || first < 0 || last > p.cache.capacity()) {
                wrong = true;
            } else if (p.cache.block_table != nullptr && last > first) {
                int row;
                entry = p.cache.entry_of(first, &row);
                pages = p.cache.entry_of(static_cast<int>(last - 1), &row) - entry + 1;
            }
        }
        ask(b + kRotaryThreads);         // the next ones' lengths are on their way meanwhile
        if (!__any_sync(0xFFFFFFFFu, pages > 2)) {
            for (int i = 0; i < pages; ++i) wrong |= gone(b, entry + i);
            continue;
        }
        int upto = pages;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int up = __shfl_up_sync(0xFFFFFFFFu, upto, d);
            if (lane >= d) upto += up;
        }
        const int all = __shfl_sync(0xFFFFFFFFu, upto, 31), from = entry - (upto - pages);
#pragma unroll 4
        for (int i = lane; i - lane < all; i += 32) {
            int of = 0;                  // whose it is: so many lanes' pages end at or before it
#pragma unroll
            for (int d = 16; d > 0; d >>= 1) of += __shfl_sync(0xFFFFFFFFu, upto, of + d - 1) <= i ? d : 0;
            const int at = __shfl_sync(0xFFFFFFFFu, from, of) + i;
            if (i < all) wrong |= gone(b0 + of * kWarps + warp, at);
        }
    }
    if (wrong) bad = 1;
    __syncthreads();
    if (threadIdx.x == 0) *p.header = WorkspaceHeader{0, 0, bad ? kStatusBadArg << 24 : 0u, 0};
}

// kTokens tokens, from cta * kTokens on, by a CTA.
template <bool kAppend, int kTokens>
__device__ __forceinline__ void turn_tokens(const RotaryParams& p, int cta) {
    constexpr int kWarpsPerToken = kRotaryThreads / 32 / kTokens;
    __shared__ __align__(16) float2 cos_sin[kTokens][64];
    __shared__ TokenPlace place[kTokens];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int token0 = cta * kTokens;

    // A thread's 16 dimensions: for halves [8 c, 8 c + 8) of each while there are pairs, behind them 16 in a row; for
    // neighbours 8 of the lower and 8 of the upper 64, so that eight threads load 128 bytes in a row.
    const int c = lane & 7;
    const bool turned = c * 8 < p.pairs;                  // halves only
    const int lo = p.adjacent || turned ? 8 * c : 16 * c;
    const int hi = p.adjacent ? 64 + 8 * c : turned ? p.pairs + 8 * c : 16 * c + 8;
    const int mine = warp / kWarpsPerToken, token = token0 + mine;
    const int heads = p.heads[0] + p.heads[1] + p.heads[2];
    const int seq = p.cu_seqlens == nullptr ? token / p.seqlen : 0, number = token - seq * p.seqlen;
    auto which_of = [&](int h) { return h < p.heads[0] ? 0 : h < p.heads[0] + p.heads[1] ? 1 : 2; };
    auto head_of = [&](int h, int which) { return h - (which > 0 ? p.heads[0] : 0) - (which > 1 ? p.heads[1] : 0); };
    auto source = [&](int h) {
        const int which = which_of(h);
        return p.src[which] + seq * p.stride[which][0] + number * p.stride[which][1] + head_of(h, which) * p.stride[which][2];
    };
    // The first head's values are on their way while the angles are computed.
    int h = (warp % kWarpsPerToken) * 4 + (lane >> 3);
    uint4 a{}, b{};
    if (token < p.total && h < heads) {
        const __nv_bfloat16* src = source(h);
        a = *reinterpret_cast<const uint4*>(src + lo);
        b = *reinterpret_cast<const uint4*>(src + hi);
    }
    if (warp < kTokens) {
        TokenPlace at = find_token(p, token0 + warp, lane);
        if (kAppend && at.valid) {
            int row;
            const int page = p.cache.page_of(at.seq, static_cast<long long>(p.cache_lens[at.seq]) + at.number, &row);
            at.k_at = p.cache.at(p.cache.k_stride, page, row, 0);
            at.v_at = p.cache.at(p.cache.v_stride, page, row, 0);
        }
        if (lane == 0) place[warp] = at;
    }
    if (p.pairs > 0) {
        for (int i = threadIdx.x; i < kTokens * 64; i += kRotaryThreads) {
            const int pair = i & 63, token = token0 + (i >> 6);
            if (pair >= p.pairs || token >= p.total) continue;
            const int seq = p.cu_seqlens == nullptr ? token / p.seqlen : 0;
            cos_sin[i >> 6][pair] = pair_angle(p, pair, seq, token - seq * p.seqlen);
        }
    }
    __syncthreads();

    const TokenPlace at = place[mine];
    if (at.valid) {
        float2 cs[8];
        const bool turn_lo = 4 * c < p.pairs, turn_hi = 32 + 4 * c < p.pairs;      // neighbours only
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int pair = p.adjacent ? (e < 4 ? 4 * c + e : 28 + 4 * c + e) : 8 * c + e;
            cs[e] = pair < p.pairs ? cos_sin[mine][pair] : make_float2(1.f, 0.f);
        }
#pragma unroll 1
        while (h < heads) {
            const int which = which_of(h), head = head_of(h, which);
            __nv_bfloat16* dst;
            if (kAppend && which > 0) {
                const long long row = which == 1 ? at.k_at : at.v_at;
                dst = row < 0 ? nullptr
                      : which == 1 ? p.cache.k + row + head * p.cache.k_stride[2] : p.cache.v + row + head * p.cache.v_stride[2];
            } else {
                dst = p.dst[which] + (static_cast<long long>(token) * p.heads[which] + head) * kHeadDim;
            }
            uint32_t x[4] = {a.x, a.y, a.z, a.w}, y[4] = {b.x, b.y, b.z, b.w};
            h += 4 * kWarpsPerToken;
            if (h < heads) {
                const __nv_bfloat16* src = source(h);
                a = *reinterpret_cast<const uint4*>(src + lo);
                b = *reinterpret_cast<const uint4*>(src + hi);
            }
            if (which < 2) {
                if (p.adjacent) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float2 u = bf16x2_to_float2(x[e]), w = bf16x2_to_float2(y[e]);
                        if (turn_lo) x[e] = pack_bf16x2(u.x * cs[e].x - u.y * cs[e].y, u.y * cs[e].x + u.x * cs[e].y);
                        if (turn_hi) y[e] = pack_bf16x2(w.x * cs[4 + e].x - w.y * cs[4 + e].y, w.y * cs[4 + e].x + w.x * cs[4 + e].y);
                    }
                } else if (turned) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float2 u = bf16x2_to_float2(x[e]), w = bf16x2_to_float2(y[e]);
                        const float2 c0 = cs[2 * e], c1 = cs[2 * e + 1];
                        x[e] = pack_bf16x2(u.x * c0.x - w.x * c0.y, u.y * c1.x - w.y * c1.y);
                        y[e] = pack_bf16x2(w.x * c0.x + u.x * c0.y, w.y * c1.x + u.y * c1.y);
                    }
                }
            }
            if (dst != nullptr) {
                *reinterpret_cast<uint4*>(dst + lo) = make_uint4(x[0], x[1], x[2], x[3]);
                *reinterpret_cast<uint4*>(dst + hi) = make_uint4(y[0], y[1], y[2], y[3]);
            }
        }
    }
}

inline int set_axes(RotaryParams& p, const b2a_rotary_axes& axes, const void* positions, int positions_64, const int64_t* stride,
             bool inverse) {
    B2A_REQUIRE(axes.pairs >= 8 && axes.pairs <= 64 && axes.pairs % 8 == 0,
                "the number of pairs must be a multiple of 8 between 8 and 64, got %d", axes.pairs);
    B2A_REQUIRE(positions != nullptr, "positions must not be NULL");
    B2A_REQUIRE(std::isfinite(axes.magnitude), "magnitude must be finite");
    for (int i = 0; i < axes.pairs; ++i) {
        B2A_REQUIRE(axes.axis[i] < axes.axes, "pair %d has axis %d of %d", i, axes.axis[i], axes.axes);
        p.turn[i] = axes.turn[i];
        p.axis[i] = axes.axis[i];
    }
    p.pairs = axes.pairs;
    p.adjacent = axes.adjacent ? 1 : 0;
    p.positions = positions;
    p.positions_64 = positions_64 ? 1 : 0;
    for (int i = 0; i < 3; ++i) p.positions_stride[i] = stride[i];
    p.sign = inverse ? -1.f : 1.f;
    p.magnitude = axes.magnitude == 0.f ? 1.f : axes.magnitude;
    return B2A_OK;
}

inline int set_source(RotaryParams& p, int which, const void* src, const int64_t* stride, int heads, const char* name) {
    B2A_REQUIRE(src != nullptr && (reinterpret_cast<uintptr_t>(src) & 0xF) == 0, "%s must be a 16-byte aligned device pointer", name);
    p.src[which] = static_cast<const __nv_bfloat16*>(src);
    p.heads[which] = heads;
    for (int i = 0; i < 3; ++i) {
        B2A_REQUIRE(stride[i] >= 0 && stride[i] % 8 == 0, "strides of %s must be multiples of 8 elements", name);
        p.stride[which][i] = stride[i];
    }
    return B2A_OK;
}

// Checks the arguments of a cache write.
inline int make_append(const b2a_append_args& a, RotaryParams& p) {
    B2A_REQUIRE(a.batch >= 1 && a.total >= 1, "batch and total must be positive");
    B2A_REQUIRE(a.cache_lens != nullptr, "cache_lens must not be NULL");
    int rc = make_cache_view(a.cache, a.batch, true, &p.cache);
    if (rc != B2A_OK) return rc;
    if (a.cu_seqlens == nullptr) {
        B2A_REQUIRE(a.seqlen >= 1 && static_cast<long long>(a.batch) * a.seqlen == a.total,
                    "fixed-length sizes must satisfy total = batch * seqlen");
    }
    B2A_REQUIRE(a.axes != nullptr || a.q == nullptr, "q is turned by positions, so it needs axes");
    if (a.axes != nullptr) rc = set_axes(p, *a.axes, a.positions, a.positions_64, a.positions_stride, false);
    if (rc == B2A_OK && a.q != nullptr) {
        B2A_REQUIRE(a.heads_q >= 1, "heads_q must be positive");
        B2A_REQUIRE(a.q_out != nullptr && (reinterpret_cast<uintptr_t>(a.q_out) & 0xF) == 0,
                    "q_out must be a 16-byte aligned device pointer");
        rc = set_source(p, 0, a.q, a.q_stride, a.heads_q, "q");
    }
    if (rc == B2A_OK) rc = set_source(p, 1, a.k, a.k_stride, a.cache.heads_k, "k");
    if (rc == B2A_OK) rc = set_source(p, 2, a.v, a.v_stride, a.cache.heads_k, "v");
    if (rc != B2A_OK) return rc;
    B2A_REQUIRE(a.workspace != nullptr && (reinterpret_cast<uintptr_t>(a.workspace) & 0xF) == 0,
                "workspace must be a 16-byte aligned device pointer");
    if (a.workspace_bytes < sizeof(WorkspaceHeader)) {
        return fail(B2A_ERR_WORKSPACE_TOO_SMALL, "workspace has %zu bytes, need %zu", a.workspace_bytes, sizeof(WorkspaceHeader));
    }
    p.dst[0] = static_cast<__nv_bfloat16*>(a.q_out);
    p.batch = a.batch;
    p.seqlen = a.seqlen;
    p.total = a.total;
    p.cache_lens = a.cache_lens;
    p.cu_seqlens = a.cu_seqlens;
    p.header = static_cast<WorkspaceHeader*>(a.workspace);
    return B2A_OK;
}

}  // namespace b2a
