// New keys and values into a cache in 8 bits, turned by their positions on the way.
//
// All slots of a block share a head's scale, so a block's new keys (or values) of a head belong to one warp: eight lanes a token with 16
// dimensions each, as in b2a_rotary.cuh, and 16 tokens on their way at once, by asynchronous copies.  It turns them in fp32, looks for
// the largest, finds the scale, turns them once more and rounds; nothing waits for another warp.  Blocks of more new tokens than 16
// are read twice, the second time from L2.  e4m3 is a floating-point format, so a scale that is a power of two costs no accuracy
// (it puts the largest value above 224, and values keep their four bits down to 2^-6, 2^-13.8 of it; down to 2^-6 times the scale where
// a block keeps an older, larger one), divides exactly, and can grow with hardly a trace: x / 2 is a number of the format as well,
// unless it is one of the smallest.  So a block whose tokens come one by one keeps its scale until a token does not fit, and then the
// tokens that it holds are read, divided and written again, at most 127 of 128 bytes.
//
// Should be bound by memory: 256 bytes in and 128 out a token and head, and q's 256 and 256.  A CTA has a block of slots and some of the
// heads, for which it computes the angles once; CTAs behind those turn q, and the first one looks for places that do not exist.
// One new token of 16 sequences, 32 + 8 heads, is 4.8 us, what a launch with four reads one after another takes.  715 of 32
// sequences: 12.2 us.  5,647 of 4: 139 MB in 35 us, of which q alone is 20 and k and v alone 21: each keeps the SMs' issue slots
// half busy (9.3 and 9.6 million instructions, most of them of the turning, which k needs twice).  That was 58 us with a piece of
// code for each of the two passes and four tokens, and a division where a product does: an instruction fetched for one use costs
// more than its work.  64 registers and four CTAs an SM: with three 39 us for 35.6, with five 37.6.
#include "b2a_cache8.cuh"
#include "b2a_rotary.cuh"

namespace b2a {

namespace {

struct Append8Params {
    RotaryParams r;              // its heads are q's alone
    CacheScales scales;
    int kv_ctas;                 // a block of slots, a part of the heads
    int heads;                   // of k and v
    int parts;                   // of them
    int part_heads;
    int seq_blocks;              // fixed-length batches: most blocks of a sequence
    int run;                     // packed tokens of many sequences: those of a CTA; otherwise 0
    int stages;                  // of shared memory a warp: 1 where it has one unit of one tile
};

// A block of slots that new tokens fall into.
struct Append8Block {
    int seq, token;              // the first of them: its number within the sequence, and
    int q_begin;                 // the row of the sequence's first
    int count;                   // of them; 0: there is nothing to do
    int held;                    // tokens before them
    int page, row;               // of the block's first slot
    int last;                    // the CTA has no other
};

// Of a sequence's n new tokens behind len, number `token` and those that share its block.
__device__ __forceinline__ void fill_block(const RotaryParams& p, int mask, int len, int n, int token, Append8Block& at) {
    const long long first = static_cast<long long>(len) + token, begin = first & ~static_cast<long long>(mask);
    const long long last = min(min(begin + mask + 1, static_cast<long long>(len) + n), static_cast<long long>(p.cache.capacity()));
    at.token = token;
    at.page = p.cache.page_of(at.seq, begin, &at.row);
    at.held = static_cast<int>(first - begin);
    at.count = at.page < 0 || last <= first ? 0 : static_cast<int>(last - first);
}

// Packed tokens of few sequences: number `item` of all their blocks, by one warp.
__device__ __forceinline__ Append8Block block_of_item(const RotaryParams& p, int shift, int item, int lane) {
    const int mask = (1 << shift) - 1;
    Append8Block at{};
    at.last = 1;
    auto blocks_of = [&](int b) -> int {
        const int begin = p.cu_seqlens[b], end = p.cu_seqlens[b + 1], len = p.cache_lens[b];
        if (begin < 0 || end <= begin || end > p.total || len < 0) return 0;
        return static_cast<int>(((len & mask) + static_cast<long long>(end - begin) - 1) >> shift) + 1;
    };
    // Which of 32 runs of sequences has the item, then which run of that one, until a run is a sequence.
    int first = 0, run = p.batch, before = 0;
#pragma unroll 1
    do {
        const int end = first + run;
        run = (run + 31) / 32;
        const int begin = first + lane * run;
        int mine = 0;
#pragma unroll 4
        for (int b = begin; b < min(begin + run, end); ++b) mine += blocks_of(b);
        int upto = mine;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int up = __shfl_up_sync(0xFFFFFFFFu, upto, d);
            if (lane >= d) upto += up;
        }
        const unsigned hit = __ballot_sync(0xFFFFFFFFu, before + upto > item);
        if (hit == 0u) return at;
        const int l = __ffs(hit) - 1;
        first += l * run;
        run = min(run, end - first);
        before += __shfl_sync(0xFFFFFFFFu, upto - mine, l);
    } while (run > 1);
    // The first block may begin with tokens that are there already.
    const int len = p.cache_lens[first], j = item - before;
    at.seq = first;
    at.q_begin = p.cu_seqlens[first];
    fill_block(p, mask, len, p.cu_seqlens[first + 1] - at.q_begin, j == 0 ? 0 : (j << shift) - (len & mask), at);
    return at;
}

// Packed tokens of many sequences: a CTA has `run` of them, and the blocks whose first new token is among them.  `token` is the first
// that has not been looked at yet.
struct PackedTokens {
    int token, end, seq;

    // Which sequence a token is in: the number of those that end at or before it, by one warp, a 32nd of those in question a step.
    __device__ __forceinline__ PackedTokens(const RotaryParams& p, long long first, int run, int lane) {
        token = static_cast<int>(first);
        end = static_cast<int>(min(first + run, static_cast<long long>(p.total)));
        seq = 0;
#pragma unroll 1
        for (int left = run == 0 ? 0 : p.batch; left > 0;) {
            const int part = (left + 31) / 32, last = (lane + 1) * part;
            const int ended = __popc(__ballot_sync(0xFFFFFFFFu, last <= left && p.cu_seqlens[seq + min(last, left)] <= token));
            seq += ended * part;
            left = part == 1 ? 0 : min(part, left - ended * part);
        }
    }

    __device__ __forceinline__ Append8Block next(const RotaryParams& p, int mask) {
        Append8Block at{};
        at.last = 1;
        while (token < end && seq < p.batch) {
            const int begin = p.cu_seqlens[seq], behind = p.cu_seqlens[seq + 1], len = p.cache_lens[seq];
            if (begin < 0 || behind <= max(token, begin) || behind > p.total || len < 0) {      // none here, or what does not fit
                ++seq;
                continue;
            }
            token = max(token, begin);
            const int inside = static_cast<int>(static_cast<unsigned>(len) + static_cast<unsigned>(token - begin)) & mask;
            const int here = min(mask + 1 - inside, behind - token);
            if (token < end && (token == begin || inside == 0)) {
                at.seq = seq;
                at.q_begin = begin;
                fill_block(p, mask, len, behind - begin, token - begin, at);
                token += here;
                at.last = token >= end;
                return at;
            }
            token += here;
        }
        return at;
    }
};

// The smallest power of two, within 2^-64 .. 2^64, of which `most` is at most 448 times: 448 = 1.75 * 2^8.
__device__ __forceinline__ float scale_for(float most) {
    const int bits = __float_as_int(most);
    const int e = (bits >> 23) - 8 + ((bits & 0x7FFFFF) > 0x600000 ? 1 : 0);
    return __int_as_float(min(max(e, 127 - 64), 127 + 64) << 23);
}

// Values divided by a scale: a power of two has an exact reciprocal, others are divided.
struct Divider {
    float scale, inverse;
    __device__ __forceinline__ explicit Divider(float s) {
        scale = s;
        inverse = (__float_as_int(s) & 0x7FFFFF) == 0 ? 1.f / s : 0.f;
    }
    template <int N>
    __device__ __forceinline__ void operator()(float (&x)[N]) const {
        if (inverse != 0.f) {
#pragma unroll
            for (int e = 0; e < N; ++e) x[e] *= inverse;
        } else {
            slowly<N>(x);
        }
    }
    template <int N>
    __device__ __forceinline__ void slowly(float (&x)[N]) const {
#pragma unroll
        for (int e = 0; e < N; ++e) x[e] = divided(x[e], scale);
    }
    static __device__ __noinline__ float divided(float x, float by) { return x / by; }
};

__device__ __forceinline__ __nv_bfloat162 as_bf16x2(uint32_t two) { return *reinterpret_cast<const __nv_bfloat162*>(&two); }

__device__ __forceinline__ void turn_pair(float& a, float& b, float cos, float sin) {
    const float x = a;
    a = x * cos - b * sin;
    b = b * cos + x * sin;
}

constexpr int kQTokens = 4;     // a CTA that turns q: 1, 2, 4, 8 take 43.4, 43.9, 35.7, 36.6 us for 5,647, all the same 6.2 for 16
constexpr int kTile8 = 16;      // tokens on their way to a warp at once
constexpr int kStage8Bytes = kTile8 * kHeadDim * static_cast<int>(sizeof(__nv_bfloat16));

__device__ __forceinline__ void copy16_or_zero(uint32_t dst, const void* src, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}

// Dynamic shared memory: one or two stages of kTile8 tokens for each warp, then the angles of the block's new tokens, 64 each.
__global__ void __launch_bounds__(kRotaryThreads, 4)
append8_tokens(const __grid_constant__ Append8Params p8) {
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ Append8Block block;
    const RotaryParams& p = p8.r;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    constexpr int kWarps = kRotaryThreads / 32;
    float2* cos_sin = reinterpret_cast<float2*>(smem + kWarps * p8.stages * kStage8Bytes);
    let_next_kernel_start();
    wait_for_previous_kernel();

    if (blockIdx.x == 0) {
        check_append(p);
    } else if (blockIdx.x > p8.kv_ctas) {
        turn_tokens<false, kQTokens>(p, blockIdx.x - 1 - p8.kv_ctas);
    } else {
        const int item = blockIdx.x - 1;
        const int mask = (1 << p8.scales.shift) - 1;
        PackedTokens packed(p, static_cast<long long>(item / p8.parts) * p8.run, p8.run, lane);
#pragma unroll 1
        for (bool more = true; more;) {
            __syncthreads();
            if (warp == 0) {
                Append8Block at{};
                if (p.cu_seqlens == nullptr) {
                    at.seq = item / p8.parts / p8.seq_blocks;
                    const int j = item / p8.parts - at.seq * p8.seq_blocks, len = p.cache_lens[at.seq];
                    const long long token = j == 0 ? 0 : (static_cast<long long>(j) << p8.scales.shift) - (len & mask);
                    if (len >= 0 && token < p.seqlen) fill_block(p, mask, len, p.seqlen, static_cast<int>(token), at);
                    at.last = 1;
                } else if (p8.run == 0) {
                    at = block_of_item(p, p8.scales.shift, item / p8.parts, lane);
                } else {
                    at = packed.next(p, mask);
                }
                if (lane == 0) block = at;
            }
            __syncthreads();
            const Append8Block at = block;
            more = at.last == 0;
            const int h0 = (item % p8.parts) * p8.part_heads, units = at.count > 0 ? 2 * min(p8.part_heads, p8.heads - h0) : 0;
            const int c = lane & 7, mine = lane >> 3;

            // A unit: K (even) or V of a head.  A thread's 16 dimensions, as in turn_tokens: of V, and behind the pairs, 16 in a row.
            const bool turned = !p.adjacent && c * 8 < p.pairs;
            auto lo_of = [&](int which) { return which == 0 && p.pairs > 0 && (p.adjacent || turned) ? 8 * c : 16 * c; };
            auto hi_of = [&](int which) {
                return which == 0 && p.pairs > 0 && p.adjacent ? 64 + 8 * c : which == 0 && turned ? p.pairs + 8 * c : 16 * c + 8;
            };
            // A unit's tiles are loaded from the first to the last, for the largest value, and back, to be written: the last one, and so
            // the only one of few tokens, once, and of two the first one once as well, which is still there.  A thread reads back what it
            // copied itself.
            const int tiles = (at.count + kTile8 - 1) / kTile8, trips = 2 * tiles - 1;
            const uint32_t stage0 = smem_u32(smem) + warp * p8.stages * kStage8Bytes + mine * 256 + c * 16;
            auto load = [&](int unit, int trip, int stage) {
                if (tiles == 2 && trip == 2) return;
                const int which = unit & 1, lo = lo_of(which), hi = hi_of(which);
                const int token0 = (trip < tiles ? trip : 2 * tiles - 2 - trip) * kTile8;
                const long long* stride = p.stride[1 + which];
                const __nv_bfloat16* src = p.src[1 + which] + (h0 + (unit >> 1)) * stride[2] +
                                           (p.cu_seqlens == nullptr ? at.seq * stride[0] + at.token * stride[1]
                                                                    : (static_cast<long long>(at.q_begin) + at.token) * stride[1]);
#pragma unroll
                for (int t = 0; t < kTile8 / 4; ++t) {
                    const int token = token0 + t * 4 + mine;
                    const __nv_bfloat16* from = src + (token < at.count ? token : 0) * stride[1];
                    const uint32_t to = stage0 + stage * kStage8Bytes + t * 1024;
                    copy16_or_zero(to, from + lo, token < at.count);
                    copy16_or_zero(to + 128, from + hi, token < at.count);
                }
            };
            int unit = warp, trip = 0, stage = 0;
            if (unit < units) load(unit, 0, 0);        // on their way while the angles are computed
            asm volatile("cp.async.commit_group;" ::: "memory");
            if (p.pairs > 0) {
                // A thread's pair stays the same, for which it looks once: lanes that read different constants wait for one another.
                const int pair = threadIdx.x & 63;
                if (pair < p.pairs) {
                    const int axis = p.axis[pair];
                    const unsigned long long turn = p.turn[pair];
                    // Packed tokens are one sequence to the positions.
                    const bool apart = p.cu_seqlens == nullptr;
                    const int seq = apart ? at.seq : 0, first = apart ? at.token : at.q_begin + at.token;
                    // The eight pairs of a thread of a token as four pieces of 16 bytes, and those of eight threads in a row.
                    const int of = p.adjacent ? pair >> 2 & 7 : pair >> 3, e = p.adjacent ? (pair & 3) + (pair >> 5) * 4 : pair & 7;
                    float2* const to = cos_sin + (e >> 1) * 16 + of * 2 + (e & 1);
                    int token = threadIdx.x >> 6;
                    long long position = token < at.count ? position_of(p, axis, seq, first + token) : 0;
#pragma unroll 1
                    while (token < at.count) {
                        const int next = token + kRotaryThreads / 64;
                        const long long next_position = next < at.count ? position_of(p, axis, seq, first + next) : 0;
                        to[token * 64] = angle_of(p, turn, position);
                        token = next;
                        position = next_position;
                    }
                }
                __syncthreads();
            }
            float most = 0.f, before = 0.f, scale = 0.f;
            bool infinite = false;          // this thread has seen an infinity in the unit
#pragma unroll 1
            while (unit < units) {
                const int next_unit = trip + 1 < trips ? unit : unit + kWarps, next_trip = trip + 1 < trips ? trip + 1 : 0;
                if (next_unit < units) load(next_unit, next_trip, stage ^ 1);
                asm volatile("cp.async.commit_group;" ::: "memory");
                asm volatile("cp.async.wait_group 1;" ::: "memory");

                const int which = unit & 1, head = h0 + (unit >> 1);
                const int lo = lo_of(which), hi = hi_of(which), token0 = (trip < tiles ? trip : 2 * tiles - 2 - trip) * kTile8;
                const int steps = (min(at.count - token0, kTile8) + 3) / 4;
                const long long token_stride = (which == 0 ? p.cache.k_stride : p.cache.v_stride)[1];
                uint8_t* rows = reinterpret_cast<uint8_t*>(which == 0 ? p.cache.k : p.cache.v) +
                                p.cache.at(which == 0 ? p.cache.k_stride : p.cache.v_stride, at.page, at.row, head);
                float* scale_at = (which == 0 ? p8.scales.k : p8.scales.v) +
                                  p8.scales.at(which == 0 ? p8.scales.k_stride : p8.scales.v_stride, at.page, at.row, head);
                if (trip == 0) {
                    most = 0.f;
                    infinite = false;
                    before = at.held > 0 ? *scale_at : 0.f;
                }
                // The first half of the steps looks for the largest, the second one writes: one piece of code, which is what a short
                // kernel's time goes to.
#pragma unroll 1
                for (int i = trip < tiles ? 0 : steps; i < (trip < tiles - 1 ? steps : 2 * steps); ++i) {
                    const bool writes = i >= steps;
                    const int t = writes ? i - steps : i, token = token0 + t * 4 + mine;
                    if (i == steps && trip == tiles - 1) {
                        // Not negative: ordered as integers.
                        most = __int_as_float(__reduce_max_sync(0xFFFFFFFFu, __float_as_int(most)));
                        scale = at.held > 0 && most <= 448.f * before ? before : scale_for(most);
                    }
                    const uint32_t from = stage0 + stage * kStage8Bytes + t * 1024;
                    const uint4 a = ld_shared_v4(from), b = ld_shared_v4(from + 128);
                    const uint32_t u[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
                    if (!writes && which == 1) {
                        // The largest of V's as they come, two at a time.
                        __nv_bfloat162 two = __habs2(as_bf16x2(u[0]));
#pragma unroll
                        for (int e = 1; e < 8; ++e) two = __hmax2(two, __habs2(as_bf16x2(u[e])));
                        const float top = fmaxf(__low2float(two), __high2float(two));
                        if (top < INFINITY) {
                            most = fmaxf(most, top);
                            continue;
                        }
                    }
                    float x[16];
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const float2 f = bf16x2_to_float2(u[e]);
                        x[2 * e] = f.x;
                        x[2 * e + 1] = f.y;
                    }
                    if (which == 0 && token < at.count) {
                        const float4* cs = reinterpret_cast<const float4*>(cos_sin + token * 64) + c;
                        if (p.adjacent) {
#pragma unroll
                            for (int e = 0; e < 8; e += 2) {
                                if ((e < 4 ? 4 * c + e : 28 + 4 * c + e) >= p.pairs) continue;
                                const float4 two = cs[4 * e];
                                turn_pair(x[2 * e], x[2 * e + 1], two.x, two.y);
                                turn_pair(x[2 * e + 2], x[2 * e + 3], two.z, two.w);
                            }
                        } else if (turned) {
#pragma unroll
                            for (int e = 0; e < 8; e += 2) {
                                const float4 two = cs[4 * e];
                                turn_pair(x[e], x[8 + e], two.x, two.y);
                                turn_pair(x[e + 1], x[9 + e], two.z, two.w);
                            }
                        }
                    }
                    // Those that are not finite have no say, and are written as NaN.  fmaxf passes NaN over by itself.
                    if (!writes) {
                        float top = 0.f;
#pragma unroll
                        for (int e = 0; e < 16; ++e) top = fmaxf(top, fabsf(x[e]));
                        if (top == INFINITY) {
                            infinite = true;
                            top = 0.f;
#pragma unroll
                            for (int e = 0; e < 16; ++e) top = fmaxf(top, fabsf(x[e]) < INFINITY ? fabsf(x[e]) : 0.f);
                        }
                        most = fmaxf(most, top);
                    } else if (token < at.count) {
                        uint32_t out[4];
                        if (infinite) {
#pragma unroll
                            for (int e = 0; e < 16; ++e) x[e] = fabsf(x[e]) < INFINITY ? x[e] : NAN;
                        }
                        Divider by(scale);
                        by(x);
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            out[e] = pack_e4m3x2(x[4 * e], x[4 * e + 1]) | pack_e4m3x2(x[4 * e + 2], x[4 * e + 3]) << 16;
                        }
                        uint8_t* row = rows + (at.held + token) * token_stride;
                        if (hi == lo + 8) {
                            *reinterpret_cast<uint4*>(row + lo) = make_uint4(out[0], out[1], out[2], out[3]);
                        } else {
                            *reinterpret_cast<uint2*>(row + lo) = make_uint2(out[0], out[1]);
                            *reinterpret_cast<uint2*>(row + hi) = make_uint2(out[2], out[3]);
                        }
                    }
                }
                if (next_trip == 0 && (at.held == 0 || scale != before)) {
                    // Tokens that the block held.
                    Divider again(scale / before);
#pragma unroll 1
                    for (int token = mine; token < at.held; token += 4) {
                        uint4* row = reinterpret_cast<uint4*>(rows + token * token_stride + c * 16);
                        const uint4 v = *row;
                        const uint32_t words[4] = {v.x, v.y, v.z, v.w};
                        uint32_t out[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float2 f = e4m3x2_to_float2(words[e] & 0xFFFFu), g = e4m3x2_to_float2(words[e] >> 16);
                            float x[4] = {f.x, f.y, g.x, g.y};
                            again(x);
                            out[e] = pack_e4m3x2(x[0], x[1]) | pack_e4m3x2(x[2], x[3]) << 16;
                        }
                        *row = make_uint4(out[0], out[1], out[2], out[3]);
                    }
                    if (lane == 0) *scale_at = scale;
                }
                unit = next_unit;
                trip = next_trip;
                stage ^= 1;
            }
        }
    }
}

int set_append8_smem() {
    const int most = kRotaryThreads / 32 * 2 * kStage8Bytes + 128 * 64 * static_cast<int>(sizeof(float2));
    B2A_CUDA_OK(cudaFuncSetAttribute(append8_tokens, cudaFuncAttributeMaxDynamicSharedMemorySize, most));
    return B2A_OK;
}

}  // namespace

}  // namespace b2a

extern "C" {

int b2a_cache8_append(const b2a_append_args* a, const b2a_cache_scales* scales, void* cuda_stream) {
    using namespace b2a;
    B2A_REQUIRE(a != nullptr && scales != nullptr, "args and scales must not be NULL");
    Append8Params p{};
    int rc = make_append(*a, p.r);
    if (rc == B2A_OK) rc = make_cache_scales(*scales, a->cache, &p.scales);
    if (rc != B2A_OK) return rc;
    DeviceInfo dev{};
    rc = current_device_info(&dev);
    if (rc != B2A_OK) return rc;
    // n tokens that begin anywhere in a block touch this many.
    const int slots = scales->block;
    auto blocks = [&](long long n) { return (n + slots - 2) / slots + 1; };
    // Packed tokens: a CTA a block that there may be, which it looks for among the sequences' lengths; of many sequences, a CTA up to
    // half of the tokens that one has on average, so that most have one block to begin or none.  Us of either, 8 tokens a sequence: 64
    // 9.8, 11.1; 256 18.9, 19.6; 1,024 100, 66; 4,096 830, 259; one token: 8.6, 7.4 for 256, 322, 80 for 4,096.
    long long items = blocks(a->seqlen) * a->batch;
    p.run = 0;
    if (a->cu_seqlens != nullptr) {
        items = std::min<long long>(a->total, static_cast<long long>(a->total) / slots + 2ll * a->batch);
        if (a->batch > 256) {
            p.run = 1;
            while (p.run < slots && 4ll * p.run * a->batch <= a->total) p.run *= 2;
            items = (a->total + p.run - 1ll) / p.run;
        }
    }
    // Heads go over to CTAs of their own, four at least, which is a unit a warp, until the GPU has enough: 357 blocks of 8 heads as
    // 714 CTAs 35.6 us, as 357 36.7.
    const int heads = a->cache.heads_k;
    p.parts = static_cast<int>(std::min<long long>((heads + 3) / 4, std::max<long long>(1, 6ll * dev.sm_count / items)));
    p.part_heads = (heads + p.parts - 1) / p.parts;
    p.parts = (heads + p.part_heads - 1) / p.part_heads;
    p.seq_blocks = a->cu_seqlens == nullptr ? static_cast<int>(blocks(a->seqlen)) : 0;
    const int q_ctas = a->q != nullptr ? (a->total - 1) / kQTokens + 1 : 0;
    B2A_REQUIRE(items * p.parts + q_ctas < INT32_MAX, "too many tokens for a call");
    p.kv_ctas = static_cast<int>(items * p.parts);
    p.heads = heads;
    p.r.heads[1] = p.r.heads[2] = 0;
    cudaStream_t stream = static_cast<cudaStream_t>(cuda_stream);
    rc = once_per_device(dev.device, 17, set_append8_smem);
    if (rc != B2A_OK) return rc;
    const int most = std::min<int>(slots, a->cu_seqlens == nullptr ? a->seqlen : a->total);
    p.stages = most <= kTile8 && 2 * p.part_heads <= kRotaryThreads / 32 ? 1 : 2;
    const size_t smem = kRotaryThreads / 32 * p.stages * kStage8Bytes + (p.r.pairs > 0 ? most * 64 * sizeof(float2) : 0);
    B2A_CUDA_OK(launch_early(append8_tokens, 1 + p.kv_ctas + q_ctas, kRotaryThreads, smem, stream, p));
    return B2A_OK;
}

}  // extern "C"
