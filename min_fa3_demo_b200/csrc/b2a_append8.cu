// New keys and values into a cache in 8 bits, turned by their positions on the way.
//
// All slots of a block share a head's scale, so a block's new tokens belong to one group of threads: 128 of a CTA for K, 128 for V, eight
// threads a token with 16 dimensions each, as in b2a_rotary.cu.  They turn the values in fp32, look for the largest, find the
// scale, and round.  e4m3 is a floating-point format, so a scale that is a power of two costs no accuracy (values keep
// their four bits down to 2^-15 of the largest), divides exactly, and can grow with hardly a trace: x / 2 is a number of the
// format as well, unless it is one of the smallest.  So a block whose tokens come one by one keeps its scale until a
// token does not fit, and then the tokens that it holds are read, divided and written again, at most 127 of 128 bytes.
//
// Bound by memory: 256 bytes in and 128 out a token and head.  The CTAs of K and V come first, a block of slots and some of the heads
// each; those behind them turn q.
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
    int seq_blocks;              // most blocks of a sequence
};

// A block of slots that new tokens fall into.
struct Append8Block {
    int seq, token;              // the first of them: its number within the sequence, and
    int q_begin;                 // the row of the sequence's first
    int count;                   // of them; 0: there is nothing to do
    int held;                    // tokens before them
    int page, row;               // of the block's first slot
};

__device__ __forceinline__ Append8Block append8_block(const RotaryParams& p, const CacheScales& s, int item, int seq_blocks, int lane) {
    Append8Block at{};
    auto tokens_of = [&](int b, int* begin) -> int {
        *begin = b * p.seqlen;
        if (p.cu_seqlens == nullptr) return p.seqlen;
        *begin = p.cu_seqlens[b];
        const int end = p.cu_seqlens[b + 1];
        return *begin < 0 || end < *begin || end > p.total ? 0 : end - *begin;
    };
    const int mask = (1 << s.shift) - 1;
    // Blocks that a sequence's new tokens touch.
    auto blocks_of = [&](int b) -> int {
        if (b >= p.batch) return 0;
        int begin;
        const int n = tokens_of(b, &begin), len = p.cache_lens[b];
        return n <= 0 || len < 0 ? 0 : static_cast<int>(((len & mask) + static_cast<long long>(n) - 1) >> s.shift) + 1;
    };
    int j = 0;
    if (p.cu_seqlens == nullptr) {
        at.seq = item / seq_blocks;
        j = item - at.seq * seq_blocks;
        if (j >= blocks_of(at.seq)) return at;
    } else {
        int before = 0, found = -1;
        for (int b = 0; b < p.batch && found < 0; b += 32) {
            const int mine = blocks_of(b + lane);
            int upto = mine;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int up = __shfl_up_sync(0xFFFFFFFFu, upto, d);
                if (lane >= d) upto += up;
            }
            const unsigned hit = __ballot_sync(0xFFFFFFFFu, before + upto > item);
            if (hit != 0u) {
                const int l = __ffs(hit) - 1;
                found = b + l;
                before += __shfl_sync(0xFFFFFFFFu, upto - mine, l);
            } else {
                before += __shfl_sync(0xFFFFFFFFu, upto, 31);
            }
        }
        if (found < 0) return at;
        at.seq = found;
        j = item - before;
    }
    const int n = tokens_of(at.seq, &at.q_begin), len = p.cache_lens[at.seq];
    const long long begin = ((static_cast<long long>(len) >> s.shift) + j) << s.shift;
    const long long first = max(begin, static_cast<long long>(len));
    const long long last = min(min(begin + mask + 1, static_cast<long long>(len) + n), static_cast<long long>(p.cache.capacity()));
    at.page = p.cache.page_of(at.seq, begin, &at.row);
    if (at.page < 0 || last <= first) return at;
    at.token = static_cast<int>(first - len);
    at.held = static_cast<int>(first - begin);
    at.count = static_cast<int>(last - first);
    return at;
}

// The smallest power of two, within 2^-64 .. 2^64, of which `most` is at most 448 times: 448 = 1.75 * 2^8.
__device__ __forceinline__ float scale_for(float most) {
    const int bits = __float_as_int(most);
    const int e = (bits >> 23) - 8 + ((bits & 0x7FFFFF) > 0x600000 ? 1 : 0);
    return __int_as_float(min(max(e, 127 - 64), 127 + 64) << 23);
}

// Values divided by a scale: a power of two has an exact reciprocal.
struct Divider {
    float scale, inverse;
    __device__ __forceinline__ explicit Divider(float s) {
        scale = s;
        inverse = (__float_as_int(s) & 0x7FFFFF) == 0 ? 1.f / s : 0.f;
    }
    __device__ __forceinline__ float operator()(float x) const { return inverse != 0.f ? x * inverse : x / scale; }
};

// Eight values in e4m3; those that are not finite as NaN.
__device__ __forceinline__ uint2 pack8(const float* x, const Divider& by) {
    uint32_t two[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float a = by(x[2 * i]), b = by(x[2 * i + 1]);
        two[i] = pack_e4m3x2(fabsf(x[2 * i]) < INFINITY ? a : NAN, fabsf(x[2 * i + 1]) < INFINITY ? b : NAN);
    }
    return make_uint2(two[0] | two[1] << 16, two[2] | two[3] << 16);
}

// kTiles: of 16 tokens, as many as a block may get.
template <int kTiles>
__global__ void __launch_bounds__(kRotaryThreads, kTiles <= 2 ? 4 : 2)
append8_tokens(const __grid_constant__ Append8Params p8) {
    extern __shared__ __align__(16) float2 cos_sin[];      // [kTiles * 16][64]
    __shared__ Append8Block block;
    __shared__ float most_of[2][2][4];                     // turn, K or V, warp
    const RotaryParams& p = p8.r;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    let_next_kernel_start();
    wait_for_previous_kernel();

    if (blockIdx.x >= p8.kv_ctas) {
        turn_tokens<false, 1>(p, blockIdx.x - p8.kv_ctas);
    } else {
        if (warp == 0) {
            const Append8Block at = append8_block(p, p8.scales, blockIdx.x / p8.parts, p8.seq_blocks, lane);
            if (lane == 0) block = at;
        }
        __syncthreads();
        const Append8Block at = block;
        if (p.pairs > 0) {
            for (int i = threadIdx.x; i < at.count * 64; i += kRotaryThreads) {
                const int pair = i & 63, number = at.token + (i >> 6);
                // Packed tokens are one sequence to the positions.
                if (pair < p.pairs) {
                    cos_sin[i] = p.cu_seqlens == nullptr ? pair_angle(p, pair, at.seq, number) : pair_angle(p, pair, 0, at.q_begin + number);
                }
            }
        }
        __syncthreads();

        // A thread's 16 dimensions, as in turn_tokens: of V, and behind the pairs, 16 in a row.
        const int which = warp >> 2, c = lane & 7, mine = (threadIdx.x & 127) >> 3;
        const int pairs = which == 0 ? p.pairs : 0;
        const bool adjacent = which == 0 && p.adjacent && pairs > 0, turned = !adjacent && c * 8 < pairs;
        const int lo = adjacent || turned ? 8 * c : 16 * c;
        const int hi = adjacent ? 64 + 8 * c : turned ? pairs + 8 * c : 16 * c + 8;
        const int h0 = (blockIdx.x % p8.parts) * p8.part_heads, h1 = min(h0 + p8.part_heads, p8.heads);
        const long long* stride = p.stride[1 + which];
        const __nv_bfloat16* src = p.src[1 + which] + (p.cu_seqlens == nullptr ? at.seq * stride[0] + at.token * stride[1]
                                                                               : (static_cast<long long>(at.q_begin) + at.token) * stride[1]);
        const long long* to_stride = which == 0 ? p.cache.k_stride : p.cache.v_stride;
        uint8_t* dst = reinterpret_cast<uint8_t*>(which == 0 ? p.cache.k : p.cache.v);
        float* scales = which == 0 ? p8.scales.k : p8.scales.v;
        if (at.count > 0) {
            dst += at.page * to_stride[0] + at.row * to_stride[1];
            scales += p8.scales.at(which == 0 ? p8.scales.k_stride : p8.scales.v_stride, at.page, at.row, 0);
        }
        const long long scale_step = which == 0 ? p8.scales.k_stride[2] : p8.scales.v_stride[2];

        uint4 a[kTiles], b[kTiles];
        auto load = [&](int h) {
#pragma unroll
            for (int t = 0; t < kTiles; ++t) {
                a[t] = b[t] = make_uint4(0u, 0u, 0u, 0u);
                if (t * 16 + mine < at.count) {
                    const __nv_bfloat16* from = src + (t * 16 + mine) * stride[1] + h * stride[2];
                    a[t] = *reinterpret_cast<const uint4*>(from + lo);
                    b[t] = *reinterpret_cast<const uint4*>(from + hi);
                }
            }
        };
        // The values of a token, in the order of lo and hi.
        auto values = [&](int t, float (&x)[16]) {
            const uint32_t u[4] = {a[t].x, a[t].y, a[t].z, a[t].w}, w[4] = {b[t].x, b[t].y, b[t].z, b[t].w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float2 f = bf16x2_to_float2(u[e]), g = bf16x2_to_float2(w[e]);
                x[2 * e] = f.x;
                x[2 * e + 1] = f.y;
                x[8 + 2 * e] = g.x;
                x[9 + 2 * e] = g.y;
            }
            const float2* cs = cos_sin + (t * 16 + mine) * 64;
            if (t * 16 + mine >= at.count) return;
            if (adjacent) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int pair = e < 4 ? 4 * c + e : 28 + 4 * c + e;
                    if (pair >= pairs) continue;
                    const float2 t2 = cs[pair];
                    const float x0 = x[2 * e], x1 = x[2 * e + 1];
                    x[2 * e] = x0 * t2.x - x1 * t2.y;
                    x[2 * e + 1] = x1 * t2.x + x0 * t2.y;
                }
            } else if (turned) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float2 t2 = cs[8 * c + e];
                    const float x0 = x[e], x1 = x[8 + e];
                    x[e] = x0 * t2.x - x1 * t2.y;
                    x[8 + e] = x1 * t2.x + x0 * t2.y;
                }
            }
        };
        if (h0 < h1) load(h0);
#pragma unroll 1
        for (int h = h0; h < h1 && at.count > 0; ++h) {
            const float before = at.held > 0 ? scales[h * scale_step] : 0.f;
            float most = 0.f;
#pragma unroll
            for (int t = 0; t < kTiles; ++t) {
                float x[16];
                values(t, x);
#pragma unroll
                for (int e = 0; e < 16; ++e) most = fmaxf(most, fabsf(x[e]) < INFINITY ? fabsf(x[e]) : 0.f);
            }
            most = __int_as_float(__reduce_max_sync(0xFFFFFFFFu, __float_as_int(most)));      // not negative: ordered as integers
            if (lane == 0) most_of[h & 1][which][warp & 3] = most;
            named_barrier_sync(1 + which, 128);
            const float* parts = most_of[h & 1][which];
            most = fmaxf(fmaxf(parts[0], parts[1]), fmaxf(parts[2], parts[3]));
            const bool keep = at.held > 0 && most <= 448.f * before;
            const float scale = keep ? before : scale_for(most);
            const Divider by(scale);
            uint8_t* rows = dst + h * to_stride[2];
#pragma unroll
            for (int t = 0; t < kTiles; ++t) {
                const int token = t * 16 + mine;
                if (token >= at.count) continue;
                float x[16];
                values(t, x);
                uint8_t* row = rows + (at.held + token) * to_stride[1];
                const uint2 first = pack8(x, by), second = pack8(x + 8, by);
                if (hi == lo + 8) {
                    *reinterpret_cast<uint4*>(row + lo) = make_uint4(first.x, first.y, second.x, second.y);
                } else {
                    *reinterpret_cast<uint2*>(row + lo) = first;
                    *reinterpret_cast<uint2*>(row + hi) = second;
                }
            }
            if (h + 1 < h1) load(h + 1);
            if (!keep) {
                // Tokens that the block held.
                const Divider again(scale / before);
                for (int token = mine; token < at.held; token += 16) {
                    uint4* row = reinterpret_cast<uint4*>(rows + token * to_stride[1] + c * 16);
                    const uint4 v = *row;
                    const uint32_t words[4] = {v.x, v.y, v.z, v.w};
                    uint32_t out[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float2 f = e4m3x2_to_float2(words[e] & 0xFFFFu), g = e4m3x2_to_float2(words[e] >> 16);
                        out[e] = pack_e4m3x2(again(f.x), again(f.y)) | pack_e4m3x2(again(g.x), again(g.y)) << 16;
                    }
                    *row = make_uint4(out[0], out[1], out[2], out[3]);
                }
                if ((threadIdx.x & 127) == 0) scales[h * scale_step] = scale;
            }
        }
    }
    if (blockIdx.x == 0) check_append(p);
}

template <int kTiles>
int set_append8_smem() {
    B2A_CUDA_OK(cudaFuncSetAttribute(append8_tokens<kTiles>, cudaFuncAttributeMaxDynamicSharedMemorySize, kTiles * 16 * 64 * static_cast<int>(sizeof(float2))));
    return B2A_OK;
}

template <int kTiles>
int launch_append8(const Append8Params& p, int ctas, const DeviceInfo& dev, int slot, cudaStream_t stream) {
    const int rc = once_per_device(dev.device, slot, set_append8_smem<kTiles>);
    if (rc != B2A_OK) return rc;
    auto kernel = append8_tokens<kTiles>;
    const size_t smem = p.r.pairs > 0 ? kTiles * 16 * 64 * sizeof(float2) : 0;
    B2A_CUDA_OK(launch_early(kernel, ctas, kRotaryThreads, smem, stream, p));
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
    const long long items = a->cu_seqlens == nullptr ? blocks(a->seqlen) * a->batch
                                                     : std::min<long long>(a->total, static_cast<long long>(a->total) / slots + 2ll * a->batch);
    // Heads go over to CTAs of their own until the GPU has enough.
    const int heads = a->cache.heads_k;
    p.parts = static_cast<int>(std::min<long long>(heads, std::max<long long>(1, 4ll * dev.sm_count / items)));
    p.part_heads = (heads + p.parts - 1) / p.parts;
    p.parts = (heads + p.part_heads - 1) / p.part_heads;
    p.seq_blocks = a->cu_seqlens == nullptr ? static_cast<int>(blocks(a->seqlen)) : 0;
    const int q_ctas = a->q != nullptr ? a->total : 0;
    B2A_REQUIRE(items * p.parts + q_ctas <= INT32_MAX, "too many tokens for a call");
    p.kv_ctas = static_cast<int>(items * p.parts);
    p.heads = heads;
    p.r.heads[1] = p.r.heads[2] = 0;
    cudaStream_t stream = static_cast<cudaStream_t>(cuda_stream);
    const int most = std::min<int>(slots, a->cu_seqlens == nullptr ? a->seqlen : a->total), ctas = p.kv_ctas + q_ctas;
    if (most <= 16) return launch_append8<1>(p, ctas, dev, 17, stream);
    if (most <= 32) return launch_append8<2>(p, ctas, dev, 18, stream);
    if (most <= 64) return launch_append8<4>(p, ctas, dev, 19, stream);
    return launch_append8<8>(p, ctas, dev, 20, stream);
}

}  // extern "C"
