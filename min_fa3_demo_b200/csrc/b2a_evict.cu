// Eviction: of a sequence that has outgrown its budget each K/V head keeps its last `recent` slots and the heaviest of the
// others, and the cache is compacted in place.
//
// With L slots and m = budget, slots [0, m - recent) of the result hold the heaviest, [m - recent, m) the last ones in their
// order.  A heavy slot below m - recent stays where it is; the slots there that are not kept are filled, in ascending
// order, with the kept ones behind (attention does not ask in which order slots lie, and a step that drops one slot of thousands
// moves one row and the last few instead of half of the cache).
//
//   evict_select   one CTA a (sequence, head): the (m - recent)-th largest weight by radix selection on the bits (8 at a time,
//                  a histogram with a copy for each lane, so that equal digits do not queue up), ties to the lower slot,
//                  then the new order and the weights in it.  Bound by latency; weights come from L2 after the first pass.
//   evict_fill     moves the kept rows from behind into the gaps.  No gap is a source and no source a gap.  Bound by
//                  memory: 512 bytes in and out a row.
//   evict_shift    moves the last rows down.  They may overlap their destination, so then one CTA a head goes upwards, a
//                  chunk in registers at a time.  After evict_fill, whose sources it may overwrite.
#include "b2a_cache.cuh"

namespace b2a {

namespace {

constexpr int kSelectThreads = 1024;
constexpr int kMoveThreads = 256;
constexpr int kFillSlots = kMoveThreads;     // slots of a CTA of evict_fill
constexpr int kShiftRows = 64;               // rows in registers: 8 warps times 8

struct EvictParams {
    CacheView cache;
    const int* cache_lens;
    const float* weights;
    long long weights_stride[2];   // sequence, head
    int batch;
    int slots;                     // of a row of weights
    int budget;
    int recent;
    int* new_lens;
    float* new_weights;            // contiguous
    int* index;                    // [batch, heads, budget]
    int* movers;                   // [batch, heads, budget]
    WorkspaceHeader* header;
};

__device__ __forceinline__ long long evict_cap(const EvictParams& p) {
    return min(p.cache.capacity(), static_cast<long long>(p.slots));
}

__device__ __forceinline__ int evict_len(const EvictParams& p, int seq) {
    return static_cast<int>(min(max(static_cast<long long>(p.cache_lens[seq]), 0ll), evict_cap(p)));
}

// A weight's rank as an unsigned number: NaN above all, -0 as 0.
__device__ __forceinline__ uint32_t weight_key(float w) {
    if (w != w) return 0xFFFFFFFFu;
    const uint32_t bits = __float_as_uint(w + 0.f);
    return (bits & 0x80000000u) ? ~bits : bits | 0x80000000u;
}

// Lengths and pages: CTA 0 finds out whether all exist and writes the header, so that no launch has to clear it.
__device__ __forceinline__ void check_evict(const EvictParams& p, int* flag) {
    if (threadIdx.x == 0) *flag = 0;
    __syncthreads();
    for (int b = 0; b < p.batch; ++b) {
        const long long len = p.cache_lens[b];
        if (len < 0 || len > evict_cap(p)) *flag = 1;
        if (p.cache.block_table == nullptr) continue;
        const int pages = (evict_len(p, b) + p.cache.page_size - 1) / p.cache.page_size;
        for (int i = threadIdx.x; i < pages; i += kSelectThreads) {
            if (p.cache.page_of(b, static_cast<long long>(i) * p.cache.page_size) < 0) *flag = 1;
        }
    }
    __syncthreads();
    if (threadIdx.x == 0) *p.header = WorkspaceHeader{0, 0, *flag ? kStatusBadArg << 24 : 0u, 0};
}

// Exclusive sums of a value of each warp, in every thread; the total in *total.
__device__ __forceinline__ int warps_before(int mine, int warp, int lane, int* shared, int* total) {
    __syncthreads();
    if (lane == 0) shared[warp] = mine;
    __syncthreads();
    const int v = shared[lane];
    int upto = v;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int up = __shfl_up_sync(0xFFFFFFFFu, upto, d);
        if (lane >= d) upto += up;
    }
    *total = __shfl_sync(0xFFFFFFFFu, upto, 31);
    return __shfl_sync(0xFFFFFFFFu, upto - v, warp);
}

__global__ void __launch_bounds__(kSelectThreads)
evict_select(const EvictParams p) {
    __shared__ int count[256][32];
    __shared__ int bin_sum[256];
    __shared__ int per_warp[32];
    __shared__ int found[2];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    let_next_kernel_start();
    wait_for_previous_kernel();
    const int heads = p.cache.heads;
    const int seq = blockIdx.x / heads, head = blockIdx.x - seq * heads;
    const int len = evict_len(p, seq), keep = min(len, p.budget);
    const float* w = p.weights + seq * p.weights_stride[0] + head * p.weights_stride[1];
    float* new_w = p.new_weights + static_cast<long long>(blockIdx.x) * p.slots;
    int* index = p.index + static_cast<long long>(blockIdx.x) * p.budget;
    if (head == 0 && threadIdx.x == 0) p.new_lens[seq] = keep;
    for (int j = keep + threadIdx.x; j < p.slots; j += kSelectThreads) new_w[j] = 0.f;
    for (int j = keep + threadIdx.x; j < p.budget; j += kSelectThreads) index[j] = -1;
    if (len <= p.budget) {
        for (int j = threadIdx.x; j < keep; j += kSelectThreads) {
            new_w[j] = w[j];
            index[j] = j;
        }
    } else {
        const int old = p.budget - p.recent;         // slots for the heaviest
        const int candidates = len - p.recent;       // more than old
        // The last ones, in their order.
        for (int j = old + threadIdx.x; j < keep; j += kSelectThreads) {
            new_w[j] = w[j + len - keep];
            index[j] = j + len - keep;
        }
        // The key of the old-th heaviest, digit by digit, and how many of that key are kept.
        uint32_t key = 0;
        int need = old;
        for (int shift = 24; shift >= 0 && old > 0; shift -= 8) {
            for (int i = threadIdx.x; i < 256 * 32; i += kSelectThreads) count[i >> 5][i & 31] = 0;
            __syncthreads();
#pragma unroll 4
            for (int j = threadIdx.x; j < candidates; j += kSelectThreads) {
                const uint32_t k = weight_key(w[j]);
                if (shift == 24 || (k >> (shift + 8)) == key) atomicAdd(&count[(k >> shift) & 255u][lane], 1);
            }
            __syncthreads();
            if (threadIdx.x < 256) {
                int sum = 0;
#pragma unroll 8
                for (int i = 0; i < 32; ++i) sum += count[threadIdx.x][(threadIdx.x + i) & 31];
                bin_sum[threadIdx.x] = sum;
            }
            __syncthreads();
            if (warp == 0) {
                // A lane has 8 bins, the highest first.
                int mine = 0;
                for (int i = 0; i < 8; ++i) mine += bin_sum[255 - (lane * 8 + i)];
                int upto = mine;
#pragma unroll
                for (int d = 1; d < 32; d <<= 1) {
                    const int up = __shfl_up_sync(0xFFFFFFFFu, upto, d);
                    if (lane >= d) upto += up;
                }
                int above = upto - mine;
                if (above < need && upto >= need) {
                    for (int i = 0; i < 8; ++i) {
                        const int bin = 255 - (lane * 8 + i), n = bin_sum[bin];
                        if (above + n >= need) {
                            found[0] = bin;
                            found[1] = need - above;
                            break;
                        }
                        above += n;
                    }
                }
            }
            __syncthreads();
            key = (key << 8) | static_cast<uint32_t>(found[0]);
            need = found[1];
        }
        if (old > 0) {
            // A warp has a run of slots, so that sums over warps keep their order.
            const int run = ((candidates + 31) / 32 + 31) / 32 * 32;
            const int first = min(warp * run, candidates), last = min(first + run, candidates);
            int equal = 0, total;
            for (int j0 = first; j0 < last; j0 += 32) {
                const bool eq = j0 + lane < last && weight_key(w[j0 + lane]) == key;
                equal += __popc(__ballot_sync(0xFFFFFFFFu, eq));
            }
            const int equal_before = warps_before(equal, warp, lane, per_warp, &total);
            // Twice over the run: count the kept slots behind the heaviest's place, then list them.
            int* movers = p.movers + static_cast<long long>(blockIdx.x) * p.budget;
            const unsigned below = (1u << lane) - 1u;
            int at = 0, gap = 0;
            for (int pass = 0; pass < 2; ++pass) {
                int eq_seen = equal_before, n = 0, gaps = 0;
                for (int j0 = first; j0 < last; j0 += 32) {
                    const int j = j0 + lane;
                    const uint32_t k = j < last ? weight_key(w[j]) : 0u;
                    const bool eq = j < last && k == key;
                    const unsigned eqs = __ballot_sync(0xFFFFFFFFu, eq);
                    const bool kept = j < last && (k > key || (eq && eq_seen + __popc(eqs & below) < need));
                    eq_seen += __popc(eqs);
                    const unsigned moves = __ballot_sync(0xFFFFFFFFu, kept && j >= old);
                    if (pass == 1 && kept && j >= old) movers[at + n + __popc(moves & below)] = j;
                    n += __popc(moves);
                    gaps += __popc(__ballot_sync(0xFFFFFFFFu, !kept && j < last && j < old));
                }
                if (pass == 0) {
                    at = warps_before(n, warp, lane, per_warp, &total);
                    gap = warps_before(gaps, warp, lane, per_warp, &total);
                }
            }
            __threadfence_block();
            __syncthreads();
            int eq_seen = equal_before;
            for (int j0 = first; j0 < last && j0 < old; j0 += 32) {
                const int j = j0 + lane;
                const uint32_t k = j < last ? weight_key(w[j]) : 0u;
                const bool eq = j < last && k == key;
                const unsigned eqs = __ballot_sync(0xFFFFFFFFu, eq);
                const bool kept = j < last && (k > key || (eq && eq_seen + __popc(eqs & below) < need));
                eq_seen += __popc(eqs);
                const bool here = j < last && j < old;
                const unsigned gaps = __ballot_sync(0xFFFFFFFFu, here && !kept);
                if (here) {
                    const int from = kept ? j : movers[gap + __popc(gaps & below)];
                    index[j] = from;
                    new_w[j] = w[from];
                }
                gap += __popc(gaps);
            }
        }
    }
    if (blockIdx.x == 0) check_evict(p, found);
}

// Rows of K and V of one slot: the lower half of a warp has K, the upper V, 16 bytes a lane.
__device__ __forceinline__ uint4* evict_row(const EvictParams& p, int seq, int head, int slot, int lane) {
    const int page = p.cache.page_of(seq, slot);
    if (page < 0) return nullptr;
    const long long* st = lane < 16 ? p.cache.k_stride : p.cache.v_stride;
    return reinterpret_cast<uint4*>((lane < 16 ? p.cache.k : p.cache.v) + page * st[0] + slot % p.cache.page_size * st[1] +
                                    head * st[2] + (lane & 15) * 8);
}

__global__ void __launch_bounds__(kMoveThreads)
evict_fill(const EvictParams p) {
    let_next_kernel_start();
    wait_for_previous_kernel();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int which = blockIdx.y, seq = which / p.cache.heads, head = which - seq * p.cache.heads;
    if (evict_len(p, seq) <= p.budget) return;
    const int old = p.budget - p.recent;
    const int j0 = blockIdx.x * kFillSlots + warp * 32;
    if (j0 >= old) return;
    const int from = j0 + lane < old ? p.index[static_cast<long long>(which) * p.budget + j0 + lane] : j0 + lane;
    unsigned moves = __ballot_sync(0xFFFFFFFFu, from != j0 + lane);
    while (moves != 0u) {
        // Four rows at a time on the way.
        uint4 data[4];
        uint4* to[4];
        int n = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            to[i] = nullptr;
            if (moves != 0u) {
                const int at = __ffs(moves) - 1;
                moves &= moves - 1u;
                const uint4* src = evict_row(p, seq, head, __shfl_sync(0xFFFFFFFFu, from, at), lane);
                to[i] = src == nullptr ? nullptr : evict_row(p, seq, head, j0 + at, lane);
                if (to[i] != nullptr) data[i] = *src;
                ++n;
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (to[i] != nullptr) *to[i] = data[i];
        }
    }
}

__global__ void __launch_bounds__(kMoveThreads)
evict_shift(const EvictParams p) {
    let_next_kernel_start();
    wait_for_previous_kernel();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int which = blockIdx.y, seq = which / p.cache.heads, head = which - seq * p.cache.heads;
    const int by = evict_len(p, seq) - p.budget;
    if (by <= 0) return;
    const bool overlap = by < p.recent;
    if (overlap && blockIdx.x > 0) return;
    const int old = p.budget - p.recent;
    const int first = overlap ? 0 : blockIdx.x * kShiftRows, last = overlap ? p.recent : min(first + kShiftRows, p.recent);
    // Upwards: a chunk is written when all of it has been read, and what it overwrites lies below the next one's source.
    for (int r0 = first; r0 < last; r0 += kShiftRows) {
        uint4 data[8];
        uint4* to[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int r = r0 + warp * 8 + i;
            to[i] = nullptr;
            if (r < last) {
                const uint4* src = evict_row(p, seq, head, old + r + by, lane);
                to[i] = src == nullptr ? nullptr : evict_row(p, seq, head, old + r, lane);
                if (to[i] != nullptr) data[i] = *src;
            }
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (to[i] != nullptr) *to[i] = data[i];
        }
    }
}

}  // namespace

}  // namespace b2a

extern "C" {

size_t b2a_cache_evict_workspace_bytes(int32_t batch, int32_t heads_k, int32_t budget) {
    if (batch < 1 || heads_k < 1 || budget < 1) return 0;   // b2a_cache_evict reports what is wrong
    return 256 + static_cast<size_t>(batch) * heads_k * budget * sizeof(int);
}

int b2a_cache_evict(const b2a_evict_args* a, void* cuda_stream) {
    using namespace b2a;
    B2A_REQUIRE(a != nullptr, "args must not be NULL");
    EvictParams p{};
    B2A_REQUIRE(a->batch >= 1, "batch must be >= 1, got %d", a->batch);
    int rc = make_cache_view(a->cache, a->batch, true, &p.cache);
    if (rc != B2A_OK) return rc;
    B2A_REQUIRE(a->cache_lens && a->weights && a->new_lens && a->new_weights && a->index,
                "cache_lens, weights, new_lens, new_weights and index must not be NULL");
    B2A_REQUIRE(a->budget >= 1, "budget must be >= 1, got %d", a->budget);
    B2A_REQUIRE(a->recent >= 0 && a->recent <= a->budget, "recent must be between 0 and the budget, got %d", a->recent);
    B2A_REQUIRE(a->weights_slots >= 1, "weights_slots must be >= 1, got %d", a->weights_slots);
    B2A_REQUIRE(a->weights_stride[0] >= 0 && a->weights_stride[1] >= 0, "strides of weights must not be negative");
    const long long rows = static_cast<long long>(a->batch) * a->cache.heads_k;
    B2A_REQUIRE(rows <= 65535, "at most 65535 sequences times K/V heads, got %lld", rows);
    B2A_REQUIRE(a->workspace != nullptr && (reinterpret_cast<uintptr_t>(a->workspace) & 0xF) == 0,
                "workspace must be a 16-byte aligned device pointer");
    const size_t need = b2a_cache_evict_workspace_bytes(a->batch, a->cache.heads_k, a->budget);
    if (a->workspace_bytes < need) {
        return fail(B2A_ERR_WORKSPACE_TOO_SMALL, "workspace has %zu bytes, need %zu", a->workspace_bytes, need);
    }
    DeviceInfo dev{};
    rc = current_device_info(&dev);
    if (rc != B2A_OK) return rc;
    p.cache_lens = a->cache_lens;
    p.weights = a->weights;
    p.weights_stride[0] = a->weights_stride[0];
    p.weights_stride[1] = a->weights_stride[1];
    p.batch = a->batch;
    p.slots = a->weights_slots;
    p.budget = a->budget;
    p.recent = a->recent;
    p.new_lens = a->new_lens;
    p.new_weights = a->new_weights;
    p.index = a->index;
    p.header = static_cast<WorkspaceHeader*>(a->workspace);
    p.movers = reinterpret_cast<int*>(static_cast<uint8_t*>(a->workspace) + 256);
    cudaStream_t stream = static_cast<cudaStream_t>(cuda_stream);
    auto select = evict_select;
    auto fill = evict_fill;
    auto shift = evict_shift;
    B2A_CUDA_OK(launch_early(select, static_cast<unsigned int>(rows), kSelectThreads, 0, stream, p));
    // Nothing moves where no sequence can be longer than the budget.
    if (std::min<long long>(p.cache.block_table == nullptr ? p.cache.page_size : static_cast<long long>(p.cache.page_size) * p.cache.table_width,
                            p.slots) <= p.budget) {
        return B2A_OK;
    }
    const int old = p.budget - p.recent;
    if (old > 0) {
        B2A_CUDA_OK(launch_early(fill, dim3((old + kFillSlots - 1) / kFillSlots, rows), kMoveThreads, 0, stream, p));
    }
    if (p.recent > 0) {
        B2A_CUDA_OK(launch_early(shift, dim3((p.recent + kShiftRows - 1) / kShiftRows, rows), kMoveThreads, 0, stream, p));
    }
    return B2A_OK;
}

}  // extern "C"
