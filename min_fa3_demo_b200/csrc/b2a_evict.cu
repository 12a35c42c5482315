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
// Where only a few rows can move, evict_select does both itself.  What can is the smaller of the cache's and the weights' slots: 16
// sequences of 4,097 cut to 4,096 take 10.9 us with weights of 4,160 slots, 18.1, 20.1 and 23.4 with 8,192, 32,768 and 65,536.
// 8 sequences of up to 16,000 slots, 8 heads, cut to 4,000 with 250 recent ones: 57 us; each by itself, with cold caches, 23, 24 (128 MB
// moved, 5.3 TB/s) and 12.
#include "b2a_cache.cuh"

namespace b2a {

namespace {

constexpr int kSelectThreads = 1024;
constexpr int kSelectKeys = 45056;           // candidates whose keys fit in shared memory: 176 KiB beside the histogram's 33
constexpr int kMoveThreads = 256;
constexpr int kFillSlots = kMoveThreads;     // slots of a CTA of evict_fill
constexpr int kInsideRows = 512;             // up to which evict_select moves the rows itself
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
    uint32_t* stays;               // [batch * heads][slots / 32], where the keys do not fit in shared memory
    int* bad;                      // [batch]: the sequence's length or a page of it does not exist
    int report;                    // which launch writes the header: 0 evict_select, 1 evict_fill, 2 evict_shift, -1 see inside
    int inside;                    // few rows move: evict_select moves them, and `bad` holds a status word for each sequence
};

__device__ __forceinline__ long long evict_cap(const EvictParams& p) { return min(p.cache.capacity(), p.slots); }

__device__ __forceinline__ int evict_len(const EvictParams& p, int seq) {
    return static_cast<int>(min(max(static_cast<long long>(p.cache_lens[seq]), 0ll), evict_cap(p)));
}

// A weight's rank as an unsigned number: NaN above all, -0 as 0.
__device__ __forceinline__ uint32_t weight_key(float w) {
    if (w != w) return 0xFFFFFFFFu;
    const uint32_t bits = __float_as_uint(w + 0.f);
    return (bits & 0x80000000u) ? ~bits : bits | 0x80000000u;
}

// Whether a sequence's length and pages exist; by one CTA.
__device__ __forceinline__ void check_evict(const EvictParams& p, int seq) {
    const long long len = p.cache_lens[seq];
    int bad = len < 0 || len > evict_cap(p);
    if (p.cache.block_table != nullptr) {
        const int pages = (evict_len(p, seq) + p.cache.page_size - 1) / p.cache.page_size;
        for (int i = threadIdx.x; i < pages; i += blockDim.x) {
            int row;
            if (p.cache.page_of(seq, static_cast<long long>(i) * p.cache.page_size, &row) < 0) bad = 1;
        }
    }
    bad = __syncthreads_or(bad);
    if (threadIdx.x == 0) p.bad[seq] = bad ? kStatusBadArg << 24 : 0;
}

// The header, written whole by one CTA of the last launch, so that no launch has to clear it.  (Where only evict_select runs,
// nothing moves, and the lengths are all there is to check.)
__device__ __forceinline__ void report_evict(const EvictParams& p, int launch) {
    if (p.report != launch || blockIdx.x != 0 || blockIdx.y != 0) return;
    int bad = 0;
    for (int b = threadIdx.x; b < p.batch; b += blockDim.x) {
        bad |= launch == 0 ? p.cache_lens[b] < 0 || p.cache_lens[b] > evict_cap(p) : p.bad[b];
    }
    bad = __syncthreads_or(bad);
    if (threadIdx.x == 0) *p.header = WorkspaceHeader{0, 0, bad ? kStatusBadArg << 24 : 0u, 0};
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

// Moves up to 32 rows of K and V by one warp: a lane finds out where one row comes from and goes to, all at once, and then the
// warp copies row by row, kAtOnce on their way, the lower half of its lanes K, the upper V, 16 bytes each.
template <int kAtOnce, typename Sync>
__device__ __forceinline__ void evict_move(const EvictParams& p, int seq, int head, bool moves, int from, int to, int lane, Sync&& sync) {
    long long src[2] = {-1, -1}, dst[2] = {-1, -1};
    if (moves) {
        int row;
        int page = p.cache.page_of(seq, from, &row);
        src[0] = p.cache.at(p.cache.k_stride, page, row, head);
        src[1] = p.cache.at(p.cache.v_stride, page, row, head);
        page = p.cache.page_of(seq, to, &row);
        dst[0] = p.cache.at(p.cache.k_stride, page, row, head);
        dst[1] = p.cache.at(p.cache.v_stride, page, row, head);
        if (src[0] < 0 || dst[0] < 0) moves = false;
    }
    unsigned left = __ballot_sync(0xFFFFFFFFu, moves);
    __nv_bfloat16* base = (lane < 16 ? p.cache.k : p.cache.v) + (lane & 15) * 8;
    do {
        uint4 data[kAtOnce];
        __nv_bfloat16* put[kAtOnce];
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
            put[i] = nullptr;
            if (left != 0u) {
                const int at = __ffs(left) - 1;
                left &= left - 1u;
                const long long k_src = __shfl_sync(0xFFFFFFFFu, src[0], at), v_src = __shfl_sync(0xFFFFFFFFu, src[1], at);
                const long long k_dst = __shfl_sync(0xFFFFFFFFu, dst[0], at), v_dst = __shfl_sync(0xFFFFFFFFu, dst[1], at);
                put[i] = base + (lane < 16 ? k_dst : v_dst);
                data[i] = *reinterpret_cast<const uint4*>(base + (lane < 16 ? k_src : v_src));
            }
        }
        sync();
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
            if (put[i] != nullptr) *reinterpret_cast<uint4*>(put[i]) = data[i];
        }
    } while (left != 0u);
}

// in_shared: the keys of all candidates fit in shared memory; otherwise each pass reads the weights again.  Loops stay rolled up: a
// CTA goes through each once, and instructions that come from memory cost more than they save (keys in registers, eight passes
// over 16 each unrolled: 53 us where rolled ones took 32, 16,000 slots of 64 heads).
__global__ void __launch_bounds__(kSelectThreads)
evict_select(const EvictParams p, const int in_shared) {
    extern __shared__ uint32_t keys[];
    __shared__ int count[256][32];
    __shared__ int bin_sum[256];
    __shared__ int per_warp[32];
    __shared__ int found[3];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    let_next_kernel_start();
    wait_for_previous_kernel();
    const int heads = p.cache.heads;
    const int seq = blockIdx.x / heads, head = blockIdx.x - seq * heads;
    const int len = evict_len(p, seq), keep = min(len, p.budget);
    const float* w = p.weights + seq * p.weights_stride[0] + head * p.weights_stride[1];
    float* new_w = p.new_weights + static_cast<long long>(blockIdx.x) * p.slots;
    int* index = p.index + static_cast<long long>(blockIdx.x) * p.budget;
    const int old = p.budget - p.recent;         // slots for the heaviest
    const int candidates = len - p.recent;       // more than old, if the sequence is too long
    // A warp has a run of slots, so that sums over warps keep their order.
    const int run = ((candidates + 31) / 32 + 31) / 32 * 32;
    const int first = min(warp * run, candidates), last = min(first + run, candidates);
    uint32_t* stays = in_shared ? keys + candidates : p.stays + static_cast<long long>(blockIdx.x) * ((p.slots + 31) / 32);
    if (in_shared && len > p.budget) {
        // Only the warp itself reads them again.
#pragma unroll 4
        for (int j = first + lane; j < last; j += 32) keys[j] = weight_key(w[j]);
        __syncwarp();
    }
    auto each = [&](auto&& take) {               // take(first of 32 slots, this lane's key)
#pragma unroll 1
        for (int j0 = first; j0 < last; j0 += 32) {
            take(j0, j0 + lane >= last ? 0u : in_shared ? keys[j0 + lane] : weight_key(w[j0 + lane]));
        }
    };
    if (head == 0 && threadIdx.x == 0) p.new_lens[seq] = keep;
    for (int j = keep + threadIdx.x; j < p.slots; j += kSelectThreads) new_w[j] = 0.f;
    for (int j = keep + threadIdx.x; j < p.budget; j += kSelectThreads) index[j] = -1;
    if (len <= p.budget) {
        for (int j = threadIdx.x; j < keep; j += kSelectThreads) {
            new_w[j] = w[j];
            index[j] = j;
        }
    } else {
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
            each([&](int j0, uint32_t k) {
                if (j0 + lane < last && (shift == 24 || (k >> (shift + 8)) == key)) atomicAdd(&count[(k >> shift) & 255u][lane], 1);
            });
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
                            found[2] = n;
                            break;
                        }
                        above += n;
                    }
                }
            }
            __syncthreads();
            key = (key << 8) | static_cast<uint32_t>(found[0]);
            need = found[1];
            if (need == found[2]) {              // all with these digits stay: the others do not matter (mostly so after three)
                key <<= shift;
                break;
            }
        }
        if (old > 0) {
            const unsigned below = (1u << lane) - 1u;
            int equal_before = 0, total;
            const bool ties = need < found[2];             // not all slots of the last key stay: the lower ones do
            if (ties) {
                int equal = 0;
                each([&](int j0, uint32_t k) { equal += __popc(__ballot_sync(0xFFFFFFFFu, j0 + lane < last && k == key)); });
                equal_before = warps_before(equal, warp, lane, per_warp, &total);
            }
            // A bit for each slot that stays; those behind the heaviest's place and the gaps in it are counted.
            int moves = 0, gaps = 0;
            each([&](int j0, uint32_t k) {
                bool yes = j0 + lane < last && k >= key;
                if (ties) {
                    const bool eq = j0 + lane < last && k == key;
                    const unsigned eqs = __ballot_sync(0xFFFFFFFFu, eq);
                    yes = yes && (!eq || equal_before + __popc(eqs & below) < need);
                    equal_before += __popc(eqs);
                }
                const unsigned stay = __ballot_sync(0xFFFFFFFFu, yes);
                const unsigned here = old - j0 >= 32 ? 0xFFFFFFFFu : old <= j0 ? 0u : (1u << (old - j0)) - 1u;
                if (lane == 0) stays[j0 >> 5] = stay;
                moves += __popc(stay & ~here);
                gaps += __popc(~stay & here);
            });
            int at = warps_before(moves, warp, lane, per_warp, &total);
            int gap = warps_before(gaps, warp, lane, per_warp, &total);
            int* movers = p.movers + static_cast<long long>(blockIdx.x) * p.budget;
#pragma unroll 1
            for (int j0 = max(first, old & ~31); j0 < last; j0 += 32) {
                const unsigned all = stays[j0 >> 5] & (old <= j0 ? 0xFFFFFFFFu : 0xFFFFFFFFu << (old - j0));
                if ((all >> lane) & 1u) movers[at + __popc(all & below)] = j0 + lane;
                at += __popc(all);
            }
            __threadfence_block();
            __syncthreads();
#pragma unroll 2
            for (int j0 = first; j0 < min(last, old); j0 += 32) {
                const unsigned stay = stays[j0 >> 5];
                if (j0 + lane < old) {
                    const int from = (stay >> lane) & 1u ? j0 + lane : movers[gap + __popc(~stay & below)];
                    index[j0 + lane] = from;
                    new_w[j0 + lane] = w[from];
                }
                gap += __popc(~stay);                       // the last group's count is not used again
            }
        }
    }
    if (head == 0) check_evict(p, seq);
    report_evict(p, 0);
    if (!p.inside) return;
    if (blockIdx.x == 0 && threadIdx.x == 0) *p.header = WorkspaceHeader{-p.batch, 0, 0u, 0};
    const int by = len - p.budget;
    if (by <= 0) return;
    // What evict_fill and evict_shift do, by this CTA.
    __threadfence_block();
    __syncthreads();
    for (int j0 = warp * 32; j0 < old; j0 += kSelectThreads) {
        const int j = j0 + lane, from = j < old ? index[j] : j;
        if (__any_sync(0xFFFFFFFFu, from != j)) evict_move<4>(p, seq, head, from != j, from, j, lane, [] {});
    }
    __syncthreads();
    for (int r0 = 0; r0 < p.recent; r0 += kSelectThreads / 8) {
        const int r = r0 + warp * 4 + lane;
        evict_move<4>(p, seq, head, lane < 4 && r < p.recent, old + r + by, old + r, lane, [] { __syncthreads(); });
    }
}

__global__ void __launch_bounds__(kMoveThreads)
evict_fill(const EvictParams p) {
    let_next_kernel_start();
    wait_for_previous_kernel();
    report_evict(p, 1);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int which = blockIdx.y, seq = which / p.cache.heads, head = which - seq * p.cache.heads;
    if (evict_len(p, seq) <= p.budget) return;
    const int old = p.budget - p.recent;
    const int j = blockIdx.x * kFillSlots + threadIdx.x;
    if (blockIdx.x * kFillSlots + warp * 32 >= old) return;
    const int from = j < old ? p.index[static_cast<long long>(which) * p.budget + j] : j;
    evict_move<8>(p, seq, head, from != j, from, j, lane, [] {});
}

__global__ void __launch_bounds__(kMoveThreads)
evict_shift(const EvictParams p) {
    let_next_kernel_start();
    wait_for_previous_kernel();
    report_evict(p, 2);
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
        const int r = r0 + warp * 8 + lane;
        evict_move<8>(p, seq, head, lane < 8 && r < last, old + r + by, old + r, lane, [] { __syncthreads(); });
    }
}

// Workspace: the header and a word for each sequence, which are kept after a call, then the movers, and a bit for each slot.
size_t evict_kept(int batch) { return align_up(sizeof(WorkspaceHeader) + batch * sizeof(int), 256); }
size_t evict_stays_at(size_t rows, int budget) { return align_up(rows * budget * sizeof(int), 256); }
size_t evict_scratch(size_t rows, int budget, int slots) {
    return evict_stays_at(rows, budget) + rows * ((static_cast<size_t>(slots) + 31) / 32) * sizeof(uint32_t);
}

size_t select_smem(long long candidates) { return (candidates + (candidates + 31) / 32) * sizeof(uint32_t); }   // keys, and a bit for each

int set_select_smem() {
    B2A_CUDA_OK(cudaFuncSetAttribute(evict_select, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     static_cast<int>(select_smem(kSelectKeys))));
    return B2A_OK;
}

}  // namespace

}  // namespace b2a

extern "C" {

size_t b2a_cache_evict_workspace_bytes(int32_t batch, int32_t heads_k, int32_t budget, int32_t weights_slots) {
    if (batch < 1 || heads_k < 1 || budget < 1 || weights_slots < 1) return 0;   // b2a_cache_evict reports what is wrong
    return b2a::evict_kept(batch) + b2a::evict_scratch(static_cast<size_t>(batch) * heads_k, budget, weights_slots);
}

size_t b2a_cache_evict_kept_workspace_bytes(int32_t batch) { return batch < 1 ? 0 : b2a::evict_kept(batch); }

int b2a_cache_evict(const b2a_evict_args* a, void* cuda_stream) {
    using namespace b2a;
    B2A_REQUIRE(a != nullptr, "args must not be NULL");
    B2A_REQUIRE(a->batch >= 1, "batch must be >= 1, got %d", a->batch);
    B2A_REQUIRE(a->workspace != nullptr && (reinterpret_cast<uintptr_t>(a->workspace) & 0xF) == 0,
                "workspace must be a 16-byte aligned device pointer");
    const size_t kept = evict_kept(a->batch), behind = a->workspace_bytes > kept ? a->workspace_bytes - kept : 0;
    return b2a_cache_evict_with_scratch(a, static_cast<uint8_t*>(a->workspace) + kept, behind, cuda_stream);
}

int b2a_cache_evict_with_scratch(const b2a_evict_args* a, void* scratch, size_t scratch_bytes, void* cuda_stream) {
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
    B2A_REQUIRE(scratch != nullptr && (reinterpret_cast<uintptr_t>(scratch) & 0xF) == 0,
                "scratch must be a 16-byte aligned device pointer");
    const size_t kept = evict_kept(a->batch), need = evict_scratch(static_cast<size_t>(rows), a->budget, a->weights_slots);
    if (a->workspace_bytes < kept) {
        return fail(B2A_ERR_WORKSPACE_TOO_SMALL, "workspace has %zu bytes, need %zu", a->workspace_bytes, kept);
    }
    if (scratch_bytes < need) return fail(B2A_ERR_WORKSPACE_TOO_SMALL, "scratch has %zu bytes, need %zu", scratch_bytes, need);
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
    uint8_t* ws = static_cast<uint8_t*>(a->workspace);
    p.bad = reinterpret_cast<int*>(ws + sizeof(WorkspaceHeader));
    p.movers = static_cast<int*>(scratch);
    p.stays = reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(scratch) + evict_stays_at(static_cast<size_t>(rows), a->budget));
    cudaStream_t stream = static_cast<cudaStream_t>(cuda_stream);
    const long long most = std::min<long long>(p.cache.block_table == nullptr ? p.cache.page_size
                                                                              : static_cast<long long>(p.cache.page_size) * p.cache.table_width,
                                               p.slots);
    const bool in_shared = most - p.recent <= kSelectKeys;
    rc = once_per_device(dev.device, 11, set_select_smem);
    if (rc != B2A_OK) return rc;
    const int old = p.budget - p.recent;
    // Where few rows move, one launch instead of three.  Us with one and with three, 8 heads, 4,096 slots kept; of 4 sequences 65 rows
    // move: 10.1, 13.2; 512: 18.6, 17.5; 1,024: 25.2, 20.5; of 16 sequences 10.2, 17.9; 24.5, 29.0; 33.3, 36.4.
    p.inside = most > p.budget && most - p.budget + p.recent <= kInsideRows && p.batch <= kFwdStatusWords;
    p.report = p.inside ? -1 : most <= p.budget ? 0 : p.recent > 0 ? 2 : 1;
    auto select = evict_select;
    auto fill = evict_fill;
    auto shift = evict_shift;
    B2A_CUDA_OK(launch_early(select, static_cast<unsigned int>(rows), kSelectThreads,
                             in_shared && most > p.recent ? select_smem(most - p.recent) : 0, stream, p, in_shared ? 1 : 0));
    // Nothing moves where no sequence can be longer than the budget.
    if (most <= p.budget || p.inside) return B2A_OK;
    if (old > 0) {
        B2A_CUDA_OK(launch_early(fill, dim3((old + kFillSlots - 1) / kFillSlots, rows), kMoveThreads, 0, stream, p));
    }
    if (p.recent > 0) {
        B2A_CUDA_OK(launch_early(shift, dim3((p.recent + kShiftRows - 1) / kShiftRows, rows), kMoveThreads, 0, stream, p));
    }
    return B2A_OK;
}

}  // extern "C"
