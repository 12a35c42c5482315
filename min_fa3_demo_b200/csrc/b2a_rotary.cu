// Rotary positions with several axes, on their own and on the way into the cache.
//
// A pair (x1, x2) of a head's dimensions is turned by the angle a = position * frequency:
//   y1 = m (x1 cos a - x2 sin a),  y2 = m (x2 cos a + x1 sin a)
// and the gradient is the same with -a.  m is 1, or what stretched frequencies want the turned dimensions multiplied by.  All heads
// of a token share the 64 angles.
//
// Far positions: a product of a position of a million and a frequency in 32 bits is off by 0.06.  The frequency comes as the
// fraction of a turn that one position makes, in units of 2^-64, so that position * turn mod 2^64 is the fraction of a turn
// that is left over; its upper 32 bits go to sincospif, as a float.  One 64-bit integer product, no reduction.  The float's 24 bits
// leave the angle within 1.1e-7 for positions up to 2^36; the frequency's own rounding, half of 2^-64 of a turn, adds 1.7e-19 for each
// position (2^45: 6e-6, a bf16 result's rounding is 4e-3).
//
// Bound by memory: 256 bytes in and out a token and head.  A CTA takes a few tokens, computes their angles once into shared
// memory, and its threads then go over the heads, eight to a head with two 16-byte loads each.  32,760 tokens of 32 + 8 heads: 672 MB
// in 110 us, 6.1 TB/s; 8 x 1,024 of 16 + 16: 134 MB in 28 us, 4.9 TB/s; 5,647 new tokens of 4 sequences with q, k and v, 32 + 8 + 8
// heads, into pages of 16 slots: 139 MB in 28.7 us.
#include "b2a_rotary.cuh"

namespace b2a {

namespace {

// Loads in flight against registers: 3, 4, 5, 6, 7 CTAs an SM take 129, 115, 111, 124, 145 us for 32,760 tokens of 32 + 8 heads.
template <bool kAppend, int kTokens>
__global__ void __launch_bounds__(kRotaryThreads, 5)
rotary_tokens(const RotaryParams p) {
    let_next_kernel_start();
    wait_for_previous_kernel();
    turn_tokens<kAppend, kTokens>(p, blockIdx.x);
    if (kAppend && blockIdx.x == 0) check_append(p);
}

// Four tokens a CTA where that fills the GPU, one where there are few: 16 tokens are then 16 CTAs' work instead of four's.  Us
// with four and with one, 32 + 8 heads: 1 token 4.1, 3.2; 64 4.7, 3.3; 1,184 9.4, 8.2; 2,368 12.1, 14.8; 9,472 37.5, 51.8.
template <bool kAppend>
int launch_rotary(const RotaryParams& p, const DeviceInfo& dev, cudaStream_t stream) {
    if (p.total >= 12 * dev.sm_count) {
        auto kernel = rotary_tokens<kAppend, 4>;
        B2A_CUDA_OK(launch_early(kernel, (p.total + 3) / 4, kRotaryThreads, 0, stream, p));
    } else {
        auto kernel = rotary_tokens<kAppend, 1>;
        B2A_CUDA_OK(launch_early(kernel, p.total, kRotaryThreads, 0, stream, p));
    }
    return B2A_OK;
}

}  // namespace

}  // namespace b2a

extern "C" {

int b2a_rotary(const b2a_rotary_args* a, void* cuda_stream) {
    using namespace b2a;
    B2A_REQUIRE(a != nullptr, "args must not be NULL");
    B2A_REQUIRE(a->axes != nullptr, "axes must not be NULL");
    B2A_REQUIRE(a->batch >= 1 && a->seqlen >= 1 && static_cast<long long>(a->batch) * a->seqlen <= INT32_MAX,
                "batch and seqlen must be positive and have fewer than 2^31 tokens");
    B2A_REQUIRE(a->heads_q >= 1 && a->heads_k >= 0, "heads_q must be positive");
    RotaryParams p{};
    int rc = set_axes(p, *a->axes, a->positions, a->positions_64, a->positions_stride, a->inverse != 0);
    if (rc == B2A_OK) rc = set_source(p, 0, a->q, a->q_stride, a->heads_q, "q");
    if (rc == B2A_OK && a->heads_k > 0) rc = set_source(p, 1, a->k, a->k_stride, a->heads_k, "k");
    if (rc != B2A_OK) return rc;
    B2A_REQUIRE(a->q_out != nullptr && (a->heads_k == 0 || a->k_out != nullptr), "q_out and k_out must not be NULL");
    B2A_REQUIRE(((reinterpret_cast<uintptr_t>(a->q_out) | reinterpret_cast<uintptr_t>(a->k_out)) & 0xF) == 0,
                "q_out and k_out must be 16-byte aligned");
    p.dst[0] = static_cast<__nv_bfloat16*>(a->q_out);
    p.dst[1] = static_cast<__nv_bfloat16*>(a->k_out);
    p.batch = a->batch;
    p.seqlen = a->seqlen;
    p.total = a->batch * a->seqlen;
    DeviceInfo dev{};
    rc = current_device_info(&dev);
    return rc != B2A_OK ? rc : launch_rotary<false>(p, dev, static_cast<cudaStream_t>(cuda_stream));
}

int b2a_cache_append(const b2a_append_args* a, void* cuda_stream) {
    using namespace b2a;
    B2A_REQUIRE(a != nullptr, "args must not be NULL");
    RotaryParams p{};
    int rc = make_append(*a, p);
    if (rc != B2A_OK) return rc;
    DeviceInfo dev{};
    rc = current_device_info(&dev);
    return rc != B2A_OK ? rc : launch_rotary<true>(p, dev, static_cast<cudaStream_t>(cuda_stream));
}

}  // extern "C"
