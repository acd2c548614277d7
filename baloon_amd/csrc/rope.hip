// rope.hip -- rows of heads normed and turned by position (ix_rope_rows; the formulas are rope.h's).
//
// Every value is read and written once, so HBM bounds it: a wave takes one token's 4 rows of 512 channels, 8 of 256, 16 of 128,
// its loads under way while it works out the token's cosines and sines, which stand in LDS for all of them. 4,096 tokens of 32 heads
// of 128, all channels turned: 67 MB in 13.6 us, 4.9 TB/s of a copy's 5.45; with a norm, 16 heads of 256 of which 64 channels turn,
// 15,059 tokens: 247 MB in 53 us, 4.7 TB/s. A single token: 3.9 us, the call's launch.
#include "rope.h"

namespace ixg {
namespace {

constexpr int kRopeThreads = 256, kRopeWaves = kRopeThreads / kWave;

__global__ void __launch_bounds__(kRopeThreads) rope_kernel(RopeRows A, Batch a, int first) {
    extern __shared__ float2 rope_tables[];
    const int lane = threadIdx.x & (kWave - 1), w = __builtin_amdgcn_readfirstlane((int)threadIdx.x / kWave);
    const long long t = ((long long)first + blockIdx.x) * kRopeWaves + w;
    if (t < a.T) rope_item(A, a, (int)t, blockIdx.y, lane, rope_tables + w * A.r.half);
}

}  // namespace

hipError_t launch_rope(const RopeRows& A, const Batch& a, hipStream_t s) {
    return launch_in_pieces((a.T + (long long)kRopeWaves - 1) / kRopeWaves, kRopeThreads, [&](long long first, unsigned n) {
        hipLaunchKernelGGL(rope_kernel, dim3(n, (unsigned)A.groups), dim3(kRopeThreads), kRopeWaves * A.r.half * sizeof(float2), s, A, a,
                           (int)first);
    });
}

}  // namespace ixg

extern "C" {

hipError_t ix_rope_rows(const ix_rope* rope, int n_seq, int total_T, const int32_t* cu_seqlens, const int32_t* kv_len, const ix_rows* x,
                        int heads, int d, uint16_t* y, hipStream_t s) {
    using namespace ixg;
    RopeRows A;
    Batch a;
    if (!make_batch(n_seq, total_T, cu_seqlens, kv_len, cu_seqlens, 1, &a)) return hipErrorInvalidValue;     // it has no table
    if (!make_rope(rope, d, &A.r) || heads <= 0 || heads > 65536) return hipErrorInvalidValue;
    if (total_T == 0) return hipSuccess;                      // of tensors without elements, whose addresses may be 0
    if (!make_rope_rows(rope, x, heads, d, y, &A)) return hipErrorInvalidValue;
    return launch_rope(A, a, s);
}

}  // extern "C"
