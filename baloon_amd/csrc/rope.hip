// rope.hip -- rows of heads normed and turned by position (ix_rope_rows; the formulas are rope.h's).
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
