// add_norm.hip -- RMS norm with the residual's addition, ahead of a layer's projections:
//
//   h = bf16(x + res);   y = h / sqrt(mean(h^2) + eps) * (w0 + w)
//
// per row, y as fp32, bf16 and/or q8_1 blocks. About 8 operations an element against 6 to 12 bytes:
// bound by memory at prompt sizes, by the launch at decode sizes. So each element is read once and held
// in registers between the sum and the product. No counterpart in the reference.
#include "gdn_common.h"

namespace ixg {
namespace {

constexpr int kNormMax = 32768;        // longest row: 1024 threads of 32 values

struct NormIo {
    const float* x;
    const uint16_t* x16;
    const uint16_t* res;
    uint16_t* res_out;
    const float* w;
    float w0, eps;
    float* y;
    uint16_t* y16;
    uint8_t* q81;
    int rows, n;
};

// q81_store for a lane that holds 8 consecutive values, entries 8 (lane & 3) .. + 7 of the block of its 4
// lanes: the same bytes (the butterfly's steps 16 and 8 cross lanes, 4, 2 and 1 stay inside).
// All 64 lanes call it; blk == nullptr stores nothing.
__device__ __forceinline__ void q81_store8(const float (&v)[8], int lane, uint8_t* blk) {
    float m = 0.0f, s[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) m = fmaxf(m, fabsf(v[e]));
    m = fmaxf(m, dpp_f32<kDppQuadXor2>(m));
    m = fmaxf(m, dpp_f32<kDppQuadXor1>(m));
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float t = v[e] + dpp_f32<kDppQuadXor2>(v[e]);
        s[e] = t + dpp_f32<kDppQuadXor1>(t);
    }
    const float sum = ((s[0] + s[4]) + (s[2] + s[6])) + ((s[1] + s[5]) + (s[3] + s[7]));
    const float d = fminf(m / 127.0f, kHalfMax);
    uint32_t q[2] = {0, 0};
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const int c = d == 0.0f ? 0 : (int)fminf(fmaxf(roundf(v[e] / d), -127.0f), 127.0f);
        q[e / 4] |= (uint32_t)(uint8_t)(int8_t)c << (8 * (e & 3));
    }
    if (!blk) return;
    uint32_t* to = reinterpret_cast<uint32_t*>(blk + 4 + 8 * (lane & 3));    // blocks are 36 bytes: 4-byte stores
    to[0] = q[0];
    to[1] = q[1];
    if ((lane & 3) == 0) {
        const float sc = fminf(fmaxf(sum, -kHalfMax), kHalfMax);
        const uint32_t hd = __builtin_bit_cast(uint16_t, (_Float16)d), hs = __builtin_bit_cast(uint16_t, (_Float16)sc);
        *reinterpret_cast<uint32_t*>(blk) = hd | (hs << 16);
    }
}

// Sum over the T threads of a row's group, in every one of them.
template <int T>
__device__ __forceinline__ float group_sum(float v, float* red) {
    v = wave_sum(v);
    if constexpr (T > kWave) {
        if ((threadIdx.x & (kWave - 1)) == 0) red[threadIdx.x / kWave] = v;
        lds_barrier();
        v = 0.0f;
#pragma unroll
        for (int i = 0; i < T / kWave; ++i) v += red[i];
    }
    return v;
}

// Rows of whole chunks of 8, every operand 16-byte aligned: T threads a row, N chunks a thread, in
// workgroups of R rows.
template <int T, int N, int R, bool F32>
__global__ void __launch_bounds__(T * R) norm_kernel(NormIo io) {
    __shared__ float red[T / kWave];
    const int t = threadIdx.x % T, lane = threadIdx.x & (kWave - 1);
    const int row = blockIdx.x * R + threadIdx.x / T;
    if (R > 1 && row >= io.rows) return;                     // whole waves
    const size_t base = (size_t)row * io.n;
    const int chunks = io.n / 8;
    float h[N][8];
    uint4 x[N][F32 ? 2 : 1] = {}, r[N] = {};
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int c = t + i * T;
        if (c >= chunks) continue;
        if constexpr (F32) {
            const uint4* p = reinterpret_cast<const uint4*>(io.x + base + 8 * c);
            x[i][0] = p[0];
            x[i][1] = p[1];
        } else {
            x[i][0] = *reinterpret_cast<const uint4*>(io.x16 + base + 8 * c);
        }
        if (io.res) r[i] = *reinterpret_cast<const uint4*>(io.res + base + 8 * c);
    }
    float sq = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int c = t + i * T;
        const bool in = c < chunks;
        uint32_t out[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            float a, b;
            if constexpr (F32) {
                const uint4& p = x[i][e / 2];
                a = __uint_as_float(e & 1 ? p.z : p.x);
                b = __uint_as_float(e & 1 ? p.w : p.y);
            } else {
                const uint32_t p = e == 0 ? x[i][0].x : e == 1 ? x[i][0].y : e == 2 ? x[i][0].z : x[i][0].w;
                a = __uint_as_float(p << 16);
                b = __uint_as_float(p & 0xffff0000u);
            }
            if (io.res) {
                const uint32_t p = e == 0 ? r[i].x : e == 1 ? r[i].y : e == 2 ? r[i].z : r[i].w;
                a += __uint_as_float(p << 16);
                b += __uint_as_float(p & 0xffff0000u);
            }
            out[e] = pack_bf16x2(a, b);                      // the stream is bf16; the norm is of what it holds
            h[i][2 * e] = in ? __uint_as_float(out[e] << 16) : 0.0f;
            h[i][2 * e + 1] = in ? __uint_as_float(out[e] & 0xffff0000u) : 0.0f;
            sq = fmaf(h[i][2 * e], h[i][2 * e], sq);
            sq = fmaf(h[i][2 * e + 1], h[i][2 * e + 1], sq);
        }
        if (io.res_out && in) *reinterpret_cast<uint4*>(io.res_out + base + 8 * c) = make_uint4(out[0], out[1], out[2], out[3]);
    }
    const float inv = 1.0f / sqrtf(group_sum<T>(sq, red) / (float)io.n + io.eps);
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int c = t + i * T;
        const bool in = c < chunks;
        float y[8];
        if (in) {
            const v4f* w = reinterpret_cast<const v4f*>(io.w + 8 * c);
            const v4f w0 = w[0], w1 = w[1];
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] = h[i][e] * inv * (io.w0 + (e < 4 ? w0[e & 3] : w1[e & 3]));
            if (io.y) {
                v4f* p = reinterpret_cast<v4f*>(io.y + base + 8 * c);
                p[0] = v4f{y[0], y[1], y[2], y[3]};
                p[1] = v4f{y[4], y[5], y[6], y[7]};
            }
            if (io.y16)
                *reinterpret_cast<uint4*>(io.y16 + base + 8 * c) = make_uint4(
                    pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3]), pack_bf16x2(y[4], y[5]), pack_bf16x2(y[6], y[7]));
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] = 0.0f;
        }
        if (io.q81) q81_store8(y, lane, in ? io.q81 + (base + 8 * c) / 32 * kQ81Bytes : nullptr);
    }
}

// Rows of any length and alignment, N values a thread (q8_1 rows are whole blocks of 32: half a wave each).
template <int T, int N>
__global__ void __launch_bounds__(T) norm_any_kernel(NormIo io) {
    __shared__ float red[T / kWave];
    const int t = threadIdx.x, lane = t & (kWave - 1);
    const size_t base = (size_t)blockIdx.x * io.n;
    float h[N], sq = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int c = t + i * T;
        h[i] = 0.0f;
        if (c < io.n) {
            float v = io.x ? io.x[base + c] : bf16_to_f32(io.x16[base + c]);
            if (io.res) v += bf16_to_f32(io.res[base + c]);
            const uint16_t b = f32_to_bf16(v);
            if (io.res_out) io.res_out[base + c] = b;
            h[i] = bf16_to_f32(b);
        }
        sq = fmaf(h[i], h[i], sq);
    }
    const float inv = 1.0f / sqrtf(group_sum<T>(sq, red) / (float)io.n + io.eps);
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int c = t + i * T;
        const bool in = c < io.n;
        const float y = in ? h[i] * inv * (io.w0 + io.w[c]) : 0.0f;
        if (in && io.y) io.y[base + c] = y;
        if (in && io.y16) io.y16[base + c] = f32_to_bf16(y);
        if (io.q81) q81_store(y, lane, in ? io.q81 + (base + c) / 32 * kQ81Bytes : nullptr);
    }
}

template <int T, int N, int R>
void launch_norm(const NormIo& io, hipStream_t s) {
    const dim3 grid((unsigned)((io.rows + R - 1) / R));
    if (io.x) hipLaunchKernelGGL((norm_kernel<T, N, R, true>), grid, dim3(T * R), 0, s, io);
    else hipLaunchKernelGGL((norm_kernel<T, N, R, false>), grid, dim3(T * R), 0, s, io);
}

bool aligned(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

}  // namespace
}  // namespace ixg

extern "C" hipError_t ix_add_rms_norm(int rows, int n, const float* x, const uint16_t* x_bf16, const uint16_t* res,
                                      uint16_t* res_out, const float* weight, float weight_offset, float eps, float* y,
                                      uint16_t* y_bf16, void* y_q8_1, hipStream_t s) {
    using namespace ixg;
    if (rows < 0 || n <= 0 || n > kNormMax || !x == !x_bf16 || !weight || (!y && !y_bf16 && !y_q8_1))
        return hipErrorInvalidValue;
    if (y_q8_1 && n % 32) return hipErrorInvalidValue;
    if (!aligned(x, 4) || !aligned(x_bf16, 2) || !aligned(res, 2) || !aligned(res_out, 2) || !aligned(weight, 4) ||
        !aligned(y, 4) || !aligned(y_bf16, 2) || !aligned(y_q8_1, 4))
        return hipErrorInvalidValue;
    if (rows == 0) return hipSuccess;
    const NormIo io{x, x_bf16, res, res_out, weight, weight_offset, eps, y, y_bf16, static_cast<uint8_t*>(y_q8_1), rows, n};
    const bool wide = n % 8 == 0 && aligned(x, 16) && aligned(x_bf16, 16) && aligned(res, 16) && aligned(res_out, 16) &&
                      aligned(weight, 16) && aligned(y, 16) && aligned(y_bf16, 16);
    if (!wide) {
        const dim3 grid((unsigned)rows);
        if (n <= 2048) hipLaunchKernelGGL((norm_any_kernel<256, 8>), grid, dim3(256), 0, s, io);
        else if (n <= 8192) hipLaunchKernelGGL((norm_any_kernel<1024, 8>), grid, dim3(1024), 0, s, io);
        else hipLaunchKernelGGL((norm_any_kernel<1024, 32>), grid, dim3(1024), 0, s, io);
        return hipGetLastError();
    }
    const int chunks = n / 8;
    if (chunks <= 64) launch_norm<64, 1, 4>(io, s);
    else if (chunks <= 256) launch_norm<256, 1, 1>(io, s);
    else if (chunks <= 512) launch_norm<512, 1, 1>(io, s);
    else if (chunks <= 1024) launch_norm<1024, 1, 1>(io, s);
    else launch_norm<1024, 4, 1>(io, s);
    return hipGetLastError();
}
