// add_norm.hip -- RMS norm with the residual's addition, ahead of a layer's projections:
//
//   h = bf16(x + res);   y = h / sqrt(mean(h^2) + eps) * (w0 + w)
//
// per row, y as fp32, bf16 and/or q8_1 blocks. About 8 operations an element against 6 to 12 bytes:
// bound by memory at prompt sizes, by the launch at decode sizes. So each element is read once and held
// in registers between the sum and the product. 8,192 rows of 2,048 bf16 with a residual, 128 MB: 25.4 us, 5.3 TB/s,
// what a copy of that size reaches; one row of 2,048: 1.6 to 1.9 us. No counterpart in the reference.
#include <type_traits>

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
    // rint, halves away from 0, of v / d by its correctly rounded reciprocal and two corrections, which leave the quotient
    // correctly rounded (Markstein; the second is needed where the first product is more than an ulp off), and 1/2 less half
    // an ulp of it: a division and roundf for each value are 3 times the instructions, and the kernel takes 4.0 us for 8
    // rows of 4,096 with them.
    const auto bounded = [](float x, float most) { return fminf(fmaxf(x, -most), most); };
    const float inv = 1.0f / d;
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        x[e] = bounded(v[e] * inv, 200.0f);
        x[e] = bounded(fmaf(fmaf(-x[e], d, v[e]), inv, x[e]), 200.0f);
        x[e] = bounded(fmaf(fmaf(-x[e], d, v[e]), inv, x[e]), 127.0f);
    }
    if (d < 1e-30f) {                                         // 1 / d or the remainders could leave the floats' range
        asm volatile("");
#pragma unroll 1
        for (int e = 0; e < 8; ++e) {
            float y = 0.0f;
#pragma unroll
            for (int f = 0; f < 8; ++f) y = f == e ? v[f] : y;
            y = d == 0.0f ? 0.0f : bounded(y / d, 127.0f);
#pragma unroll
            for (int f = 0; f < 8; ++f) x[f] = f == e ? y : x[f];
        }
    }
    uint32_t q[2] = {0, 0};
#pragma unroll
    for (int e = 0; e < 8; ++e)
        q[e / 4] |= (uint32_t)(uint8_t)(int8_t)(int)(x[e] + copysignf(0x1.fffffep-2f, x[e])) << (8 * (e & 3));
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

// 8 values at any address that their type allows (the target reads and writes words unaligned), or the first `left`.
template <class V, class E>
__device__ __forceinline__ V load8(const E* p, int left) {
    V x = {};
    if (left >= 8) {
        __builtin_memcpy(&x, p, sizeof(x));
    } else {
        E v[8] = {};
#pragma unroll
        for (int e = 0; e < 7; ++e)
            if (e < left) v[e] = p[e];
        __builtin_memcpy(&x, v, sizeof(x));
    }
    return x;
}
template <class V, class E>
__device__ __forceinline__ void store8(E* p, const V& x, int left) {
    if (left >= 8) {
        __builtin_memcpy(p, &x, sizeof(x));
    } else {
        E v[8];
        __builtin_memcpy(v, &x, sizeof(x));
#pragma unroll
        for (int e = 0; e < 7; ++e)
            if (e < left) p[e] = v[e];
    }
}
struct F8 {
    float v[8];
};

// T threads a row, N chunks of 8 a thread. kTail: the last chunk may be a part of one. Rows that do not begin at 16 bytes
// take longer (128 MB in rows of 1,001: 38 us), by single values they took twice that.
template <int T, int N, bool F32, bool kTail>
__global__ void __launch_bounds__(T) norm_kernel(NormIo io) {
    __shared__ float red[T / kWave];
    const int t = threadIdx.x, lane = t & (kWave - 1);
    const size_t base = (size_t)blockIdx.x * io.n;
    const int chunks = kTail ? (io.n + 7) / 8 : io.n / 8;
    const auto left = [&](int c) { return kTail ? io.n - 8 * c : 8; };
    float h[N][8];
    typename std::conditional<F32, F8, uint4>::type x[N] = {};
    uint4 r[N] = {};
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int c = t + i * T;
        if (c >= chunks) continue;
        if constexpr (F32) x[i] = load8<F8>(io.x + base + 8 * c, left(c));
        else x[i] = load8<uint4>(io.x16 + base + 8 * c, left(c));
        if (io.res) r[i] = load8<uint4>(io.res + base + 8 * c, left(c));
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
                a = x[i].v[2 * e];
                b = x[i].v[2 * e + 1];
            } else {
                const uint32_t p = e == 0 ? x[i].x : e == 1 ? x[i].y : e == 2 ? x[i].z : x[i].w;
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
        if (io.res_out && in) store8(io.res_out + base + 8 * c, make_uint4(out[0], out[1], out[2], out[3]), left(c));
    }
    const float inv = 1.0f / sqrtf(group_sum<T>(sq, red) / (float)io.n + io.eps);
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int c = t + i * T;
        const bool in = c < chunks;
        float y[8];
        if (in) {
            const F8 w = load8<F8>(io.w + 8 * c, left(c));
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] = h[i][e] * inv * (io.w0 + w.v[e]);
            if (io.y) store8(io.y + base + 8 * c, F8{{y[0], y[1], y[2], y[3], y[4], y[5], y[6], y[7]}}, left(c));
            if (io.y16)
                store8(io.y16 + base + 8 * c, make_uint4(pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3]),
                                                         pack_bf16x2(y[4], y[5]), pack_bf16x2(y[6], y[7])), left(c));
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] = 0.0f;
        }
        if (io.q81) q81_store8(y, lane, in ? io.q81 + (base + 8 * c) / 32 * kQ81Bytes : nullptr);
    }
}

template <int T, int N>
hipError_t launch_norm(const NormIo& io, hipStream_t s) {
    return launch_in_pieces(io.rows, T, [&](long long first, unsigned rows) {
        const size_t at = (size_t)first * io.n;
        NormIo p = io;
        if (first > 0) {
            if (p.x) p.x += at;
            if (p.x16) p.x16 += at;
            if (p.res) p.res += at;
            if (p.res_out) p.res_out += at;
            if (p.y) p.y += at;
            if (p.y16) p.y16 += at;
            if (p.q81) p.q81 += at / 32 * kQ81Bytes;
        }
        const auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(rows), dim3(T), 0, s, p); };
        if (io.n % 8) io.x ? launch(&norm_kernel<T, N, true, true>) : launch(&norm_kernel<T, N, false, true>);
        else io.x ? launch(&norm_kernel<T, N, true, false>) : launch(&norm_kernel<T, N, false, false>);
    });
}

bool aligned(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

}  // namespace
}  // namespace ixg

extern "C" hipError_t ix_add_rms_norm(int rows, int n, const float* x, const uint16_t* x_bf16, const uint16_t* res,
                                      uint16_t* res_out, const float* weight, float weight_offset, float eps, float* y,
                                      uint16_t* y_bf16, void* y_q8_1, hipStream_t s) {
    using namespace ixg;
    if (rows < 0 || n <= 0 || n > kNormMax || (y_q8_1 && n % 32)) return hipErrorInvalidValue;
    if (rows == 0) return hipSuccess;                         // of tensors without elements, whose addresses may be 0
    if (!x == !x_bf16 || !weight || (!y && !y_bf16 && !y_q8_1)) return hipErrorInvalidValue;
    if (!aligned(x, 4) || !aligned(x_bf16, 2) || !aligned(res, 2) || !aligned(res_out, 2) || !aligned(weight, 4) ||
        !aligned(y, 4) || !aligned(y_bf16, 2) || !aligned(y_q8_1, 4))
        return hipErrorInvalidValue;
    const NormIo io{x, x_bf16, res, res_out, weight, weight_offset, eps, y, y_bf16, static_cast<uint8_t*>(y_q8_1), rows, n};
    // A chunk a thread, as few threads as hold the row: one row takes 1.9 to 2.6 us up to 8,192 values (2.6 to 3.8 with 4
    // chunks a thread), and 128 MB 25 to 27 (27 to 29).
    const int chunks = (n + 7) / 8;
    if (chunks <= 64) return launch_norm<64, 1>(io, s);
    if (chunks <= 256) return launch_norm<256, 1>(io, s);
    if (chunks <= 512) return launch_norm<512, 1>(io, s);
    if (chunks <= 1024) return launch_norm<1024, 1>(io, s);
    if (chunks <= 2048) return launch_norm<1024, 2>(io, s);
    return launch_norm<1024, 4>(io, s);
}
