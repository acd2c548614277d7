// rope.h -- a head's row normed and turned by its token's position (ix_rope, include/ix_gdn.h): its checks on the host and
// what the kernels share.
//
//   f = x / sqrt(mean(x^2) + eps) * (norm_offset + norm)   (f = x without a norm)
//   y_a = f_a cos - f_b sin,  y_b = f_b cos + f_a sin        for each pair (a, b) of the first `rot` channels
//
// A lane holds 8 consecutive channels of a row, 2^per_log lanes the row: y = (x A + partner B) / root, with A = w cos and B = -+ w' sin
// worked out once for all heads of a token. In the halves' layout the 8 partners are read from memory again (the row's other lanes have just read the same lines); so a row's reads must all be done before a lane
// writes where it lies, which the wave's order gives: one wave reads and writes a row.
#pragma once
#include "kv8.h"

namespace ixg {

struct Rope {
    const float *freq, *norm;
    float amplitude, norm_offset, eps, per_channel;       // 1 / d
    int rot, half, pairs, d, per_log;
    int whole;                    // every lane's channels are turned alike: all, none, all first or all second ones of pairs
};

inline bool make_rope(const ix_rope* r, int d, Rope* out) {
    if (!r || r->rot < 0 || r->rot > d || r->rot % 2 || (r->layout != IX_ROPE_HALVES && r->layout != IX_ROPE_PAIRS)) return false;
    if (d <= 0 || d > 512 || d % 8 || (r->rot && !r->freq) || !ptr_aligned(r->freq, 4) || !ptr_aligned(r->norm, 4)) return false;
    int per_log = 3;
    while (8 << per_log < d) ++per_log;
    const int half = r->rot / 2, pairs = r->layout == IX_ROPE_PAIRS;
    *out = Rope{r->freq, r->norm, r->amplitude, r->norm_offset, r->eps, 1.0f / (float)d, r->rot, half, pairs, d, per_log, (pairs ? r->rot : half) % 8 == 0};
    return true;
}

// cos and sin of pos * freq, times the amplitude. The angle is taken in turns in 64 bits, and a far position's whole turns are gone
// before it is rounded to 32: that is 2^-26 of a turn, 2^-23.3, and the two products and their constant (2^-53, 2^-53 and 2^-53.8)
// are 2^-51.6 of the angle.
__device__ __forceinline__ float2 cos_sin(const Rope& r, int pos, float freq) {
    double turns = (double)pos * (double)freq * 0.15915494309189535;
    turns -= rint(turns);
    float s, c;
    sincospif(2.0f * (float)turns, &s, &c);
    return make_float2(c * r.amplitude, s * r.amplitude);
}

__device__ __forceinline__ void widen8(const uint4& x, float (&f)[8]) {
    const uint32_t u[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = __uint_as_float(e & 1 ? u[e / 2] & 0xffff0000u : u[e / 2] << 16);
}

// What does not change from row to row: of channels c .. c + 7.
struct RopeLane {
    int c;
    float w[8], wp[8];            // the norm's factors, and those of the partners

    // c as a number of its own: conditions on each of a lane's channels are worked out where they are used (8 and more of
    // them kept for the whole kernel would spill the scalar registers).
    __device__ __forceinline__ int here() const {
        int x = c;
        asm volatile("" : "+v"(x));
        return x;
    }
    // The partner of channel ch < rot in the halves' layout.
    static __device__ __forceinline__ int partner(const Rope& r, int ch) { return ch < r.half ? ch + r.half : ch - r.half; }

    __device__ __forceinline__ void begin(const Rope& r, int lane) {
        c = (lane & ((1 << r.per_log) - 1)) * 8;
        if (!r.norm) return;
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e] = wp[e] = 0.0f;
        if (c < r.d) __builtin_memcpy(w, r.norm + c, sizeof(w));
        if (!r.pairs && r.whole) {
            if (c < r.rot) __builtin_memcpy(wp, r.norm + partner(r, c), sizeof(wp));
        } else if (!r.pairs) {
            const int x = here();
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (x + e < r.rot) wp[e] = r.norm[partner(r, x + e)];
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e] += r.norm_offset, wp[e] += r.norm_offset;
    }
    // The partners of this lane's channels `own`, zeros of those behind rot: as 8 values where they lie side by side.
    template <class Load8>
    __device__ __forceinline__ uint4 load_other(const Rope& r, const uint16_t* row, const uint4& own, Load8 load8) const {
        const uint4 none = make_uint4(0, 0, 0, 0);
        if (r.pairs) {
            uint32_t u[4] = {own.x, own.y, own.z, own.w};
            const int last = r.rot - here();
#pragma unroll
            for (int e = 0; e < 4; ++e) u[e] = 2 * e < last ? __builtin_amdgcn_alignbit(u[e], u[e], 16) : 0;
            return make_uint4(u[0], u[1], u[2], u[3]);
        }
        if (r.whole) return c < r.rot ? load8(row + partner(r, c)) : none;
        const int x = here();
        uint32_t u[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) u[e] = x + e < r.rot ? row[partner(r, x + e)] : 0;
        return make_uint4(u[0] | u[1] << 16, u[2] | u[3] << 16, u[4] | u[5] << 16, u[6] | u[7] << 16);
    }
    // A and B of this lane's channels, from a table of cos and sin for each pair. A channel that passes takes 1 and -0: its partner
    // is 0, and x + 0 * -0 is x, -0 too.
    __device__ __forceinline__ void factors(const Rope& r, const float2* table, float (&A)[8], float (&B)[8]) const {
#pragma unroll
        for (int e = 0; e < 8; ++e) A[e] = 1.0f, B[e] = -0.0f;
        if (!r.whole) {
            const int x = here();
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int ch = x + e;
                if (ch >= r.rot) continue;
                const bool second = r.pairs ? e & 1 : ch >= r.half;
                const float2 t = table[r.pairs ? ch >> 1 : second ? ch - r.half : ch];
                A[e] = t.x;
                B[e] = second ? t.y : -t.y;
            }
        } else if (c < r.rot && r.pairs) {
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
                const float2 t = table[(c + e) / 2];
                A[e] = A[e + 1] = t.x;
                B[e] = -t.y;
                B[e + 1] = t.y;
            }
        } else if (c < r.rot) {
            const float2* at = table + (c < r.half ? c : c - r.half);
            const float sign = c < r.half ? -1.0f : 1.0f;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                A[e] = at[e].x;
                B[e] = at[e].y * sign;
            }
        }
        if (!r.norm) return;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            A[e] *= w[e];
            B[e] *= r.pairs ? w[e ^ 1] : wp[e];
        }
    }
    // A row's 8 values, rounded to bf16. Every lane of the row takes part, those behind d with zeros.
    __device__ __forceinline__ uint4 turned(const Rope& r, const uint4& own, const uint4& other, const float (&A)[8], const float (&B)[8]) const {
        float y[8], p[8];
        widen8(own, y);
        widen8(other, p);
        float inv = 1.0f;
        if (r.norm) {
            float sum = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; ++e) sum = fmaf(y[e], y[e], sum);
            sum += dpp_f32<kDppQuadXor1>(sum);
            sum += dpp_f32<kDppQuadXor2>(sum);
            sum += dpp_f32<kDppRowHalfMirror>(sum);
            if (r.per_log > 3) sum += dpp_f32<kDppRowMirror>(sum);
            if (r.per_log > 4) sum = pair_sum16(sum);
            if (r.per_log > 5) sum = pair_sum32(sum);
            inv = __builtin_amdgcn_rsqf(fmaf(sum, r.per_channel, r.eps));                  // within an ulp of 32 bits, for a bf16 result
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = fmaf(p[e], B[e], y[e] * A[e]) * inv;
        return make_uint4(pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3]), pack_bf16x2(y[4], y[5]), pack_bf16x2(y[6], y[7]));
    }
};

// Token rows of heads that are turned into packed ones: a wave's item is one token's kRopeSteps 2^(6 - per_log) heads.
// With 2, 4 and 8 steps the kernel takes, over four inputs in turn (us): 4,096 tokens of 32 heads of 128 16.1, 16.8 and 14.0,
// 15,800 of 16 of 256 60.5, 53.5 and 53.2, 2,541 of these far on 11.1, 10.8 and 11.6, a single one 3.2, 3.8
// and 4.9, 256 of 32 of 128 3.6, 4.2 and 5.5. The append's grid holds 3 waves a SIMD with 8, 5 with 4 (it spills scalar registers with 8).
constexpr int kRopeSteps = 4;
struct RopeRows {
    Rope r;
    const uint16_t* x;
    long long stride;
    uint16_t* y;                  // [T][heads][d]
    int heads, groups;            // items of a token
};
inline bool make_rope_rows(const ix_rope* rope, const ix_rows* x, int heads, int d, uint16_t* y, RopeRows* out) {
    if (!make_rope(rope, d, &out->r) || heads <= 0 || heads > 65536) return false;
    if (!rows_ok(x, (long long)heads * d) || !y || !ptr_aligned(y, 2)) return false;
    const int per_item = kRopeSteps << (6 - out->r.per_log);
    out->x = x->p;
    out->stride = x->stride;
    out->y = y;
    out->heads = heads;
    out->groups = (heads + per_item - 1) / per_item;
    return true;
}

// rope.hip: the items of a batch as a launch of their own.
hipError_t launch_rope(const RopeRows& A, const Batch& a, hipStream_t s);

// `table`: this wave's own, of r.half pairs.
__device__ __forceinline__ void rope_item(const RopeRows& A, const Batch& a, int t, int group, int lane, float2* table) {
    const Rope& r = A.r;
    const int b = wave_search(a.n_seq, t, lane, [&](int i) { return a.start(i); });
    const int s0 = a.start(b), end = a.start(b + 1);
    if (t < s0 || t >= end) return;                           // before the first sequence's rows, or behind the last's
    RopeLane L;
    L.begin(r, lane);
    const int heads0 = group * (kRopeSteps << (6 - r.per_log)) + (lane >> r.per_log);
    uint4 own[kRopeSteps], other[kRopeSteps];
#pragma unroll
    for (int i = 0; i < kRopeSteps; ++i) {
        const int h = heads0 + (i << (6 - r.per_log));
        const uint16_t* row = A.x + (long long)t * A.stride + (size_t)h * r.d;
        const bool any = h < A.heads && L.c < r.d;
        own[i] = any ? load_row8(row + L.c) : make_uint4(0, 0, 0, 0);
        other[i] = any ? L.load_other(r, row, own[i], load_row8) : make_uint4(0, 0, 0, 0);
    }
    const int pos = a.kv_len[b] - (end - t);
#pragma unroll 1
    for (int i = lane; i < r.half; i += kWave) table[i] = cos_sin(r, pos, r.freq[i]);
    wave_lds_sync();
    float F[8], S[8];
    L.factors(r, table, F, S);
#pragma unroll
    for (int i = 0; i < kRopeSteps; ++i) {
        const int h = heads0 + (i << (6 - r.per_log));
        const uint4 y = L.turned(r, own[i], other[i], F, S);
        __builtin_amdgcn_sched_barrier(0);                    // one row's registers at a time
        if (h < A.heads && L.c < r.d) __builtin_memcpy(A.y + ((size_t)t * A.heads + h) * r.d + L.c, &y, sizeof(y));
    }
    wave_lds_sync();                                          // the table is free again
}

}  // namespace ixg
