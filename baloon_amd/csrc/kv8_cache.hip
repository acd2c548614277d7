// kv8_cache.hip -- keys and values into the paged 8-bit cache, and back out of it.
//
// A page holds `page` tokens of every kv head; each (page, head) has one scale s for its keys and one for
// its values, and a value stands as s * code. New tokens can be larger than what a page's scale covers:
//
//   s' = max(s if the page holds older tokens, max|x| / 127);  older codes <- rint(code * (s / s')) where
//   s' > s;  new codes = rint(x / s')
//
// so that a page is at any time within half a quantum of its largest value's scale (one more half for each
// time the scale grew). Divisions are IEEE's and rint is to nearest even: the codes are defined bit for bit.
//
// Keys lie token by token ([page][d], the rows of K Q^T), values channel by channel ([d][page], the rows of
// V^T P^T), so that the attention's lanes read either operand of its matrix products as 16 consecutive bytes.
//
// One workgroup per (page with new tokens, head, K or V): it alone reads and writes that scale and those
// codes, reads the rows once into LDS, and turns the values there. 16 sequences of 1 to 2,048 new tokens, 2 heads of
// 256, 15,059 tokens in all: 46 MB in 15 us, 3.1 TB/s of a copy's 5.3. A workgroup's pass is a chain (its place, the
// rows, their largest value, the codes), 3 workgroups a CU of it side by side; a read of the same tokens takes 10 to 11 us.
// One token for each of 64 sequences: 5.2 and 4.2 us, launches and that chain.
#include <type_traits>

#include "kv8.h"

namespace ixg {
namespace {

// The page that slot j of the grid stands for. Sequence b owns the slots from cu[b] / page + 2 b on: at most
// q / page + 2 pages hold its q new tokens, so no prefix sum over the sequences is needed.
struct PageJob {
    int b, id, held, end, row;      // slots held .. end - 1 of page id take the rows from `row` on
};
__device__ __forceinline__ bool page_job(const Batch& a, const Kv8& c, int j, int lane, PageJob* out) {
    const int b = wave_search(a.n_seq, j, lane, [&](int i) { return (a.start(i) >> c.page_log) + 2 * i; });
    const int s0 = a.start(b), q = a.start(b + 1) - s0, kv = a.kv_len[b];
    const int first = kv - q, from = max(first, 0);         // tokens before position 0 are not held
    const int slot = j - ((s0 >> c.page_log) + 2 * b);      // negative before the first sequence's rows
    const int p = (from >> c.page_log) + slot;
    if (q <= 0 || kv <= 0 || slot < 0 || p > (kv - 1) >> c.page_log) return false;
    const int at = p << c.page_log;
    const int lo = max(from, at);
    out->b = b;
    out->id = a.page_at(b, p, c.n_pages);
    out->held = lo - at;
    out->end = min(kv - at, c.page);
    out->row = s0 + lo - first;
    return out->id >= 0;
}

__device__ __forceinline__ float max_abs(const uint4& x) {
    float m = 0.0f;
    const uint32_t u[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int e = 0; e < 4; ++e)
        m = fmaxf(m, fmaxf(fabsf(__uint_as_float(u[e] << 16)), fabsf(__uint_as_float(u[e] & 0xffff0000u))));
    return m;
}

// Eight codes rint(x / s) by the correctly rounded reciprocal y of s and one correction, q + (x - q s) y with q = x y (a
// division is 10 instructions). Before its last rounding that is within 2^-21 ulp of x / s, so it can only be rounded
// otherwise, and the code with it, where x / s lies that near half an ulp from a tie n + 1/2. x has 8 significant bits:
// x = (n + 1/2)(1 +- 2^-k) s + that little has no solution but s = 2^e (1 - 2^-24), x = s rounded up / 2, which comes
// out right. 1.5 2^23 added to a number leaves its nearest integer, to even, in the sum's low bits.
constexpr float kMagic = 12582912.0f, kLeast = 1e-30f;
__device__ __forceinline__ float code_bits(float x, float s, float y) {
    const float q = x * y;
    return fmaf(fmaf(-q, s, x), y, q) + kMagic;
}
__device__ __forceinline__ uint2 codes_of(const uint4& x, float s, float y) {
    const uint32_t u[4] = {x.x, x.y, x.z, x.w};
    uint32_t two[4];
#pragma unroll
    for (int e = 0; e < 4; ++e)
        two[e] = __builtin_amdgcn_perm(__float_as_uint(code_bits(__uint_as_float(u[e] & 0xffff0000u), s, y)),
                                       __float_as_uint(code_bits(__uint_as_float(u[e] << 16), s, y)), 0x0c0c0400u);
    return make_uint2(__builtin_amdgcn_perm(two[1], two[0], 0x05040100u), __builtin_amdgcn_perm(two[3], two[2], 0x05040100u));
}
// The same where s is under kLeast.
__device__ __forceinline__ uint2 codes_of_small(const uint4& x, float s) {
    const uint32_t u[4] = {x.x, x.y, x.z, x.w};
    uint32_t q[2] = {0, 0};
    if (s > 0.0f)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float v = __uint_as_float(e & 1 ? u[e / 2] & 0xffff0000u : u[e / 2] << 16);
            q[e / 4] |= (uint32_t)(uint8_t)(int8_t)(int)fminf(fmaxf(rintf(v / s), -127.0f), 127.0f) << (8 * (e & 3));
        }
    return make_uint2(q[0], q[1]);
}

// 4 x 4 bytes: row i of the results is byte i of each operand.
__device__ __forceinline__ void transpose4(uint32_t (&x)[4]) {
    const uint32_t a = __builtin_amdgcn_perm(x[1], x[0], 0x05010400u), b = __builtin_amdgcn_perm(x[3], x[2], 0x05010400u);
    const uint32_t c = __builtin_amdgcn_perm(x[1], x[0], 0x07030602u), d = __builtin_amdgcn_perm(x[3], x[2], 0x07030602u);
    x[0] = __builtin_amdgcn_perm(b, a, 0x05040100u);
    x[1] = __builtin_amdgcn_perm(b, a, 0x07060302u);
    x[2] = __builtin_amdgcn_perm(d, c, 0x05040100u);
    x[3] = __builtin_amdgcn_perm(d, c, 0x07060302u);
}

// Four codes times r, each rounded again.
__device__ __forceinline__ uint32_t recode4(uint32_t c, float r) {
    uint32_t out = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float v = (float)(int8_t)(c >> (8 * e));
        out |= (uint32_t)(uint8_t)(int8_t)(int)rintf(v * r) << (8 * e);
    }
    return out;
}

// The first `keep` of four codes, and four of which the first `keep` are older ones.
__device__ __forceinline__ uint32_t first_mask(int keep) { return keep <= 0 ? 0u : keep >= 4 ? ~0u : (1u << (8 * keep)) - 1; }
__device__ __forceinline__ uint32_t first(uint32_t q, int keep) { return q & first_mask(keep); }
__device__ __forceinline__ uint32_t older(uint32_t was, uint32_t now, float r, int keep) {
    return first(recode4(was, r), keep) | (now & ~first_mask(keep));
}

// 8 values of a row, bf16, at any 2-byte address (the target reads words unaligned).
__device__ __forceinline__ uint4 load8(const uint16_t* p) {
    uint4 x;
    __builtin_memcpy(&x, p, sizeof(x));
    return x;
}

// A page's values pass through LDS slot by slot. A lane takes 4 channels of 16 slots, which it turns 4 x 4 bytes at
// a time; consecutive lanes take the 16s of the same channels, which lie side by side in the page.
struct Turn {
    int ch, s0;                                               // channels ch .. + 3, slots s0 .. + 15
};
__device__ __forceinline__ Turn turn_of(int i, int span_log) {
    return Turn{(i >> span_log) * 4, (i & ((1 << span_log) - 1)) * 16};
}

// Two passes over the page's new rows, in chunks of 8 channels: the largest value, then the codes. LDS holds a slot's
// chunks of 16 bytes in between; a chunk's codes take its first or, in odd 16s of slots, second half (the turn reads
// the 16s together). The second pass is a rolled loop: every launch begins with an empty instruction cache, and with it
// unrolled 8, 4 and 2 times a single token for 64 sequences took 7.9, 6.6 and 5.5 us of the kernel's time.
constexpr int kBatch = 4;
template <int kThreads>
__global__ void __launch_bounds__(kThreads)
append_kernel(Kv8 c, Batch a, const uint16_t* __restrict__ kr, long long k_stride, const uint16_t* __restrict__ vr,
              long long v_stride, int first_slot) {
    extern __shared__ uint4 raw[];
    __shared__ float red[kThreads / kWave];
    const int tid = threadIdx.x, lane = tid & (kWave - 1), h = blockIdx.y;
    const bool is_v = blockIdx.z;
    PageJob job;
    if (!page_job(a, c, first_slot + (int)blockIdx.x, lane, &job)) return;
    const int per_log = c.d == 64 ? 3 : c.d == 128 ? 4 : 5, chunks = (job.end - job.held) << per_log;
    const long long stride = is_v ? v_stride : k_stride;
    const uint16_t* rows = (is_v ? vr : kr) + (long long)job.row * stride + (size_t)h * c.d;
    const size_t ph = (size_t)job.id * c.h_kv + h;
    float* scale = (is_v ? c.v_scale : c.k_scale) + ph;
    int8_t* codes = (is_v ? c.v : c.k) + ph * c.page * c.d;
    const auto load = [&](int i) { return load8(rows + (i >> per_log) * stride + ((i & ((1 << per_log) - 1)) << 3)); };

    const float old = job.held > 0 ? *scale : 0.0f;
    float m = 0.0f;
    uint4* held = raw + (job.held << per_log);
    for (int i0 = tid; i0 < chunks; i0 += kBatch * kThreads) {
        uint4 x[kBatch];
#pragma unroll
        for (int y = 0; y < kBatch; ++y) x[y] = i0 + y * kThreads < chunks ? load(i0 + y * kThreads) : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int y = 0; y < kBatch; ++y) {
            m = fmaxf(m, max_abs(x[y]));
            if (i0 + y * kThreads < chunks) held[i0 + y * kThreads] = x[y];
        }
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor(m, off, kWave));
    if (lane == 0) red[tid / kWave] = m;
    __syncthreads();                                          // every thread has read the old scale, too
#pragma unroll
    for (int i = 0; i < kThreads / kWave; ++i) m = fmaxf(m, red[i]);
    const float s = fmaxf(old, m / 127.0f);
    const bool grown = job.held > 0 && s > old;
    const float ratio = grown ? old / s : 1.0f, inv = 1.0f / s;
    if (tid == 0) *scale = s;

#pragma unroll 1
    for (int i = tid; i < chunks; i += kThreads) {       // a thread's own chunks
        const int slot = job.held + (i >> per_log);
        const uint2 q = s < kLeast ? codes_of_small(held[i], s) : codes_of(held[i], s, inv);
        if (is_v) reinterpret_cast<uint2*>(held + i)[slot >> 4 & 1] = q;
        else *reinterpret_cast<uint2*>(codes + slot * c.d + ((i & ((1 << per_log) - 1)) << 3)) = q;
    }
    if (!is_v) {
        if (grown) {
            uint4* p = reinterpret_cast<uint4*>(codes);
            for (int i = tid; i < job.held * c.d / 16; i += kThreads) {
                const uint4 o = p[i];
                p[i] = make_uint4(recode4(o.x, ratio), recode4(o.y, ratio), recode4(o.z, ratio), recode4(o.w, ratio));
            }
        }
        return;
    }
    __syncthreads();
    // Channel rows of 16 slots: whole ones at once (slots behind the new tokens hold nothing yet, and get
    // zeros), the one with older tokens in it by bytes, or as a whole where the older ones change too.
    const int span_log = c.page_log - 4;
    for (int i = tid; i < (c.d / 4) << span_log; i += kThreads) {
        const Turn u = turn_of(i, span_log);
        if (u.s0 >= job.end || (u.s0 + 16 <= job.held && !grown)) continue;
        const int keep = job.end - u.s0;                      // slots that hold tokens
        const uint8_t* tile = reinterpret_cast<const uint8_t*>(raw) + (u.ch >> 3) * 16 + (u.s0 >> 4 & 1) * 8 + (u.ch & 7);
        uint32_t n[4][4];                                     // [4 slots][channel]
#pragma unroll
        for (int y = 0; y < 4; ++y) {
#pragma unroll
            for (int z = 0; z < 4; ++z) n[y][z] = *reinterpret_cast<const uint32_t*>(tile + (u.s0 + 4 * y + z) * c.d * 2);
            transpose4(n[y]);
        }
#pragma unroll
        for (int z = 0; z < 4; ++z) {
            int8_t* to = codes + ((u.ch + z) << c.page_log) + u.s0;
            if (u.s0 < job.held && !grown) {
                for (int y = job.held - u.s0; y < min(16, job.end - u.s0); ++y)
                    to[y] = (int8_t)tile[(u.s0 + y) * c.d * 2 + z];
                continue;
            }
            uint4 v = make_uint4(first(n[0][z], keep), first(n[1][z], keep - 4), first(n[2][z], keep - 8), first(n[3][z], keep - 12));
            if (u.s0 < job.held) {
                const uint4 o = *reinterpret_cast<const uint4*>(to);
                v = make_uint4(older(o.x, v.x, ratio, job.held - u.s0), older(o.y, v.y, ratio, job.held - u.s0 - 4),
                               older(o.z, v.z, ratio, job.held - u.s0 - 8), older(o.w, v.w, ratio, job.held - u.s0 - 12));
            }
            *reinterpret_cast<uint4*>(to) = v;
        }
    }
}

__device__ __forceinline__ uint4 values8(uint32_t lo, uint32_t hi, float s) {
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = (float)(int8_t)((e < 4 ? lo : hi) >> (8 * (e & 3))) * s;
    return make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
}

template <int kThreads>
__global__ void __launch_bounds__(kThreads)
read_kernel(Kv8 c, Batch a, uint16_t* __restrict__ ko, uint16_t* __restrict__ vo, int first_slot) {
    extern __shared__ uint8_t tile[];
    const int tid = threadIdx.x, lane = tid & (kWave - 1), h = blockIdx.y;
    const bool is_v = blockIdx.z;
    uint16_t* out = is_v ? vo : ko;
    PageJob job;
    if (!out || !page_job(a, c, first_slot + (int)blockIdx.x, lane, &job)) return;
    const size_t ph = (size_t)job.id * c.h_kv + h;
    const float s = (is_v ? c.v_scale : c.k_scale)[ph];
    const int8_t* codes = (is_v ? c.v : c.k) + ph * c.page * c.d;
    const int per_log = c.d == 64 ? 3 : c.d == 128 ? 4 : 5, pitch = c.d + 4, span_log = c.page_log - 4;      // rows of slots 4 bytes longer: 16 slots on, other banks
    if (is_v) {
        for (int i = tid; i < (c.d / 4) << span_log; i += kThreads) {
            const Turn u = turn_of(i, span_log);
            if (u.s0 >= job.end || u.s0 + 16 <= job.held) continue;
            uint32_t n[4][4];                                 // [4 slots][channel]
#pragma unroll
            for (int z = 0; z < 4; ++z) {
                const uint4 o = *reinterpret_cast<const uint4*>(codes + ((u.ch + z) << c.page_log) + u.s0);
                n[0][z] = o.x; n[1][z] = o.y; n[2][z] = o.z; n[3][z] = o.w;
            }
#pragma unroll
            for (int y = 0; y < 4; ++y) {
                transpose4(n[y]);
#pragma unroll
                for (int z = 0; z < 4; ++z) *reinterpret_cast<uint32_t*>(tile + (u.s0 + 4 * y + z) * pitch + u.ch) = n[y][z];
            }
        }
        __syncthreads();
    }
    for (int i = tid + (job.held << per_log); i < job.end << per_log; i += kThreads) {
        const int slot = i >> per_log, col = (i & ((1 << per_log) - 1)) << 3;
        uint2 q;
        if (is_v) {
            const uint32_t* p = reinterpret_cast<const uint32_t*>(tile + slot * pitch + col);
            q = make_uint2(p[0], p[1]);
        } else {
            q = *reinterpret_cast<const uint2*>(codes + slot * c.d + col);
        }
        const uint4 v = values8(q.x, q.y, s);
        uint16_t* to = out + ((size_t)(job.row + slot - job.held) * c.h_kv + h) * c.d + col;
        __builtin_memcpy(to, &v, sizeof(v));                  // at any 2-byte address
    }
}

long long page_slots(const Kv8& c, const Batch& a) { return (a.T >> c.page_log) + 2ll * a.n_seq; }

// A thread for 32 values of a page; in appends for 64 where the sequences have less than a page of new tokens each. A
// workgroup is bound by the chain of its reads: more threads make it shorter where there is work for them, and keep other
// workgroups from the CU where not. With 16, 32, 64 and 128 values a thread an append takes, us: 16 x 1,024 tokens on 8 heads
// of 128, pages of 64, 32, 24, 26, 30; on 2 heads of 256, pages of 16, 16, 14, 15, 15; 64 x 16 tokens on the former 10.7,
// 9.2, 8.1, 9.7; 256 single tokens 16.7, 14.2, 14.2, 14.8, and on 2 heads of 256, pages of 64, 9.9, 8.7, 8.6, 9.7. A read of
// the first takes 17.9, 17.7, 17.9, 17.6, of 64 pages of 16 tokens on 2 heads of 256 3.3, 3.5, 3.6, 3.6, of 1 x 4,096 4.5,
// 4.6, 5.2, 5.2.
template <class F>
hipError_t with_threads(int n, F launch) {
    if (n <= 64) return launch(std::integral_constant<int, 64>{});
    if (n <= 128) return launch(std::integral_constant<int, 128>{});
    if (n <= 256) return launch(std::integral_constant<int, 256>{});
    return launch(std::integral_constant<int, 512>{});
}

template <int kThreads>
hipError_t launch_append(const Kv8& c, const Batch& a, const ix_rows* k, const ix_rows* v, hipStream_t s) {
    static OncePerDevice once;
    const hipError_t ready = allow_lds(once, &append_kernel<kThreads>, 128 * 256 * sizeof(uint16_t), s);
    if (ready != hipSuccess) return ready;
    return launch_in_pieces(page_slots(c, a), kThreads, [&](long long first, unsigned n) {
        hipLaunchKernelGGL((append_kernel<kThreads>), dim3(n, (unsigned)c.h_kv, 2), dim3(kThreads), c.page * c.d * sizeof(uint16_t), s,
                           c, a, k->p, k->stride, v->p, v->stride, (int)first);
    });
}

template <int kThreads>
hipError_t launch_read(const Kv8& c, const Batch& a, uint16_t* k, uint16_t* v, hipStream_t s) {
    return launch_in_pieces(page_slots(c, a), kThreads, [&](long long first, unsigned n) {
        hipLaunchKernelGGL((read_kernel<kThreads>), dim3(n, (unsigned)c.h_kv, 2), dim3(kThreads), c.page * (c.d + 4), s, c, a, k, v,
                           (int)first);
    });
}

}  // namespace
}  // namespace ixg

extern "C" {

hipError_t ix_kv8_append(const ix_kv8* cache, int n_seq, int total_T, const int32_t* cu_seqlens, const int32_t* kv_len,
                         const int32_t* table, int width, const ix_rows* k, const ix_rows* v, hipStream_t s) {
    using namespace ixg;
    Kv8 c;
    Batch a;
    if (!make_kv8(cache, &c) || !make_batch(n_seq, total_T, cu_seqlens, kv_len, table, width, &a)) return hipErrorInvalidValue;
    if (total_T == 0) return hipSuccess;                      // of tensors without elements, whose addresses may be 0
    if (!rows_ok(k, (long long)c.h_kv * c.d) || !rows_ok(v, (long long)c.h_kv * c.d)) return hipErrorInvalidValue;
    const int few = a.T < (long long)c.page * a.n_seq ? 2 : 1;
    return with_threads(c.page * c.d / 32 / few, [&](auto n) { return launch_append<n>(c, a, k, v, s); });
}

hipError_t ix_kv8_read(const ix_kv8* cache, int n_seq, int total_T, const int32_t* cu_seqlens, const int32_t* kv_len,
                       const int32_t* table, int width, uint16_t* k, uint16_t* v, hipStream_t s) {
    using namespace ixg;
    Kv8 c;
    Batch a;
    if (!make_kv8(cache, &c) || !make_batch(n_seq, total_T, cu_seqlens, kv_len, table, width, &a)) return hipErrorInvalidValue;
    if (total_T == 0) return hipSuccess;
    if ((!k && !v) || !ptr_aligned(k, 2) || !ptr_aligned(v, 2)) return hipErrorInvalidValue;
    return with_threads(c.page * c.d / 32, [&](auto n) { return launch_read<n>(c, a, k, v, s); });
}

}  // extern "C"
