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
// codes, reads the rows once into registers, and turns the values' tile through LDS.
#include "kv8.h"

namespace ixg {
namespace {

constexpr int kCacheThreads = 256;

// The page that slot j of the grid stands for. Sequence b owns the slots from cu[b] / page + 2 b on: at most
// q / page + 2 pages hold its q new tokens, so no prefix sum over the sequences is needed.
struct PageJob {
    int b, id, held, end, row;      // slots held .. end - 1 of page id take the rows from `row` on
};
__device__ __forceinline__ bool page_job(const Batch& a, const Kv8& c, int j, int lane, PageJob* out) {
    const int b = wave_search(a.n_seq, j, lane, [&](int i) { return (a.start(i) >> c.page_log) + 2 * i; });
    const int s0 = a.start(b), q = a.start(b + 1) - s0, kv = a.kv_len[b];
    const int first = kv - q, from = max(first, 0);         // tokens before position 0 are not held
    const int p = (from >> c.page_log) + j - ((s0 >> c.page_log) + 2 * b);
    if (q <= 0 || kv <= 0 || p > (kv - 1) >> c.page_log) return false;
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

__device__ __forceinline__ uint32_t code_of(float x, float s) {
    return (uint8_t)(int8_t)(int)fminf(fmaxf(rintf(x / s), -127.0f), 127.0f);
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

// 8 values of a row, bf16.
__device__ __forceinline__ uint4 load8(const uint16_t* p, bool wide) {
    if (wide) return *reinterpret_cast<const uint4*>(p);
    uint32_t u[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) u[e] = p[2 * e] | ((uint32_t)p[2 * e + 1] << 16);
    return make_uint4(u[0], u[1], u[2], u[3]);
}

// LDS tile of a page's values, [d][page] with rows 4 bytes longer.
constexpr int kTilePad = 4;

// Thread t holds the 8 channels 8 (t % (d/8)) .. + 7 of NC consecutive slots of the page, from slot
// NC (t / (d/8)) on: one 16-byte load a slot, and NC codes of a channel side by side for the values' tile.
template <int NC>
__global__ void __launch_bounds__(kCacheThreads)
append_kernel(Kv8 c, Batch a, const uint16_t* __restrict__ kr, long long k_stride, const uint16_t* __restrict__ vr,
              long long v_stride, bool k_wide, bool v_wide) {
    extern __shared__ uint8_t tile[];
    __shared__ float red[kCacheThreads / kWave];
    const int tid = threadIdx.x, lane = tid & (kWave - 1), h = blockIdx.y;
    const bool is_v = blockIdx.z;
    PageJob job;
    if (!page_job(a, c, blockIdx.x, lane, &job)) return;
    const int per = c.d / 8, col = (tid % per) * 8, slot0 = tid / per * NC;
    const uint16_t* rows = is_v ? vr : kr;
    const long long stride = is_v ? v_stride : k_stride;
    const bool wide = is_v ? v_wide : k_wide;
    const size_t ph = (size_t)job.id * c.h_kv + h;
    float* scale = (is_v ? c.v_scale : c.k_scale) + ph;
    int8_t* codes = (is_v ? c.v : c.k) + ph * c.page * c.d;

    uint4 x[NC];
    float m = 0.0f;
#pragma unroll
    for (int i = 0; i < NC; ++i) {
        const int slot = slot0 + i;
        x[i] = make_uint4(0, 0, 0, 0);
        if (slot >= job.held && slot < job.end)
            x[i] = load8(rows + (long long)(job.row + slot - job.held) * stride + (size_t)h * c.d + col, wide);
    }
    const float old = job.held > 0 ? *scale : 0.0f;
#pragma unroll
    for (int i = 0; i < NC; ++i) m = fmaxf(m, max_abs(x[i]));
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor(m, off, kWave));
    if (lane == 0) red[tid / kWave] = m;
    __syncthreads();                                          // every thread has read the old scale, too
    m = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    const float s = fmaxf(old, m / 127.0f);
    const bool grown = job.held > 0 && s > old;
    const float ratio = grown ? old / s : 1.0f;
    if (tid == 0) *scale = s;

    uint32_t q[NC][2];
#pragma unroll
    for (int i = 0; i < NC; ++i) {
        const uint32_t u[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
        q[i][0] = q[i][1] = 0;
        if (s > 0.0f && slot0 + i >= job.held && slot0 + i < job.end)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t two = code_of(__uint_as_float(u[e] << 16), s) |
                                     code_of(__uint_as_float(u[e] & 0xffff0000u), s) << 8;
                q[i][e / 2] |= two << (16 * (e & 1));
            }
    }
    if (!is_v) {
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            const int slot = slot0 + i;
            if (slot >= job.held && slot < job.end)
                *reinterpret_cast<uint2*>(codes + slot * c.d + col) = make_uint2(q[i][0], q[i][1]);
        }
        if (grown) {
            uint4* p = reinterpret_cast<uint4*>(codes);
            for (int i = tid; i < job.held * c.d / 16; i += kCacheThreads) {
                const uint4 o = p[i];
                p[i] = make_uint4(recode4(o.x, ratio), recode4(o.y, ratio), recode4(o.z, ratio), recode4(o.w, ratio));
            }
        }
        return;
    }
    const int pitch = c.page + kTilePad;
    if (slot0 < c.page) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
#pragma unroll
            for (int i = 0; i < NC; ++i) tile[(col + e) * pitch + slot0 + i] = (uint8_t)(q[i][e / 4] >> (8 * (e & 3)));
    }
    __syncthreads();
    // Channel rows of 16 slots: whole ones at once (slots behind the new tokens hold nothing yet, and get
    // zeros), the one with older tokens in it by bytes, or as a whole where the older ones change too.
    const int spans = c.page / 16;
    for (int i = tid; i < c.d * spans; i += kCacheThreads) {
        const int ch = i / spans, s0 = (i - ch * spans) * 16;
        if (s0 >= job.end || (s0 + 16 <= job.held && !grown)) continue;
        const uint8_t* from = tile + ch * pitch + s0;
        int8_t* to = codes + ch * c.page + s0;
        uint32_t n[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) n[e] = *reinterpret_cast<const uint32_t*>(from + 4 * e);
        if (s0 < job.held) {
            if (!grown) {
                for (int e = job.held - s0; e < min(16, job.end - s0); ++e) to[e] = (int8_t)from[e];
                continue;
            }
            const uint4 o = *reinterpret_cast<const uint4*>(to);
            const uint32_t was[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int keep = min(max(job.held - s0 - 4 * e, 0), 4);          // older slots among these four
                const uint32_t mask = keep == 4 ? 0xffffffffu : (1u << (8 * keep)) - 1;
                n[e] = (recode4(was[e], ratio) & mask) | (n[e] & ~mask);
            }
        }
        *reinterpret_cast<uint4*>(to) = make_uint4(n[0], n[1], n[2], n[3]);
    }
}

__device__ __forceinline__ uint4 values8(uint32_t lo, uint32_t hi, float s) {
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = (float)(int8_t)((e < 4 ? lo : hi) >> (8 * (e & 3))) * s;
    return make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
}

__global__ void __launch_bounds__(kCacheThreads)
read_kernel(Kv8 c, Batch a, uint16_t* __restrict__ ko, uint16_t* __restrict__ vo, bool wide) {
    extern __shared__ uint8_t tile[];
    const int tid = threadIdx.x, lane = tid & (kWave - 1), h = blockIdx.y;
    const bool is_v = blockIdx.z;
    uint16_t* out = is_v ? vo : ko;
    PageJob job;
    if (!out || !page_job(a, c, blockIdx.x, lane, &job)) return;
    const size_t ph = (size_t)job.id * c.h_kv + h;
    const float s = (is_v ? c.v_scale : c.k_scale)[ph];
    const int8_t* codes = (is_v ? c.v : c.k) + ph * c.page * c.d;
    const int per = c.d / 8, pitch = c.page + kTilePad, spans = c.page / 16;
    if (is_v) {
        for (int i = tid; i < c.d * spans; i += kCacheThreads) {
            const int ch = i / spans, s0 = (i - ch * spans) * 16;
            const uint4 o = *reinterpret_cast<const uint4*>(codes + ch * c.page + s0);
            uint32_t* to = reinterpret_cast<uint32_t*>(tile + ch * pitch + s0);
            to[0] = o.x; to[1] = o.y; to[2] = o.z; to[3] = o.w;
        }
        __syncthreads();
    }
    for (int i = tid + job.held * per; i < job.end * per; i += kCacheThreads) {
        const int slot = i / per, col = (i - slot * per) * 8;
        uint2 q;
        if (is_v) {
            uint32_t u[2] = {0, 0};
#pragma unroll
            for (int e = 0; e < 8; ++e) u[e / 4] |= (uint32_t)tile[(col + e) * pitch + slot] << (8 * (e & 3));
            q = make_uint2(u[0], u[1]);
        } else {
            q = *reinterpret_cast<const uint2*>(codes + slot * c.d + col);
        }
        const uint4 v = values8(q.x, q.y, s);
        uint16_t* to = out + ((size_t)(job.row + slot - job.held) * c.h_kv + h) * c.d + col;
        if (wide) {
            *reinterpret_cast<uint4*>(to) = v;
        } else {
            const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int e = 0; e < 8; ++e) to[e] = (uint16_t)(u[e / 2] >> (16 * (e & 1)));
        }
    }
}

dim3 page_grid(const Kv8& c, const Batch& a) {
    return dim3((unsigned)(a.T >> c.page_log) + 2u * (unsigned)a.n_seq, (unsigned)c.h_kv, 2);
}

template <int NC>
void launch_append(const Kv8& c, const Batch& a, const ix_rows* k, const ix_rows* v, hipStream_t s) {
    hipLaunchKernelGGL((append_kernel<NC>), page_grid(c, a), dim3(kCacheThreads), c.d * (c.page + kTilePad), s, c, a, k->p,
                       k->stride, v->p, v->stride, rows_wide(k), rows_wide(v));
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
    if (!rows_ok(k, (long long)c.h_kv * c.d) || !rows_ok(v, (long long)c.h_kv * c.d)) return hipErrorInvalidValue;
    if (total_T == 0) return hipSuccess;
    switch (c.page * c.d / 8 / kCacheThreads) {
        case 0: launch_append<1>(c, a, k, v, s); break;       // 16 x 64: half the threads
        case 1: launch_append<1>(c, a, k, v, s); break;
        case 2: launch_append<2>(c, a, k, v, s); break;
        case 4: launch_append<4>(c, a, k, v, s); break;
        case 8: launch_append<8>(c, a, k, v, s); break;
        default: launch_append<16>(c, a, k, v, s); break;
    }
    return hipGetLastError();
}

hipError_t ix_kv8_read(const ix_kv8* cache, int n_seq, int total_T, const int32_t* cu_seqlens, const int32_t* kv_len,
                       const int32_t* table, int width, uint16_t* k, uint16_t* v, hipStream_t s) {
    using namespace ixg;
    Kv8 c;
    Batch a;
    if (!make_kv8(cache, &c) || !make_batch(n_seq, total_T, cu_seqlens, kv_len, table, width, &a)) return hipErrorInvalidValue;
    if ((!k && !v) || !ptr_aligned(k, 2) || !ptr_aligned(v, 2)) return hipErrorInvalidValue;
    if (total_T == 0) return hipSuccess;
    hipLaunchKernelGGL(read_kernel, page_grid(c, a), dim3(kCacheThreads), c.d * (c.page + kTilePad), s, c, a, k, v,
                       ptr_aligned(k, 16) && ptr_aligned(v, 16));
    return hipGetLastError();
}

}  // extern "C"
