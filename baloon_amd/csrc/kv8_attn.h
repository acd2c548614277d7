// kv8_attn.h -- what the kernels of the attention over the paged 8-bit cache share (kv8_attn.hip, kv8_shared.hip).
#pragma once
#include <algorithm>
#include <type_traits>

#include "kv8.h"

namespace ixg {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr float kLog2e = 0x1.715476p+0f;
// p is formed relative to a reference m that follows the running maximum only once that is kLag above it, and
// 2^kLift times itself: between 2^-24 2^-kLift (fp16's smallest subnormal) and 2^(kLift + kLag), so that neither
// a rescaling per tile nor a loss of small p comes of holding it in fp16.
constexpr float kLag = 7.0f, kLift = 8.0f;

struct AttnArgs {
    Kv8 c;
    Batch a;
    const uint16_t *q, *gate;
    long long q_stride, gate_stride;
    uint16_t* o;
    float* part;              // partial results, see Parts
    float scale2;             // scale * log2(e)
    int h_q, G, window, sinks;
    int narrow;               // the batch has fewer than 2^31 tiles for split_kernel
    int small;                // sequences of more (token, head) rows a kv head than this are block_kernel's
    float* block_part;        // partial results of its blocks, see BlockParts
    int slots, items;         // workgroups of it that the chip holds, and parts of blocks at most
    int first, blocks;        // where a launch of it begins, and its workgroups in all launches
    // Of a batch with shared tokens (kv8_shared.hip):
    const int32_t *groups, *shared;   // sequences groups[g] .. groups[g + 1] - 1 have their first shared[g] tokens in common
    int n_groups, max_q;
    struct SeqPlan* seq;      // [n_seq]
    struct SharedItem* shared_items;  // of block_kernel, each for all heads
    float *item_part, *shared_part;   // partial results of few_kernel's items and of block_kernel's over shared tokens
    int n_items, n_shared;    // room for them
    int many;                 // the groups' rows may be block_kernel's
    float *row_o, *row_ml;    // partial results of rows whose own tokens are block_kernel's: [T][h_q][d], (m, lse) [T][h_q][2]
};

// Which tokens block_kernel takes: of a sequence all, or those behind the shared ones; or of a group those that its sequences share,
// all of its rows together. The latter two leave partial results.
enum Tokens { kAll, kOwn, kShared };
struct SharedItem {
    int s0, rows, r0, row;    // the group's first row of tokens and rows a head, the item's first, and the table's row (-1: there is no item)
    int t0, t1;               // tiles t0 .. t1 - 1 (one at least)
    int kv, unused;
};
// What is where of a sequence: its first own token (0: it shares none), its first item over them and the parts of each of its
// blocks of rows; its group's first item, first row and parts (0: none), and the rows of a block.
struct SeqPlan {
    int from, item, parts;
    int shared_item, s0, shared_parts, shared_rows;
    int unused;
};

// The kernel's argument (its only one) read from memory again where it is used next: keeping all of it in
// scalar registers over the main loop would spill them.
__device__ __forceinline__ const AttnArgs& args_again() {
    auto p = (const __attribute__((address_space(4))) AttnArgs*)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
    return *(const AttnArgs*)p;
}

// A uniform value that waits in a vector register while the main loop needs the scalar ones.
__device__ __forceinline__ int parked(int x) {
    asm volatile("" : "+v"(x));
    return x;
}
__device__ __forceinline__ int taken(int x) { return __builtin_amdgcn_readfirstlane(x); }

__device__ __forceinline__ float pair_max16(float v) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float pair_max32(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// A page's value scale vs weighs its values, not its tokens, so the sum of p has a reference of its own. The values'
// product takes p' = p vs = 2^(score + log2 vs) relative to the largest of those; the sum takes p = 2^score relative to 2^kFar
// of a score among the lane's own tokens, so that it can grow by 2^kFar. A lane's tokens of a tile are of one page: p is p' times
// one factor for all of them. Where that would be above 1 (the page's values next to nothing beside others) p' may be
// gone from 32 bits, and p is worked out by itself; else what 32 bits lose of p' is under 2^(kFar - 126) of the sum.
constexpr float kFar = 60.0f;
// log2 of a page's scale. A page of zeros has none and only takes part in the sum: 2^kNoValue is so far under the least
// scale, 2^-149, that what the product loses when such a page's p' is its largest is under any bf16 number.
constexpr float kNoValue = -200.0f;
__device__ __forceinline__ float log2_scale(float vs) { return vs == 0.0f ? kNoValue : log2f(vs); }

// The sum of a lane's p: l 2^ref.
struct LaneSum {
    float l = 0.0f, ref = -__builtin_inff();
    // What the sum of a tile's p' counts in l. The lane's tokens have p' = 2^(x[] - from) relative to 2^to, the largest of them 2^most
    // (0 where none is seen); lv is log2 vs. 6 instructions and a power for most tiles.
    template <int N>
    __device__ __forceinline__ float factor(const float (&x)[N], float from, float most, float to, float lv) {
        float f;
        if (usual(most, to, lv, &f)) return f;
        asm volatile("");                                     // a branch: not taken at a lane's first tokens, then hardly ever
        return unusual(x, from, most, to, lv);
    }
    __device__ __forceinline__ bool usual(float most, float to, float lv, float* f) const {
        const float a = ref - to + lv;                        // p' is p relative to 2^ref times 2^a
        *f = __builtin_amdgcn_fmed3f(__builtin_amdgcn_exp2f(-a), 0.0f, 1.0f);
        // more than the least that is rare: a if that is >= 0, else next to everything
        return !(most > fminf(a, a * 0x1p100f));
    }
    template <int N>
    __device__ __forceinline__ float unusual(const float (&x)[N], float from, float most, float to, float lv) {
        float a = ref - to + lv;
        if (most > a) {
            const float was = a;
            ref = most + kFar - lv + to;
            a = ref - to + lv;
            l *= __builtin_amdgcn_exp2f(was - a);
        }
        if (a < 0.0f) {
#pragma unroll
            for (int y = 0; y < N; ++y) l += __builtin_amdgcn_exp2f(x[y] - from - a);
        }
        return a < 0.0f ? 0.0f : __builtin_amdgcn_exp2f(-a);
    }
    // log2 of the sum of a row's four lanes, less `to` (finite, near to ref or far below all): itself a score is as large as it likes,
    // and a power of its rounding would be in the result.
    __device__ __forceinline__ float log2_row(float to) const {
        const float top = pair_max32(pair_max16(ref));
        const float f = ref == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(ref - top);
        return top - to + __builtin_amdgcn_logf(pair_sum32(pair_sum16(l * f)));
    }
};

// The largest |x| among bf16 pairs as bits, on which NaN is above infinity.
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ u16x2 max_abs_bits(u16x2 m, const uint4& x) {
    const uint32_t u[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, u[e] & 0x7fff7fffu));
    return m;
}

// 16 bf16 values (a, b) times inv, at most 32639 of them, as 16-bit integers 256 hi + lo of two int8: hi in a, lo
// in b. 1.5 2^23 added to a number leaves its nearest integer in the sum's low bits.
__device__ __forceinline__ void split_q(uint4& a, uint4& b, float inv) {
    constexpr float kMagic = 12582912.0f;
    const uint32_t u[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    uint32_t hi[4], lo[4], two[2];
#pragma unroll
    for (int x = 0; x < 8; ++x) {
        const uint32_t q0 = __float_as_uint(fmaf(__uint_as_float(u[x] << 16), inv, kMagic));
        const uint32_t q1 = __float_as_uint(fmaf(__uint_as_float(u[x] & 0xffff0000u), inv, kMagic));
        two[x & 1] = __builtin_amdgcn_perm(q1, q0, 0x05040100u);
        if (x & 1) {
            lo[x / 2] = __builtin_amdgcn_perm(two[1], two[0], 0x06040200u);
#pragma unroll
            for (int y = 0; y < 2; ++y) two[y] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(u16x2, two[y]) + u16x2{128, 128});
            hi[x / 2] = __builtin_amdgcn_perm(two[1], two[0], 0x07050301u);
        }
    }
    a = make_uint4(hi[0], hi[1], hi[2], hi[3]);
    b = make_uint4(lo[0], lo[1], lo[2], lo[3]);
}

// Inclusive sum over lanes 0 .. l (the steps of wave_scan), and a lane's value in all, for 32 and 64 bits.
template <int Ctrl, int RowMask>
__device__ __forceinline__ int dpp_add(int v) {
    return v + __builtin_amdgcn_update_dpp(0, v, Ctrl, RowMask, 0xF, RowMask == 0xF);
}
template <int Ctrl, int RowMask>
__device__ __forceinline__ long long dpp_add(long long v) {
    const int lo = __builtin_amdgcn_update_dpp(0, (int)v, Ctrl, RowMask, 0xF, RowMask == 0xF);
    const int hi = __builtin_amdgcn_update_dpp(0, (int)(v >> 32), Ctrl, RowMask, 0xF, RowMask == 0xF);
    return v + (long long)(((unsigned long long)(unsigned)hi << 32) | (unsigned)lo);
}
template <class Int>
__device__ __forceinline__ Int wave_scan_int(Int v) {
    v = dpp_add<0x111, 0xF>(v);
    v = dpp_add<0x112, 0xF>(v);
    v = dpp_add<0x114, 0xF>(v);
    v = dpp_add<0x118, 0xF>(v);
    v = dpp_add<0x142, 0xA>(v);
    return dpp_add<0x143, 0xC>(v);
}
__device__ __forceinline__ int lane_of(int v, int l) { return __builtin_amdgcn_readlane(v, l); }
__device__ __forceinline__ long long lane_of(long long v, int l) {
    const unsigned lo = __builtin_amdgcn_readlane((int)v, l), hi = __builtin_amdgcn_readlane((int)(v >> 32), l);
    return (long long)(((unsigned long long)hi << 32) | lo);
}

// The largest of all lanes' v.
template <int Ctrl, int RowMask>
__device__ __forceinline__ int dpp_max(int v) {
    return max(v, __builtin_amdgcn_update_dpp(v, v, Ctrl, RowMask, 0xF, false));
}
__device__ __forceinline__ int wave_max_int(int v) {
    v = dpp_max<0x111, 0xF>(v);
    v = dpp_max<0x112, 0xF>(v);
    v = dpp_max<0x114, 0xF>(v);
    v = dpp_max<0x118, 0xF>(v);
    v = dpp_max<0x142, 0xA>(v);
    return lane_of(dpp_max<0x143, 0xC>(v), kWave - 1);
}
// The lowest n bits, of a n that may lie anywhere.
__device__ __forceinline__ uint32_t low_bits(int n) { return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1; }

// 4 codes to fp16: 0x6400 + (code + 128) is 1024 + code + 128, exactly.
__device__ __forceinline__ void halves(uint32_t raw, f16x2* out) {
    const uint32_t u = raw ^ 0x80808080u;
    const f16x2 bias = {(_Float16)1152.0f, (_Float16)1152.0f};
    out[0] = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) - bias;
    out[1] = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) - bias;
}
__device__ __forceinline__ f16x8 halves8(uint32_t a, uint32_t b) {
    f16x2 h[4];
    halves(a, h);
    halves(b, h + 2);
    return f16x8{h[0][0], h[0][1], h[1][0], h[1][1], h[2][0], h[2][1], h[3][0], h[3][1]};
}

// sigmoid for a bf16 result: v_exp and v_rcp are within an ulp of 32 bits.
__device__ __forceinline__ float sigmoid_16(float x) {
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(x * -kLog2e));
}

__device__ __forceinline__ uint2 load_gate(const AttnArgs& A, int t, int h, int d) {
    uint2 z = make_uint2(0, 0);
    if (A.gate) __builtin_memcpy(&z, A.gate + (long long)t * A.gate_stride + (size_t)h * A.c.d + d, sizeof(z));
    return z;
}
// 4 outputs of a row from its sum of p', o 2^m, and the logarithm of its sum of p, m + lse: o 2^-lse, of which the power alone can
// leave the floats' range.
__device__ __forceinline__ v4f outputs(v4f o, float lse) {
    if (lse == -__builtin_inff()) return v4f{0, 0, 0, 0};
    const float f = __builtin_amdgcn_exp2f(-0.5f * lse);
    return o * f * f;
}
constexpr float kNone = -__FLT_MAX__;      // m of a part without a token: finite, so that lse, -inf, is 0 as a power, without a question
// Partial results (m, lse, o) of a row put together.
struct Joined {
    float m = kNone, top = kNone, total = 0.0f;              // total 2^(m + top): the sum of p
    v4f o = {0, 0, 0, 0};
    // Several that are at hand: m of all, then top of all, then what they add.
    __device__ __forceinline__ void meet_m(float pm) { m = fmaxf(m, pm); }
    __device__ __forceinline__ void meet_sum(float pm, float lse) { top = fmaxf(top, pm - m + lse); }
    __device__ __forceinline__ void add(float pm, float lse, const v4f& po) {
        total += __builtin_amdgcn_exp2f(pm - m + lse - top);
        o += po * __builtin_amdgcn_exp2f(pm - m);
    }
    // One more.
    __device__ __forceinline__ void more(float pm, float lse, const v4f& po) {
        const float now = fmaxf(m, pm), was = m - now + top;
        o *= __builtin_amdgcn_exp2f(m - now);
        m = now;
        top = fmaxf(fmaxf(was, pm - m + lse), kNone);
        total *= __builtin_amdgcn_exp2f(was - top);
        add(pm, lse, po);
    }
    __device__ __forceinline__ float log2_sum() const { return top + __builtin_amdgcn_logf(total); }
};
// 4 channels of a row's partial result.
__device__ __forceinline__ void store_row_part(const AttnArgs& A, int t, int h, int d, const v4f& o, float m, float lse) {
    const size_t row = (size_t)t * A.h_q + h;
    *reinterpret_cast<v4f*>(A.row_o + row * A.c.d + d) = o;
    if (d == 0) *reinterpret_cast<float2*>(A.row_ml + 2 * row) = make_float2(m, lse);
}
// Writes 4 outputs of a row, gated by z.
__device__ __forceinline__ void store_out(const AttnArgs& A, int t, int h, int d, v4f v, uint2 z) {
    if (A.gate) {
        v[0] *= sigmoid_16(__uint_as_float(z.x << 16));
        v[1] *= sigmoid_16(__uint_as_float(z.x & 0xffff0000u));
        v[2] *= sigmoid_16(__uint_as_float(z.y << 16));
        v[3] *= sigmoid_16(__uint_as_float(z.y & 0xffff0000u));
    }
    const uint2 y = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
    __builtin_memcpy(A.o + ((size_t)t * A.h_q + h) * A.c.d + d, &y, sizeof(y));
}
__device__ __forceinline__ void store_out(const AttnArgs& A, int t, int h, int d, v4f v) {
    store_out(A, t, h, d, v, load_gate(A, t, h, d));
}

constexpr int kSplitRows = 16;        // (token, head) rows of a segment of split_kernel and of an item of few_kernel
constexpr int kBlockRows = 128, kBlockTok = 64;               // rows of a block of block_kernel, tokens of its tiles
template <int D>
constexpr float kPartCost = D == 256 ? 4.0f : 8.0f;           // tiles in the time of a part's start, its sums and their joining
constexpr int kLeastPart = 4;         // tiles
// Partial results: sums [item][kRows][D], then (m, lse) [item][kRows][2].
template <int kRows, int D>
struct ItemParts {
    float *o, *ml;
    __device__ __forceinline__ ItemParts(float* p, int n) : o(p), ml(p + (size_t)n * kRows * D) {}
    static size_t bytes(long long n) { return (size_t)n * kRows * (D + 2) * sizeof(float); }
};

// The workgroups and ways of a batch (kv8_attn.hip).
struct Plan {
    bool block, cut;          // block_kernel for sequences of more than kSplitMost rows; in parts
    int n_wg, slots;          // workgroups that the chip holds: of split_kernel two a CU, of block_kernel one or two
    long long full;           // whole blocks that the batch's rows fill
    int max_q;
};
Plan attn_plan(int d, int h_kv, int G, int T, int max_q, hipStream_t s);
size_t attn_bytes(int d, const Plan& p);
// Sequences of more rows a kv head than this are block_kernel's.
int attn_small(const AttnArgs& A, const Plan& p);
// Their partial results over their own tokens, and those of all groups over the shared ones.
hipError_t launch_own_blocks(AttnArgs& A, const Plan& p, hipStream_t s);
hipError_t launch_shared_blocks(AttnArgs& A, int n_wg, hipStream_t s);
// What the calls check alike: the batch (a call without tokens needs no more), and its operands.
bool make_attn(const ix_kv8* cache, int n_seq, int T, int max_q, const int32_t* cu, const int32_t* kv_len, const int32_t* table, int width,
               int h_q, float scale, AttnArgs* A);
bool make_operands(const ix_rows* q, const ix_rows* gate, uint16_t* o, void* workspace, size_t bytes, size_t need, AttnArgs* A);
bool attn_shape_ok(const Kv8& c, int n_seq, int T, int max_q, int h_q);

}  // namespace ixg
