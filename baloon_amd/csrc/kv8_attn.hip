// kv8_attn.hip -- attention of new tokens over the paged 8-bit cache (ix_kv8, kv8.h).
//
//   o_r = sum_j p_rj v_j / sum_j p_rj,  p_rj = exp(scale q_r . k_j)  over the tokens j that row r sees
//
// with k_j = ks c_j and v_j = vs d_j, c and d the codes and ks, vs the scales of the token's page.
#include <type_traits>

#include "kv8.h"

namespace ixg {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
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
    bool q_wide, gate_wide, o_wide;
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

// The largest |x| among bf16 pairs as bits, on which NaN is above infinity.
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ u16x2 max_abs_bits(u16x2 m, const uint4& x) {
    const uint32_t u[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, u[e] & 0x7fff7fffu));
    return m;
}

__device__ __forceinline__ uint4 load_row8(const uint16_t* p, bool wide) {
    if (wide) return *reinterpret_cast<const uint4*>(p);
    uint32_t u[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) u[e] = p[2 * e] | ((uint32_t)p[2 * e + 1] << 16);
    return make_uint4(u[0], u[1], u[2], u[3]);
}

// What the rows of one sequence see together: `ns` tiles of sinks and the tiles lo .. hi - 1.
struct Span {
    int s0, q, kv, first;     // rows s0 .. s0 + q - 1, at positions first ..
    int ns, lo, nt, nrb;      // nt tiles in all (1 where nothing is seen: zeros are written), nrb blocks of rows
    __device__ __forceinline__ int tile(int t) const { return t < ns ? t : lo + t - ns; }
};
template <int ROWS, int TOK>
__device__ __forceinline__ Span span_of(const AttnArgs& A, int b) {
    Span s;
    s.s0 = A.a.start(b);
    s.q = max(A.a.start(b + 1) - s.s0, 0);
    s.kv = max(A.a.kv_len[b], 0);
    s.first = s.kv - s.q;
    s.lo = A.window > 0 ? max(s.first - A.window + 1, 0) / TOK : 0;
    s.ns = A.window > 0 ? min(A.sinks / TOK + (A.sinks % TOK != 0), s.lo) : 0;
    s.nt = max(s.ns + s.kv / TOK + (s.kv % TOK != 0) - s.lo, 1);
    s.nrb = (int)(((long long)s.q * A.G + ROWS - 1) / ROWS);
    return s;
}
template <int ROWS, int TOK>
__device__ __forceinline__ long long work_of(const AttnArgs& A, int b) {
    const Span s = span_of<ROWS, TOK>(A, b);
    return (long long)s.nrb * s.nt * A.c.h_kv;
}

__device__ __forceinline__ long long wave_scan64(long long v, int lane) {
#pragma unroll
    for (int off = 1; off < kWave; off <<= 1) {
        const long long u = __shfl_up(v, off, kWave);
        v += lane >= off ? u : 0;
    }
    return v;
}

// The batch's tiles, numbered through over sequences, kv heads, row blocks and tiles, are shared out evenly:
// workgroup w takes [w per, (w + 1) per). Every wave works the shares out by itself from the lengths.
constexpr int kMinShare = 4;          // tiles: one for each wave
struct Shares {
    long long total, per;
};
template <int ROWS, int TOK>
__device__ __forceinline__ Shares shares(const AttnArgs& A, int n_wg, int lane) {
    long long v = 0;
    for (int b = lane; b < A.a.n_seq; b += kWave) v += work_of<ROWS, TOK>(A, b);
    Shares s;
    s.total = __shfl(wave_scan64(v, lane), kWave - 1, kWave);
    s.per = max((s.total + n_wg - 1) / n_wg, (long long)kMinShare);
    return s;
}
// The sequence that tile `at` belongs to (at < total), and the number of its first tile.
template <int ROWS, int TOK>
__device__ __forceinline__ int locate(const AttnArgs& A, long long at, int lane, long long* base) {
    long long carry = 0;
    for (int b0 = 0;; b0 += kWave) {
        const long long v = b0 + lane < A.a.n_seq ? work_of<ROWS, TOK>(A, b0 + lane) : 0;
        const long long incl = wave_scan64(v, lane);
        const unsigned long long hit = __ballot(carry + incl > at);
        if (hit) {
            const int l = __builtin_ctzll(hit);
            *base = carry + __shfl(incl - v, l, kWave);
            return b0 + l;
        }
        carry += __shfl(incl, kWave - 1, kWave);
    }
}

// Partial results: workgroup w leaves that of the segment it starts in the middle of (or cuts at both
// ends) in slot 2 w, that of another one it ends in the middle of in slot 2 w + 1.
template <int ROWS, int D>
struct Parts {
    float *o, *ml;
    __device__ __forceinline__ Parts(float* p, int n_wg) : o(p), ml(p + (size_t)2 * n_wg * ROWS * D) {}
    static size_t bytes(int n_wg) { return (size_t)2 * n_wg * ROWS * (D + 2) * sizeof(float); }
};

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

// Writes 4 outputs of a row, gated.
__device__ __forceinline__ void store_out(const AttnArgs& A, int t, int h, int d, v4f v) {
    if (A.gate) {
        const uint16_t* g = A.gate + (long long)t * A.gate_stride + (size_t)h * A.c.d + d;
        if (A.gate_wide) {
            const uint2 z = *reinterpret_cast<const uint2*>(g);
            v[0] *= sigmoid_f(__uint_as_float(z.x << 16));
            v[1] *= sigmoid_f(__uint_as_float(z.x & 0xffff0000u));
            v[2] *= sigmoid_f(__uint_as_float(z.y << 16));
            v[3] *= sigmoid_f(__uint_as_float(z.y & 0xffff0000u));
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] *= sigmoid_f(bf16_to_f32(g[e]));
        }
    }
    uint16_t* o = A.o + ((size_t)t * A.h_q + h) * A.c.d + d;
    if (A.o_wide) {
        *reinterpret_cast<uint2*>(o) = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = f32_to_bf16(v[e]);
    }
}

constexpr int kSplitThreads = 256, kSplitWaves = kSplitThreads / kWave, kSplitRows = 16;
// Tokens a wave takes at a time. Keys, values and sums of a 64-token tile are 3/4 D registers, which
// leaves none at D = 256.
template <int D>
constexpr int kSplitTok = D == 256 ? 32 : 64;

// Split over the cache: single tokens and drafted windows.
//
// A segment is a block of 16 (token, head) rows of one sequence and kv head with the tiles its sequence
// sees. A wave takes a tile of 16 S = 64 or 32 tokens by itself, all in registers:
//   S^T = K Q^T on v_mfma_i32_16x16x64_i8: the codes as they are, q as two int8 (q = qs (256 hi + lo), 16 bits of
//     its row's largest value), so the scores are exact integers;
//   P in fp16, its rows where the products left them: a lane's S x 4 scores are 4 S consecutive tokens of
//     one row, because row 4 g + i of product t is made token 4 S g + 4 t + i;
//   O^T += V^T P^T on v_mfma_f32_16x16x32_f16, V's codes converted on the way.
// The page's value scale goes into the exponent (p' = p vs, held relative to its own maximum), and 1 / vs
// into the sum of p.
template <int D>
__global__ void __launch_bounds__(kSplitThreads, 2) split_kernel(AttnArgs A) {
    constexpr int kC = D / 64, kM = D / 16, kPitch = D + 4, kTok = kSplitTok<D>, kS = kTok / 16;
    typedef typename std::conditional<kS == 4, uint4, uint2>::type Codes;     // 4 S values of a channel
    extern __shared__ float lds[];
    float* lo_o = lds;                                        // [waves][16][kPitch]
    float* lo_ml = lds + kSplitWaves * kSplitRows * kPitch;   // [waves][16][2]
    float* lo_qc = lo_ml + kSplitWaves * kSplitRows * 2;      // [16]
    uint4* lo_q = reinterpret_cast<uint4*>(lo_qc + kSplitRows);   // [kC][hi, lo][lane]
    const int tid = threadIdx.x, lane = tid & (kWave - 1), w = __builtin_amdgcn_readfirstlane(tid / kWave);
    const int n = lane & 15, g = lane >> 4, mine = 4 * kS * g, keys = 4 * kS * (n >> 2);
    int b, e, rb, t0, left;
    Span s;
    {
        const AttnArgs& Z = args_again();
        const Shares sh = shares<kSplitRows, kTok>(Z, gridDim.x, lane);
        const long long cur = blockIdx.x * sh.per;
        if (cur >= sh.total) return;
        left = __builtin_amdgcn_readfirstlane((int)min(sh.per, sh.total - cur));
        long long base;
        b = __builtin_amdgcn_readfirstlane(locate<kSplitRows, kTok>(Z, cur, lane, &base));
        s = span_of<kSplitRows, kTok>(Z, b);
        const long long rel = cur - base;
        const int seg = (int)(rel / s.nt);
        t0 = __builtin_amdgcn_readfirstlane((int)(rel - (long long)seg * s.nt));
        e = __builtin_amdgcn_readfirstlane(seg / s.nrb);
        rb = __builtin_amdgcn_readfirstlane(seg - seg / s.nrb * s.nrb);
    }
    for (int piece = 0; left > 0; ++piece) {
        const int t1 = min(s.nt, t0 + left), r0 = rb * kSplitRows, rows = s.q * args_again().G;
        // q as two int8 of 16 bits: wave c takes channels 64 c + 16 g .. + 15 of every row (row n its lanes')
        if (w < kC) {
            const AttnArgs& Z = args_again();
            const int rc = min(r0 + n, rows - 1), qi = rc / Z.G;
            const uint16_t* qp = Z.q + (long long)(s.s0 + qi) * Z.q_stride + (size_t)(e * Z.G + rc - qi * Z.G) * D + 16 * g;
            u16x2 mb = {0, 0};
            uint4 raw[2];
#pragma unroll
            for (int c = 0; c < kC; ++c)
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const uint4 x = load_row8(qp + 64 * c + 8 * k, Z.q_wide);
                    if (c == w) raw[k] = x;
                    mb = max_abs_bits(mb, x);
                }
            uint32_t mu = max((uint32_t)mb[0], (uint32_t)mb[1]);
            mu = max(mu, (uint32_t)__shfl_xor((int)mu, 16, kWave));
            mu = max(mu, (uint32_t)__shfl_xor((int)mu, 32, kWave));
            const float m = __uint_as_float(mu << 16);        // a row that is not finite gets scores that are none
            const float inv = m > 1e-33f ? 32639.0f / m : 0.0f;
            if (w == 0 && g == 0) lo_qc[n] = m * (1.0f / 32639.0f) * Z.scale2;
            uint32_t hi[4] = {0, 0, 0, 0}, lw[4] = {0, 0, 0, 0};
#pragma unroll
            for (int x = 0; x < 16; ++x) {
                const uint4& p = raw[x / 8];
                const uint32_t u = (x & 7) / 2 == 0 ? p.x : (x & 7) / 2 == 1 ? p.y : (x & 7) / 2 == 2 ? p.z : p.w;
                const float v = __uint_as_float(x & 1 ? u & 0xffff0000u : u << 16);
                const int q = (int)rintf(v * inv), h = (q + 128) >> 8;
                hi[x / 4] |= (uint32_t)(h & 255) << (8 * (x & 3));
                lw[x / 4] |= (uint32_t)((q - 256 * h) & 255) << (8 * (x & 3));
            }
            lo_q[(2 * w) * kWave + lane] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
            lo_q[(2 * w + 1) * kWave + lane] = make_uint4(lw[0], lw[1], lw[2], lw[3]);
        }
        __syncthreads();
        const int w_left = parked(left), w_e = parked(e), w_rb = parked(rb), w_b = parked(b), w_s0 = parked(s.s0),
                  w_nrb = parked(s.nrb), w_nt = parked(s.nt), w_rows = parked(rows), w_t0 = parked(t0), w_t1 = parked(t1),
                  w_piece = parked(piece);
        const AttnArgs& Y = args_again();
        const int page_log = Y.c.page_log, window = Y.window, sinks = Y.sinks;
        const int pos = r0 + n < rows ? s.first + (r0 + n) / Y.G : -1;
        const int from = window > 0 ? pos - window + 1 : 0;   // the row sees from .. pos, and the sinks
        // tiles that every row sees as a whole: those starting at full_lo .. full_hi
        const int full_hi = s.first + r0 / Y.G - kTok + 1;
        const int full_lo = window > 0 ? s.first + (min(r0 + kSplitRows, rows) - 1) / Y.G - window + 1 : 0;
        const float qc = lo_qc[n];

        // A tile's places in the cache: this lane's values, scores and scales are of its tokens `mine` on, its
        // keys of those from `keys` on (both within 16 tokens of a page). A lost page's memory is page 0's,
        // hidden below.
        const int32_t* tab = Y.a.table + (size_t)b * Y.a.width;
        const int kv = (int)min((long long)s.kv, (long long)Y.a.width << page_log), n_pages = Y.c.n_pages, h_kv = Y.c.h_kv;
        const int8_t *kb = Y.c.k + ((size_t)e << page_log) * D, *vb = Y.c.v + ((size_t)e << page_log) * D;
        const float *ksb = Y.c.k_scale + e, *vsb = Y.c.v_scale + e;
        asm volatile("" : "+v"(ksb), "+v"(vsb));              // in vector registers, like the parked values
        const uint32_t page_bytes = (uint32_t)(h_kv << page_log) * D;
        const auto page_of = [&](int t, int off) {
            const int j = s.tile(t) * kTok + off;
            const int id = t < t1 && j < kv ? tab[j >> page_log] : -1;
            return (unsigned)id < (unsigned)n_pages ? id : -1;
        };
        const auto slot_of = [&](int t, int off) { return (s.tile(t) * kTok + off) & ((1 << page_log) - 1); };
        uint4 kr[kS][kC];
        Codes vr[kM];
        const auto load_k = [&](int t, int page) {
            const int8_t* p = kb + (size_t)max(page, 0) * page_bytes + (slot_of(t, keys) + (n & 3)) * D + 16 * g;
#pragma unroll
            for (int i = 0; i < kS; ++i)
#pragma unroll
                for (int c = 0; c < kC; ++c) kr[i][c] = *reinterpret_cast<const uint4*>(p + 4 * i * D + 64 * c);
        };
        const auto values_at = [&](int t, int page) {
            return vb + (size_t)max(page, 0) * page_bytes + (n << page_log) + slot_of(t, mine);
        };

        v4f acc[kM];
#pragma unroll
        for (int m = 0; m < kM; ++m) acc[m] = v4f{0, 0, 0, 0};
        float mref = -__builtin_inff(), l = 0.0f;

        int t = t0 + w;
        int pv = page_of(t, mine), pk_next = page_of(t + kSplitWaves, keys), pv_next = page_of(t + kSplitWaves, mine);
        float ks = 0.0f, vs = 0.0f;
        if (t < t1) {
            load_k(t, page_of(t, keys));
            const int8_t* p = values_at(t, pv);
#pragma unroll
            for (int m = 0; m < kM; ++m) vr[m] = *reinterpret_cast<const Codes*>(p + ((size_t)(16 * m) << page_log));
            ks = ksb[(size_t)max(pv, 0) * h_kv];
            vs = vsb[(size_t)max(pv, 0) * h_kv];
        }
        for (; t < t1; t += kSplitWaves) {
            const bool more = t + kSplitWaves < t1;
            const int at = s.tile(t) * kTok;
            asm volatile("" ::: "memory");                    // q is read from LDS again: there are no registers to keep it
            // A block of zeros has scale 0, and its codes are 0.
            const float lv = vs == 0.0f ? 0.0f : log2f(vs);
            const float iv = vs > 0.0f && vs < __builtin_inff() ? 1.0f / vs : 1.0f;
            const float cs = qc * ks;
            float p[4 * kS], top = -__builtin_inff();
#pragma unroll
            for (int i = 0; i < kS; ++i) {
                i32x4 h = {0, 0, 0, 0}, lw = {0, 0, 0, 0};
#pragma unroll
                for (int c = 0; c < kC; ++c) {
                    const i32x4 k = __builtin_bit_cast(i32x4, kr[i][c]);
                    h = __builtin_amdgcn_mfma_i32_16x16x64_i8(k, __builtin_bit_cast(i32x4, lo_q[2 * c * kWave + lane]), h, 0, 0, 0);
                    lw = __builtin_amdgcn_mfma_i32_16x16x64_i8(k, __builtin_bit_cast(i32x4, lo_q[(2 * c + 1) * kWave + lane]), lw, 0, 0, 0);
                }
#pragma unroll
                for (int x = 0; x < 4; ++x) p[4 * i + x] = fmaf((float)((h[x] << 8) + lw[x]), cs, lv);
            }
            const int pv_now = pv;
            __builtin_amdgcn_sched_barrier(0);
            if (more) {
                load_k(t + kSplitWaves, pk_next);
                ks = ksb[(size_t)max(pv_next, 0) * h_kv];
                vs = vsb[(size_t)max(pv_next, 0) * h_kv];
            }
            if (at < full_lo || at > full_hi || __ballot(pv_now < 0)) {
                // of the lane's tokens j0 + y
                const int j0 = at + mine;
                const int last = pv_now < 0 ? -1 : pos - j0;
                const uint32_t seen = low_bits(last + 1) & (low_bits(sinks - j0) | ~low_bits(from - j0));
#pragma unroll
                for (int y = 0; y < 4 * kS; ++y) p[y] = (seen >> y) & 1 ? p[y] : -__builtin_inff();
            }
#pragma unroll
            for (int y = 0; y < 4 * kS; ++y) top = fmaxf(top, p[y]);
            top = pair_max32(pair_max16(top));
            if (__ballot(top > mref + kLag)) {
                const float now = fmaxf(mref, top);
                const float f = now == -__builtin_inff() ? 1.0f : __builtin_amdgcn_exp2f(mref - now);
                mref = now;
                l *= f;
#pragma unroll
                for (int m = 0; m < kM; ++m) acc[m] *= f;
            }
            const float ref = mref == -__builtin_inff() ? 0.0f : mref - kLift;
            f16x8 pf[kS / 2];
#pragma unroll
            for (int y = 0; y < 4 * kS; ++y) {
                const float v = __builtin_amdgcn_exp2f(p[y] - ref);
                l = fmaf(v, iv, l);
                pf[y / 8][y & 7] = (_Float16)v;
            }
            pv = pv_next;
            const int8_t* vp = values_at(t + kSplitWaves, pv);
            pk_next = page_of(t + 2 * kSplitWaves, keys);
            pv_next = page_of(t + 2 * kSplitWaves, mine);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int m0 = 0; m0 < kM; m0 += 4) {
#pragma unroll
                for (int m = m0; m < m0 + 4; ++m)
                    acc[m] = __builtin_amdgcn_mfma_f32_16x16x32_f16(halves8(vr[m].x, vr[m].y), pf[0], acc[m], 0, 0, 0);
                if constexpr (kS == 4) {
#pragma unroll
                    for (int m = m0; m < m0 + 4; ++m)
                        acc[m] = __builtin_amdgcn_mfma_f32_16x16x32_f16(halves8(vr[m].z, vr[m].w), pf[1], acc[m], 0, 0, 0);
                }
                if (more)
#pragma unroll
                    for (int m = m0; m < m0 + 4; ++m) vr[m] = *reinterpret_cast<const Codes*>(vp + ((size_t)(16 * m) << page_log));
                __builtin_amdgcn_sched_barrier(0);
            }
        }

        // the four waves' parts together
        left = taken(w_left), e = taken(w_e), rb = taken(w_rb), b = taken(w_b), t0 = taken(w_t0), piece = taken(w_piece);
        const int s0 = taken(w_s0), nrb = taken(w_nrb), nt = taken(w_nt), rows_ = taken(w_rows), t1_ = taken(w_t1), r0_ = rb * kSplitRows;
        const AttnArgs& Z = args_again();
        l = pair_sum32(pair_sum16(l));
        if (g == 0) {
            lo_ml[(w * kSplitRows + n) * 2] = mref;
            lo_ml[(w * kSplitRows + n) * 2 + 1] = l;
        }
#pragma unroll
        for (int m = 0; m < kM; ++m) *reinterpret_cast<v4f*>(lo_o + (w * kSplitRows + n) * kPitch + 16 * m + 4 * g) = acc[m];
        __syncthreads();
        const bool whole = t0 == 0 && t1_ == nt;
        const int slot = 2 * blockIdx.x + (piece > 0);
        const Parts<kSplitRows, D> parts(Z.part, gridDim.x);
        for (int i = tid; i < kSplitRows * D / 4; i += kSplitThreads) {
            const int row = i / (D / 4), d = i % (D / 4) * 4;
            if (r0_ + row >= rows_) break;
            float top = -__builtin_inff(), total = 0.0f;
            v4f sum = {0, 0, 0, 0};
#pragma unroll
            for (int k = 0; k < kSplitWaves; ++k) top = fmaxf(top, lo_ml[(k * kSplitRows + row) * 2]);
#pragma unroll
            for (int k = 0; k < kSplitWaves; ++k) {
                const float m = lo_ml[(k * kSplitRows + row) * 2];
                const float f = m == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(m - top);
                total = fmaf(lo_ml[(k * kSplitRows + row) * 2 + 1], f, total);
                sum += *reinterpret_cast<const v4f*>(lo_o + (k * kSplitRows + row) * kPitch + d) * f;
            }
            if (whole) {
                const int token = (r0_ + row) / Z.G;
                store_out(Z, s0 + token, e * Z.G + r0_ + row - token * Z.G, d, sum * (total == 0.0f ? 0.0f : 1.0f / total));
            } else {
                *reinterpret_cast<v4f*>(parts.o + ((size_t)slot * kSplitRows + row) * D + d) = sum;
                if (d == 0) {
                    parts.ml[((size_t)slot * kSplitRows + row) * 2] = top;
                    parts.ml[((size_t)slot * kSplitRows + row) * 2 + 1] = total;
                }
            }
        }
        __syncthreads();                                      // lo_o, lo_ml and lo_q are free again
        left -= t1_ - t0;
        if (t1_ == nt && left > 0) {                         // the next segment: row block, head, sequence
            t0 = 0;
            if (++rb == nrb) {
                rb = 0;
                if (++e == Z.c.h_kv) {
                    e = 0;
                    do s = span_of<kSplitRows, kTok>(Z, ++b);       // left > 0: a sequence with rows follows
                    while (s.nrb == 0);
                }
            }
        }
    }
}

// Segments that several workgroups share: the one that lies across the end of workgroup w's tiles, if it
// began in them. Partial results are joined in the workgroups' order.
template <int D>
__global__ void __launch_bounds__(256) join_kernel(AttnArgs A, int n_wg) {
    constexpr int kTok = kSplitTok<D>;
    const int tid = threadIdx.x, lane = tid & (kWave - 1), w = blockIdx.x;
    const Shares sh = shares<kSplitRows, kTok>(A, n_wg, lane);
    const long long edge = (w + 1) * sh.per;
    if (edge >= sh.total) return;
    long long base;
    const int b = __builtin_amdgcn_readfirstlane(locate<kSplitRows, kTok>(A, edge, lane, &base));
    const Span s = span_of<kSplitRows, kTok>(A, b);
    const int seg = (int)((edge - base) / s.nt);
    const long long from = base + (long long)seg * s.nt;
    if (from >= edge || from / sh.per != w) return;
    const int last = (int)((from + s.nt - 1) / sh.per), first_slot = 2 * w + (from > w * sh.per);
    const int e = seg / s.nrb, r0 = (seg - e * s.nrb) * kSplitRows, rows = s.q * A.G;
    const Parts<kSplitRows, D> parts(A.part, n_wg);
    for (int i = tid; i < kSplitRows * D / 4; i += 256) {
        const int row = i / (D / 4), d = i % (D / 4) * 4;
        if (r0 + row >= rows) break;
        float top = -__builtin_inff(), total = 0.0f;
        v4f sum = {0, 0, 0, 0};
        for (int k = w; k <= last; ++k) {
            const size_t at = (size_t)(k == w ? first_slot : 2 * k) * kSplitRows + row;
            const float m = parts.ml[2 * at], lk = parts.ml[2 * at + 1];
            const v4f o = *reinterpret_cast<const v4f*>(parts.o + at * D + d);
            const float now = fmaxf(top, m);
            const float f = top == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(top - now);
            const float fk = m == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(m - now);
            total = fmaf(lk, fk, total * f);
            sum = sum * f + o * fk;
            top = now;
        }
        const int token = (r0 + row) / A.G;
        store_out(A, s.s0 + token, e * A.G + r0 + row - token * A.G, d, sum * (total == 0.0f ? 0.0f : 1.0f / total));
    }
}

template <int D>
void launch_split(const AttnArgs& A, int n_wg, hipStream_t s) {
    const unsigned lds = (kSplitWaves * kSplitRows * (D + 4 + 2) + kSplitRows) * sizeof(float) + D / 64 * 2 * kWave * sizeof(uint4);
    hipLaunchKernelGGL((split_kernel<D>), dim3((unsigned)n_wg), dim3(kSplitThreads), lds, s, A);
    if (n_wg > 1) hipLaunchKernelGGL((join_kernel<D>), dim3((unsigned)n_wg - 1), dim3(256), 0, s, A, n_wg);
}

size_t parts_bytes(int d, int n_wg) {
    return d == 64 ? Parts<kSplitRows, 64>::bytes(n_wg) : d == 128 ? Parts<kSplitRows, 128>::bytes(n_wg)
                                                                   : Parts<kSplitRows, 256>::bytes(n_wg);
}

bool attn_shape_ok(const Kv8& c, int n_seq, int T, int max_q, int h_q) {
    return n_seq > 0 && n_seq <= 65535 && T >= 0 && max_q >= 0 && (T == 0 || max_q > 0) && h_q > 0 && h_q % c.h_kv == 0 &&
           h_q <= 65536;
}

// Two workgroups a CU.
int split_groups(hipStream_t s) { return 2 * device_cu_count(s); }

}  // namespace
}  // namespace ixg

extern "C" {

size_t ix_kv8_attn_workspace_size(const ix_kv8* cache, int n_seq, int total_T, int max_q, int h_q) {
    using namespace ixg;
    Kv8 c;
    if (!make_kv8(cache, &c) || !attn_shape_ok(c, n_seq, total_T, max_q, h_q)) return 0;
    return parts_bytes(c.d, split_groups(nullptr));
}

hipError_t ix_kv8_attn(const ix_kv8* cache, int n_seq, int total_T, int max_q, const int32_t* cu_seqlens,
                       const int32_t* kv_len, const int32_t* table, int width, const ix_rows* q, int h_q, float scale,
                       int window, int sinks, const ix_rows* gate, uint16_t* o, void* workspace, size_t workspace_bytes,
                       hipStream_t s) {
    using namespace ixg;
    AttnArgs A{};
    if (!make_kv8(cache, &A.c) || !make_batch(n_seq, total_T, cu_seqlens, kv_len, table, width, &A.a)) return hipErrorInvalidValue;
    if (!attn_shape_ok(A.c, n_seq, total_T, max_q, h_q) || window < 0 || window > 1 << 30 || sinks < 0) return hipErrorInvalidValue;
    if (!rows_ok(q, (long long)h_q * A.c.d) || (gate && !rows_ok(gate, (long long)h_q * A.c.d))) return hipErrorInvalidValue;
    if (!o || !ptr_aligned(o, 2)) return hipErrorInvalidValue;
    if (!workspace || !ptr_aligned(workspace, 256) ||
        workspace_bytes < ix_kv8_attn_workspace_size(cache, n_seq, total_T, max_q, h_q))
        return hipErrorInvalidValue;
    if (total_T == 0) return hipSuccess;
    A.q = q->p;
    A.q_stride = q->stride;
    A.q_wide = rows_wide(q);
    if (gate) {
        A.gate = gate->p;
        A.gate_stride = gate->stride;
        A.gate_wide = rows_wide(gate);
    }
    A.o = o;
    A.o_wide = ptr_aligned(o, 8);
    A.part = static_cast<float*>(workspace);
    A.scale2 = scale * kLog2e;
    A.h_q = h_q;
    A.G = h_q / A.c.h_kv;
    A.window = window;
    A.sinks = sinks;
    const int n_wg = split_groups(s);
    switch (A.c.d) {
        case 64: launch_split<64>(A, n_wg, s); break;
        case 128: launch_split<128>(A, n_wg, s); break;
        default: launch_split<256>(A, n_wg, s); break;
    }
    return hipGetLastError();
}

}  // extern "C"
