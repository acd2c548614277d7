// kv8_attn.hip -- attention of new tokens over the paged 8-bit cache (ix_kv8, kv8.h).
//
//   o_r = sum_j p_rj v_j / sum_j p_rj,  p_rj = exp(scale q_r . k_j)  over the tokens j that row r sees
//
// with k_j = ks c_j and v_j = vs d_j, c and d the codes and ks, vs the scales of the token's page.
#include "kv8_attn.h"

namespace ixg {
namespace {

// What the rows of one sequence see together: `ns` tiles of sinks and those from `lo` on.
struct Span {
    int s0, q, kv, first;     // rows s0 .. s0 + q - 1, at positions first ..
    int ns, lo, nt, nrb;      // nt tiles in all (1 where nothing is seen: zeros are written), nrb blocks of rows
    __device__ __forceinline__ int tile(int t) const { return t < ns ? t : lo + t - ns; }
};
template <int ROWS, int TOK>
__device__ __forceinline__ Span span_of(const AttnArgs& A, int s0, int q, int kv) {
    Span s;
    s.s0 = s0;
    s.q = (long long)q * A.G <= A.small ? q : 0;
    s.kv = kv;
    s.first = s.kv - q;
    s.lo = A.window > 0 ? max(s.first - A.window + 1, 0) / TOK : 0;
    s.ns = A.window > 0 ? min(A.sinks / TOK + (A.sinks % TOK != 0), s.lo) : 0;
    const int held = (int)min((long long)kv, (long long)A.a.width << A.c.page_log);      // what the table has places for
    s.nt = max(s.ns + max(held / TOK + (held % TOK != 0) - s.lo, 0), 1);
    s.nrb = (int)(((long long)s.q * A.G + ROWS - 1) / ROWS);
    return s;
}
template <int ROWS, int TOK>
__device__ __forceinline__ Span span_at(const AttnArgs& A, int b) {
    const int s0 = A.a.start(b);
    return span_of<ROWS, TOK>(A, s0, max(A.a.start(b + 1) - s0, 0), max(A.a.kv_len[b], 0));
}

// a / b for a >= 0: in 64 bits (below 2^50) through the correctly rounded division in double.
__device__ __forceinline__ int quotient(int a, int b) { return (int)((unsigned)a / (unsigned)b); }
__device__ __forceinline__ long long quotient(long long a, int b) { return (long long)((double)a / (double)b); }

// The batch's tiles, numbered through over sequences, kv heads, row blocks and tiles, are shared out evenly:
// workgroup w takes [w per, (w + 1) per). In front of each segment's tiles `start` more are counted for what a
// workgroup does to begin one, where the shares are long enough for it to matter (37 sequences of 8 kv heads, 296
// segments over 512 workgroups, took 52 us without and 40 with 3 or 6). Every wave works its share out by itself from the
// lengths, in 32 bits where the batch cannot have 2^31 tiles (each launch fetches its instructions anew: 250 of them
// took 1.3 us).
//
// A share is at least kMinShare tiles, one for each wave, but a segment where those have fewer on average, and where
// there is a workgroup for each and they have up to kWhole: joining costs more than a few tiles one after another. 64
// sequences over 8 heads of 128 take, us, with 1 token each 9.3 (18.6 as 4 tiles), 32 with 300 10.2 (15.3) and with 800 16.0
// (18.0); 128 over 2 of 256 with 200 12.9 (20.1) and with 450, 15 tiles, 18.3 (23.5). From 16 tiles on few segments are
// slower whole: 8 sequences over 8 heads of 128, 1,020 tokens each, 13.6 (10.7). Where the limit lies depends on how many
// workgroups are free, which the rule asks only as yes or no. Neither rule keeps a share from lying across two
// segments and beginning both: lengths that a share's tiles do not divide can take more than longer ones that they do (1
// sequence over 2 heads of 256: 900 tokens 13.9, 1,001 11.3, 1,100 14.9).
constexpr int kMinShare = 4, kWhole = 15;
constexpr int kStart = 6;             // tiles of 16 KiB in the time of a segment's start
struct Share {
    int per, left, start;             // counts of every workgroup and of this one, and in front of a segment
    int b, e, rb, v0;                 // where it begins: count v0 of a segment
    Span s;
};
template <int ROWS, int TOK, class Int>
__device__ __forceinline__ bool share_in(const AttnArgs& A, int n_wg, int w, int lane, Share* out) {
    const int n = A.a.n_seq, h_kv = A.c.h_kv;
    Span s{};
    const auto span = [&](int b0) {                          // of sequence b0 + lane; no rows behind the last
        s.nrb = 0;
        if (b0 + lane < n) s = span_at<ROWS, TOK>(A, b0 + lane);
    };
    Int tiles = 0, segments = 0;
#pragma unroll 4
    for (int b0 = (n - 1) & ~(kWave - 1); b0 >= 0; b0 -= kWave) {
        span(b0);
        tiles += (Int)s.nrb * s.nt * h_kv;
        segments += (Int)s.nrb * h_kv;
    }
    tiles = lane_of(wave_scan_int(tiles), kWave - 1);
    segments = lane_of(wave_scan_int(segments), kWave - 1);
    int start = (int)min((Int)kStart, quotient(tiles, 2 * n_wg));
    if (segments * start < n_wg) start = 0;                   // less than a tile for each
    const Int total = tiles + segments * start;
    out->start = start;
    const int mean = (int)min((Int)(kWhole + 1), quotient((Int)(tiles + segments - 1), (int)max(segments, (Int)1)));
    const int least = mean <= kMinShare || (mean <= kWhole && segments <= n_wg) ? mean + start : kMinShare;
    out->per = max((int)quotient((Int)(total + n_wg - 1), n_wg), least);
    const Int cur = (Int)w * out->per;
    if (cur >= total) return false;
    out->left = (int)min((Int)out->per, (Int)(total - cur));
    Int carry = 0;
    for (int b0 = 0;; b0 += kWave) {
        if (b0) span(b0);
        const Int v = (Int)s.nrb * (s.nt + start) * h_kv, incl = wave_scan_int(v);
        const unsigned long long hit = __ballot(carry + incl > cur);
        if (hit) {
            const int l = __builtin_amdgcn_readfirstlane(__builtin_ctzll(hit));
            const Int rel = cur - carry - lane_of((Int)(incl - v), l);
            out->b = b0 + l;
            out->s = span_of<ROWS, TOK>(A, lane_of(s.s0, l), lane_of(s.q, l), lane_of(s.kv, l));
            const int seg = __builtin_amdgcn_readfirstlane((int)quotient(rel, out->s.nt + start));
            out->v0 = __builtin_amdgcn_readfirstlane((int)(rel - (Int)seg * (out->s.nt + start)));
            out->e = quotient(seg, out->s.nrb);
            out->rb = seg - out->e * out->s.nrb;
            return true;
        }
        carry += lane_of(incl, kWave - 1);
    }
}
template <int ROWS, int TOK>
__device__ __forceinline__ bool share_of(const AttnArgs& A, int n_wg, int w, int lane, Share* out) {
    return A.narrow ? share_in<ROWS, TOK, int>(A, n_wg, w, lane, out) : share_in<ROWS, TOK, long long>(A, n_wg, w, lane, out);
}

// Partial results: workgroup w leaves that of the segment it starts in the middle of (or cuts at both
// ends) in slot 2 w, that of another one it ends in the middle of in slot 2 w + 1; and for the segment that lies
// across the end of its tiles, where its parts are.
struct Cut {
    int first, last, slot;            // workgroups first .. last; slot of the first (2 w for the others)
    int row, e, r0, rows;             // its sequence's first row, kv head, first row of the block, rows of the sequence
    int any;
};
template <int ROWS, int D>
struct Parts {
    float *o, *ml;
    Cut* cut;
    __device__ __forceinline__ Parts(float* p, int n_wg)
        : o(p), ml(p + (size_t)2 * n_wg * ROWS * D), cut(reinterpret_cast<Cut*>(ml + (size_t)2 * n_wg * ROWS * 2)) {}
    static size_t bytes(int n_wg) { return (size_t)2 * n_wg * ROWS * (D + 2) * sizeof(float) + n_wg * sizeof(Cut); }
};

constexpr int kSplitThreads = 256, kSplitWaves = kSplitThreads / kWave;
// Tokens a wave takes at a time. Keys, values and sums of a 64-token tile are 3/4 D registers, which
// leaves none at D = 256. Tiles of 32 at D = 128 are faster for some short sequences (48 windows of 1,028 tokens over 4 heads
// 18.6 us for 20.4) and slower for others (16 sequences of 1,000 over 8 heads 15.1 for 13.6), long ones take the same;
// at D = 64 they are slower throughout (64 sequences of 8,000 over 8 heads 103 for 98).
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
// The page's value scale goes into the exponent (p' = p vs, held relative to its own maximum); the sum of p is LaneSum's.
//
// Bound by memory: 128 tokens over 8,000 each, 32 heads over 8 of 128, read 2.1 GB in 360 us, 5.8 of the 6.2 TB/s that reads
// reach, 64 over 1 to 8,192, 16 heads over 2 of 256, 252 MB in 54 and join_kernel's 6. Short contexts are bound by the way to
// the first tile (lengths, pages, codes: about 5 us with the launch), by whole tiles for each of four waves, and by the
// second launch: 48 windows of 1,028 tokens over 4 heads of 128, 51 MB, take 21.0 us where reading takes 8.2.
template <int D>
__global__ void __launch_bounds__(kSplitThreads, 2) split_kernel(AttnArgs A) {
    constexpr int kC = D / 64, kM = D / 16, kPitch = D + 4, kTok = kSplitTok<D>, kS = kTok / 16;
    typedef typename std::conditional<kS == 4, uint4, uint2>::type Codes;     // 4 S values of a channel
    extern __shared__ float lds[];
    float* lo_o = lds;                                        // [waves][16][kPitch]
    float* lo_ml = lds + kSplitWaves * kSplitRows * kPitch;   // [waves][16][2]
    uint32_t* lo_qm = reinterpret_cast<uint32_t*>(lo_ml + kSplitWaves * kSplitRows * 2);   // [waves][16]
    uint4* lo_q = reinterpret_cast<uint4*>(lo_qm + kSplitWaves * kSplitRows);               // [kC][hi, lo][lane]
    const int tid = threadIdx.x, lane = tid & (kWave - 1), w = __builtin_amdgcn_readfirstlane(tid / kWave);
    const int n = lane & 15, g = lane >> 4, mine = 4 * kS * g, keys = 4 * kS * (n >> 2);
    int b, e, rb, v0, left, w_per, start;
    Span s;
    {
        const AttnArgs& Z = args_again();
        Share sh;
        if (!share_of<kSplitRows, kTok>(Z, gridDim.x, blockIdx.x, lane, &sh)) {
            if (tid == 0) Parts<kSplitRows, D>(Z.part, gridDim.x).cut[blockIdx.x].any = 0;
            return;
        }
        b = sh.b, e = sh.e, rb = sh.rb, v0 = sh.v0, left = sh.left, w_per = parked(sh.per), start = sh.start, s = sh.s;
    }

    // The sums of a piece (the part of a segment in this share), for rows n: of 2^(kLift - mref) p' v / vs, and of p.
    v4f acc[kM];
    float mref;
    LaneSum sum;
    // What is left to do for the piece whose sums these are, in vector registers: the main loop needs the scalar ones.
    int o_e = 0, o_r0 = 0, o_rows = 0, o_s0 = 0, o_slot = 0;        // o_slot -1: the whole segment
    bool open = false;
    int pieces = 0;
    Cut cut{};
    for (;;) {
        // The next piece, whose first loads are on their way while the last one's waves are joined.
        int t0 = 0, t1 = 0;
        if (left > 0) {
            t0 = max(v0 - start, 0);
            t1 = min(s.nt, t0 + left - max(start - v0, 0));         // t1 <= t0: only counts of its start are left
        }
        const bool any = t1 > t0;
        if (!any && !open) break;
        const int r0 = rb * kSplitRows, rows = s.q * args_again().G;
        const AttnArgs& Y = args_again();
        const int page_log = Y.c.page_log, window = Y.window, sinks = Y.sinks;
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
        // q: wave c takes channels 64 c + 16 g .. + 15 of every row (row n its lanes')
        uint4 raw[2];
        int t = t0 + w;
        int pk = -1, pv = -1, pk_next = -1, pv_next = -1;
        float ks = 0.0f, vs = 0.0f;
        if (any) {
            if (w < kC) {
                const AttnArgs& Z = args_again();
                const int rc = min(r0 + n, rows - 1), qi = rc / Z.G;
                const uint16_t* qp = Z.q + (long long)(s.s0 + qi) * Z.q_stride + (size_t)(e * Z.G + rc - qi * Z.G) * D + 64 * w + 16 * g;
                raw[0] = load_row8(qp);
                raw[1] = load_row8(qp + 8);
            }
            pk = page_of(t, keys), pv = page_of(t, mine), pk_next = page_of(t + kSplitWaves, keys), pv_next = page_of(t + kSplitWaves, mine);
            if (t < t1) {
                load_k(t, pk);
                const int8_t* p = values_at(t, pv);
#pragma unroll
                for (int m = 0; m < kM; ++m) vr[m] = *reinterpret_cast<const Codes*>(p + ((size_t)(16 * m) << page_log));
                ks = ksb[(size_t)max(pv, 0) * h_kv];
                vs = vsb[(size_t)max(pv, 0) * h_kv];
            }
        }

        if (open) {                                           // the four waves' parts of the last piece together
            const AttnArgs& Z = args_again();
            const int x_r0 = taken(o_r0), x_rows = taken(o_rows), x_slot = taken(o_slot);
            const float m = mref == -__builtin_inff() ? kNone : mref - kLift, lse = sum.log2_row(m);
            if (g == 0) {
                lo_ml[(w * kSplitRows + n) * 2] = m;
                lo_ml[(w * kSplitRows + n) * 2 + 1] = lse;
            }
#pragma unroll
            for (int m = 0; m < kM; ++m) *reinterpret_cast<v4f*>(lo_o + (w * kSplitRows + n) * kPitch + 16 * m + 4 * g) = acc[m];
            lds_barrier();
            const Parts<kSplitRows, D> parts(Z.part, gridDim.x);
            for (int i = tid; i < kSplitRows * D / 4; i += kSplitThreads) {
                const int row = i / (D / 4), d = i % (D / 4) * 4;
                if (x_r0 + row >= x_rows) break;
                Joined to;
#pragma unroll
                for (int k = 0; k < kSplitWaves; ++k) to.meet_m(lo_ml[(k * kSplitRows + row) * 2]);
#pragma unroll
                for (int k = 0; k < kSplitWaves; ++k) to.meet_sum(lo_ml[(k * kSplitRows + row) * 2], lo_ml[(k * kSplitRows + row) * 2 + 1]);
#pragma unroll
                for (int k = 0; k < kSplitWaves; ++k)
                    to.add(lo_ml[(k * kSplitRows + row) * 2], lo_ml[(k * kSplitRows + row) * 2 + 1],
                           *reinterpret_cast<const v4f*>(lo_o + (k * kSplitRows + row) * kPitch + d));
                if (x_slot < 0) {
                    const int token = (x_r0 + row) / Z.G;
                    store_out(Z, taken(o_s0) + token, taken(o_e) * Z.G + x_r0 + row - token * Z.G, d, outputs(to.o, to.log2_sum()));
                } else {
                    *reinterpret_cast<v4f*>(parts.o + ((size_t)x_slot * kSplitRows + row) * D + d) = to.o;
                    if (d == 0) {
                        parts.ml[((size_t)x_slot * kSplitRows + row) * 2] = to.m;
                        parts.ml[((size_t)x_slot * kSplitRows + row) * 2 + 1] = to.log2_sum();
                    }
                }
            }
            lds_barrier();                                    // lo_o and lo_ml are free again
        }
        if (!any) break;

        // q as two int8 of 16 bits
        if (w < kC) {
            u16x2 mb = max_abs_bits(max_abs_bits(u16x2{0, 0}, raw[0]), raw[1]);
            uint32_t mu = max((uint32_t)mb[0], (uint32_t)mb[1]);
            mu = max(mu, (uint32_t)__shfl_xor((int)mu, 16, kWave));
            mu = max(mu, (uint32_t)__shfl_xor((int)mu, 32, kWave));
            if (g == 0) lo_qm[w * kSplitRows + n] = mu;
        }
        lds_barrier();
        uint32_t mu = lo_qm[n];
#pragma unroll
        for (int c = 1; c < kC; ++c) mu = max(mu, lo_qm[c * kSplitRows + n]);
        const float qm = __uint_as_float(mu << 16);           // a row that is not finite gets scores that are none
        const float qc = qm * (1.0f / 32639.0f) * Y.scale2;
        if (w < kC) {
            const float inv = qm > 1e-33f ? 32639.0f / qm : 0.0f;
            split_q(raw[0], raw[1], inv);
            lo_q[(2 * w) * kWave + lane] = raw[0];
            lo_q[(2 * w + 1) * kWave + lane] = raw[1];
        }
        const int pos = r0 + n < rows ? s.first + (r0 + n) / Y.G : -1;
        const int from = window > 0 ? pos - window + 1 : 0;   // the row sees from .. pos, and the sinks
        // tiles that every row sees as a whole: those starting at full_lo .. full_hi
        const int full_hi = s.first + r0 / Y.G - kTok + 1;
        const int full_lo = window > 0 ? s.first + (min(r0 + kSplitRows, rows) - 1) / Y.G - window + 1 : 0;
        lds_barrier();
#pragma unroll
        for (int m = 0; m < kM; ++m) acc[m] = v4f{0, 0, 0, 0};
        mref = -__builtin_inff(), sum = LaneSum{};

        // Where its parts go, and whether it is cut at its end.
        o_e = parked(e), o_r0 = parked(r0), o_rows = parked(rows), o_s0 = parked(s.s0);
        o_slot = parked(t0 == 0 && t1 == s.nt ? -1 : 2 * (int)blockIdx.x + (pieces > 0));
        open = true;
        ++pieces;
        if (t1 < s.nt && tid == 0) {
            const int x = blockIdx.x, per = taken(w_per), before = v0 > start ? (v0 - start + per - 1) / per : 0;
            // the first part is its workgroup's only one so far where the segment began at or before the share
            cut = Cut{x - before, x + (s.nt + start - (t1 + start) + per - 1) / per, before ? 2 * (x - before) + (v0 < before * per) : o_slot,
                      s.s0, e, r0, rows, 1};
        }
        const int n_left = parked(left - (s.nt + start - v0)), n_rb = parked(rb), n_b = parked(b), n_nrb = parked(s.nrb), n_start = parked(start);

        for (; t < t1; t += kSplitWaves) {
            const bool more = t + kSplitWaves < t1;
            const int at = s.tile(t) * kTok;
            asm volatile("" ::: "memory");                    // q is read from LDS again: there are no registers to keep it
            const float lv = log2_scale(vs);
            const float cs = qc * ks;
            float p[4 * kS], most = -__builtin_inff();
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
                asm volatile("");                             // a branch: most tiles are seen as a whole
                // of the lane's tokens j0 + y
                const int j0 = at + mine;
                const int last = pv_now < 0 ? -1 : pos - j0;
                const uint32_t seen = low_bits(last + 1) & (low_bits(sinks - j0) | ~low_bits(from - j0));
#pragma unroll
                for (int y = 0; y < 4 * kS; ++y) p[y] = (seen >> y) & 1 ? p[y] : -__builtin_inff();
            }
#pragma unroll
            for (int y = 0; y < 4 * kS; ++y) most = fmaxf(most, p[y]);
            const float top = pair_max32(pair_max16(most));
            if (__ballot(top > mref + kLag)) {
                const float now = fmaxf(mref, top);
                const float f = now == -__builtin_inff() ? 1.0f : __builtin_amdgcn_exp2f(mref - now);
                mref = now;
#pragma unroll
                for (int m = 0; m < kM; ++m) acc[m] *= f;
            }
            const float ref = mref == -__builtin_inff() ? 0.0f : mref - kLift;
            const float counts = sum.factor(p, ref, most - ref, ref, lv);
            f16x8 pf[kS / 2];
#pragma unroll
            for (int y = 0; y < 4 * kS; ++y) {
                const float v = __builtin_amdgcn_exp2f(p[y] - ref);
                sum.l = fmaf(v, counts, sum.l);
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


        // the next segment: row block, head, sequence
        left = taken(n_left), rb = taken(n_rb) + 1, b = taken(n_b), e = taken(o_e), start = taken(n_start);
        v0 = 0;
        if (left > 0 && rb == taken(n_nrb)) {
            const AttnArgs& Z = args_again();
            rb = 0;
            if (++e == Z.c.h_kv) {
                e = 0;
                do s = span_at<kSplitRows, kTok>(Z, ++b);     // left > 0: a sequence with rows follows
                while (s.nrb == 0);
            }
        }
    }
    if (tid == 0) Parts<kSplitRows, D>(args_again().part, gridDim.x).cut[blockIdx.x] = cut;
}

// Outputs from .. to - 1 (in fours, row by row) of a segment whose partial results are k0 .. k1, the rows of k at at(k).
// Where the outputs are fewer than the threads, several threads take every so many partial results of one and are
// joined in LDS. The order of the sums is fixed.
constexpr int kJoinThreads = 256;
template <int D, Tokens P, class At>
__device__ __forceinline__ void join_outputs(const AttnArgs& A, const float* po, const float* ml, int k0, int k1, At at_part, int from,
                                             int to, int s0, int e, int r0) {
    __shared__ v4f lo_o[kJoinThreads];
    __shared__ float lo_m[kJoinThreads], lo_l[kJoinThreads];
    int wide = 1;                                             // outputs at a time
    while (wide < to - from && wide < kJoinThreads) wide *= 2;
    const int ways = kJoinThreads / wide, way = threadIdx.x / wide;
    for (int x0 = from; x0 < to; x0 += wide) {
        const int x = min(x0 + (int)(threadIdx.x & (wide - 1)), to - 1), row = x / (D / 4), d = x % (D / 4) * 4;
        Joined sum;
#pragma unroll 4
        for (int k = k0 + way; k <= k1; k += ways) {
            const size_t at = at_part(k) + row;
            sum.more(ml[2 * at], ml[2 * at + 1], *reinterpret_cast<const v4f*>(po + at * D + d));
        }
        for (int half = ways / 2; half > 0; half /= 2) {
            lo_o[threadIdx.x] = sum.o;
            lo_m[threadIdx.x] = sum.m;
            lo_l[threadIdx.x] = sum.log2_sum();
            __syncthreads();
            const int other = threadIdx.x + half * wide;
            if (way < half) sum.more(lo_m[other], lo_l[other], lo_o[other]);
            __syncthreads();
        }
        if (way == 0 && x0 + (int)threadIdx.x < to) {
            const int token = (r0 + row) / A.G, t = s0 + token, h = e * A.G + r0 + row - token * A.G;
            if constexpr (P == kOwn) store_row_part(A, t, h, d, sum.o, sum.m, sum.log2_sum());
            else store_out(A, t, h, d, outputs(sum.o, sum.log2_sum()));
        }
    }
}

// Segments that several workgroups share. One that lies across n ends of shares has n workgroups here,
// which take even parts of its outputs.
template <int D>
__global__ void __launch_bounds__(kJoinThreads) join_kernel(AttnArgs A, int n_wg) {
    const Parts<kSplitRows, D> parts(A.part, n_wg);
    const Cut c = parts.cut[blockIdx.x];
    if (!c.any) return;
    const int n = c.last - c.first, i = blockIdx.x - c.first;
    const int all = min(kSplitRows, c.rows - c.r0) * (D / 4);
    const int from = (int)((long long)all * i / n), to = (int)((long long)all * (i + 1) / n);
    const auto at = [&](int k) { return (size_t)(k == c.first ? c.slot : 2 * k) * kSplitRows; };
    join_outputs<D, kAll>(A, parts.o, parts.ml, c.first, c.last, at, from, to, c.row, c.e, c.r0);
}

// Blocks of rows: prompts.
//
// A workgroup of 8 waves takes 128 (token, head) rows of one sequence and kv head, 16 a wave, and the tiles of 64
// tokens that they see one after another through LDS: keys as codes, values as fp16 (converted once for all the
// rows). The products are split_kernel's: S^T = K Q^T in int8 (q in two halves), O^T += V^T P^T in fp16, P where
// the first product left it, because row 4 g + i of key product t is token 16 g + 4 t + i.
//
// 256 rows, 32 a wave on the 32 x 32 shapes, read half as much of LDS but took 231 us for a prompt of 4,096 tokens
// (16 heads over 2 of 256) against 176: it is 256 blocks of 1 to 64 tiles then, one to a CU, and the sums leave no
// registers to read ahead. At D <= 128 two workgroups share a CU.
//
// Those 176 us are 780 TFLOP/s (a large bf16 product reaches 1,240), with the matrix units busy for 33% of it, vector
// instructions issued in 41% and LDS in 36%: the waves of a workgroup pass through products and exponentials together.
// Half of them half a tile behind, with two barriers a tile, took 236 us, the next tile's scores between a tile's
// exponentials and its second product 204 to 212.
constexpr int kBlockThreads = 512;

// LDS of block_kernel, two buffers of each: keys [64 tokens][D], values [D][64 tokens] fp16, and of each 16
// tokens ks and log2 vs.
template <int D>
struct BlockLds {
    static constexpr int kChunks = D / 16;                    // of a token's keys
    static constexpr int kK = kBlockTok * D, kV = 2 * kBlockTok * D, kS = kBlockTok / 16 * 8;
    static constexpr int kVAt = 2 * kK, kSAt = kVAt + 2 * kV, kBytes = kSAt + 2 * kS;
    // Byte offset of 16-byte chunk c of token t's keys, and of chunk c (8 tokens) of channel d's values: both are
    // what they are for c = 0, xor 16 c. A 16-byte read takes 16 lanes at a time over 256 bytes of banks, lanes
    // 0-3, 12-15, 20-23, 24-27 and the others of a half wave: these put the chunks of each such set at different places
    // (with chunks placed for sets of 8 lanes 40% of the LDS cycles were conflicts).
    static __device__ __forceinline__ int k_at(int t, int c) {
        const int r = (t >> 2 & 12) | (t & 3);                // the row of its product
        return t * D + ((c ^ (D == 64 ? (r >> 2) + 3 & 3 : D == 128 ? r >> 1 : r)) << 4);
    }
    static __device__ __forceinline__ int v_at(int d, int c) { return kVAt + d * 128 + ((c ^ ((d >> 1) + 6 & 7)) << 4); }
};

// f of 0 and, if there are two, of 1, as constants.
template <int N, class F>
__device__ __forceinline__ void each(F f) {
    f(std::integral_constant<int, 0>{});
    if constexpr (N == 2) f(std::integral_constant<int, 1>{});
}

// Where the blocks are fewer than the workgroups that the chip holds, several workgroups take parts of a block's tiles,
// as many for each block as fill the chip best, and block_join_kernel joins them: 512 tokens of 32 heads over 8 of 128
// behind 16,384, 128 blocks, took 356 us whole and take 170.
struct BlockCut {
    int first, parts, step;                                   // partial results first, first + step ..
    int s0, e, r0, rows, unused;                              // as in Cut
};
template <int D>
struct BlockParts {
    float *o, *ml;
    BlockCut* cut;
    __device__ __forceinline__ BlockParts(float* p, int slots)
        : o(p), ml(p + (size_t)2 * slots * kBlockRows * D),
          cut(reinterpret_cast<BlockCut*>(ml + (size_t)2 * slots * kBlockRows * 2)) {}
    static size_t bytes(int slots) {
        return (size_t)2 * slots * kBlockRows * (D + 2) * sizeof(float) + (size_t)slots * sizeof(BlockCut);
    }
};
// The blocks of a sequence.
__device__ __forceinline__ int blocks_of(const AttnArgs& A, int b) {
    if (b >= A.a.n_seq) return 0;
    const int rows = max(A.a.start(b + 1) - A.a.start(b), 0) * A.G;
    return rows > A.small ? (rows + kBlockRows - 1) / kBlockRows : 0;
}
// The blocks of all sequences and heads, and in how many parts each is taken: lane p - 1 knows the time of p, in tiles,
// from the rounds of workgroups and the longest block's tiles.
struct Blocks {
    int n, parts;
};
template <int D, Tokens P>
__device__ __forceinline__ Blocks all_blocks(const AttnArgs& A, int lane) {
    int sum = 0, kv = 0;
#pragma unroll 4
    for (int b0 = 0; b0 < A.a.n_seq; b0 += kWave) {
        const int at = min(b0 + lane, A.a.n_seq - 1), v = blocks_of(A, b0 + lane);
        const int held = P == kOwn ? max(A.a.kv_len[at], 0) - A.seq[at].from : A.a.kv_len[at];
        sum += v;
        kv = max(kv, v > 0 ? held : 0);
    }
    Blocks out;
    out.n = lane_of(wave_scan_int(sum), kWave - 1) * A.c.h_kv;
    kv = wave_max_int(kv);
    if (A.window > 0 && A.window < kv) kv = A.window + min(A.sinks, kv - A.window);
    const int p = lane + 1, rounds = (out.n * p + A.slots - 1) / A.slots;
    float cost = (float)rounds * ((float)kv / (float)(kBlockTok * p) + (p > 1 ? kPartCost<D> : 0.0f));
    if (p > 1 && (long long)out.n * p > A.items) cost = __builtin_inff();
    const int least = -wave_max_int(-__float_as_int(cost));   // numbers >= 0 are in the order of their bits
    out.parts = __builtin_amdgcn_readfirstlane(__builtin_ctzll(__ballot(__float_as_int(cost) == least))) + 1;
    return out;
}

template <int D, bool kCut, Tokens P>
__global__ void __launch_bounds__(kBlockThreads, D == 256 ? 2 : 4) block_kernel(AttnArgs A) {
    constexpr int kC = D / 64, kM = D / 16;
    constexpr int kUnits = kBlockTok * D / 16, kPer = (kUnits + kBlockThreads - 1) / kBlockThreads;
    typedef BlockLds<D> Lds;
    extern __shared__ __align__(16) uint8_t block_lds[];
    uint8_t* lds = block_lds;
    const int tid = threadIdx.x, lane = tid & (kWave - 1), w = __builtin_amdgcn_readfirstlane(tid / kWave);
    const int n = lane & 15, g = lane >> 4;

    // Block j of the grid, from the last: of the causal blocks the longest start first. Sequence b owns the
    // blocks from cu[b] G / 128 + b on; consecutive workgroups, which different XCDs take, are different heads.
    const int block = kCut ? (int)blockIdx.x : A.first + (int)blockIdx.x;
    const int e = block % A.c.h_kv;
    int b, rb, parts = 1, part = 0;
    [[maybe_unused]] SharedItem it;
    if constexpr (P == kShared) {
        it = A.shared_items[block / A.c.h_kv];
        if (it.row < 0) return;
        rb = 0, b = it.row;
    } else if constexpr (kCut) {
        const Blocks all = all_blocks<D, P>(A, lane);
        if ((int)blockIdx.x >= all.n * all.parts) return;
        const int i = blockIdx.x / A.c.h_kv;
        parts = all.parts;
        part = i % parts;
        rb = all.n / A.c.h_kv - 1 - i / parts;
        for (int b0 = 0;; b0 += kWave) {
            const int v = blocks_of(A, b0 + lane), incl = wave_scan_int(v);
            const unsigned long long hit = __ballot(incl > rb);
            if (hit) {
                const int l = __builtin_amdgcn_readfirstlane(__builtin_ctzll(hit));
                b = b0 + l;
                rb -= lane_of(incl - v, l);
                break;
            }
            rb -= lane_of(incl, kWave - 1);
        }
    } else {
        const int j = A.blocks / A.c.h_kv - 1 - block / A.c.h_kv;
        const auto key = [&](int b) { return (int)((long long)A.a.start(b) * A.G / kBlockRows) + b; };
        b = wave_search(A.a.n_seq, j, lane, key);
        rb = j - key(b);
    }
    const int s0 = P == kShared ? it.s0 : A.a.start(b), q = P == kShared ? 0 : A.a.start(b + 1) - s0;
    const int r0 = P == kShared ? it.r0 : rb * kBlockRows, rows = P == kShared ? it.rows : max(q, 0) * A.G;
    if (P != kShared && !kCut && (rows <= A.small || rb < 0 || r0 >= rows)) return;      // rb < 0: before the first sequence's rows
    const int kv = P == kShared ? it.kv : max(A.a.kv_len[b], 0), first = kv - q, own = P == kOwn ? A.seq[b].from : 0;
    const auto place = [&](int qi) { return P == kShared ? kv - 1 : first + qi; };       // of new token qi

    // q of row n of the wave, channels 64 c + 16 g .. + 15
    const int w0 = r0 + 16 * w;
    int pos;                                                  // taken from here, the places of the wave below stay scalar
    uint4 qh[kC], ql[kC];
    float qc;
    {
        const int r = w0 + n, rc = min(r, rows - 1), qi = rc / A.G;
        pos = r < rows ? place(qi) : -1;
        const uint16_t* qp = A.q + (long long)(s0 + qi) * A.q_stride + (size_t)(e * A.G + rc - qi * A.G) * D + 16 * g;
        u16x2 mb = {0, 0};
#pragma unroll
        for (int c = 0; c < kC; ++c) {
            qh[c] = load_row8(qp + 64 * c);
            ql[c] = load_row8(qp + 64 * c + 8);
            mb = max_abs_bits(max_abs_bits(mb, qh[c]), ql[c]);
        }
        uint32_t mu = max((uint32_t)mb[0], (uint32_t)mb[1]);
        mu = max(mu, (uint32_t)__shfl_xor((int)mu, 16, kWave));
        mu = max(mu, (uint32_t)__shfl_xor((int)mu, 32, kWave));
        const float m = __uint_as_float(mu << 16), inv = m > 1e-33f ? 32639.0f / m : 0.0f;
        qc = m * (1.0f / 32639.0f) * A.scale2;
#pragma unroll
        for (int c = 0; c < kC; ++c) split_q(qh[c], ql[c], inv);
    }
    // Of the wave's positions wave_first .. wave_last: tiles that start from full_lo to full_hi every row sees as a
    // whole, those below some_lo (the sinks aside) and above wave_last none does.
    const int wave_first = place(min(w0, rows - 1) / A.G), wave_last = place((min(w0 + 16, rows) - 1) / A.G);
    const int full_hi = wave_first - kBlockTok + 1, full_lo = P == kOwn ? own : A.window > 0 ? wave_last - A.window + 1 : 0;
    const int some_lo = P == kAll && A.window > 0 ? wave_first - A.window + 1 - kBlockTok + 1 : 0;

    // the block's tiles
    const int block_first = place(r0 / A.G), block_last = place((min(r0 + kBlockRows, rows) - 1) / A.G);
    const int lo = P == kOwn ? own / kBlockTok : A.window > 0 ? max(block_first - A.window + 1, 0) / kBlockTok : 0;
    const int ns = P == kAll && A.window > 0 ? min(A.sinks / kBlockTok + (A.sinks % kBlockTok != 0), lo) : 0;
    const int all = block_last < 0 ? 0 : max(ns + block_last / kBlockTok + 1 - lo, 0);
    int begin = 0, nt = all;                                  // this part's: tiles begin .. begin + nt - 1
    if constexpr (P == kShared) {
        begin = it.t0;
        nt = it.t1 - it.t0;
    } else if constexpr (kCut) {
        if (parts > 1) {
            const int i = blockIdx.x / A.c.h_kv / parts;
            parts = min(parts, max(all / kLeastPart, 1));
            if (part == 0 && tid == 0)
                BlockParts<D>(A.block_part, A.slots).cut[i * A.c.h_kv + e] = BlockCut{(int)blockIdx.x, parts, A.c.h_kv, s0, e, r0, rows, 0};
            if (part >= parts) return;
            begin = all / parts * part + min(part, all % parts);
            nt = all / parts + (part < all % parts);
        }
    }
    const auto tile = [&](int t) { return (begin + t < ns ? begin + t : lo + begin + t - ns) * kBlockTok; };

    // Copies of a tile: 16-byte pieces 512 i + tid of its keys, token by token, and of its values, page by page
    // and in a page (or 64 tokens of it) channel by channel. The pieces of one wave's i are in one page.
    const int page_log = A.c.page_log, part_log = min(page_log, 6);
    constexpr int kDLog = D == 64 ? 6 : D == 128 ? 7 : 8;
    const int32_t* tab = A.a.table + (size_t)b * A.a.width;
    const int kv_held = (int)min((long long)kv, (long long)A.a.width << page_log);
    // Lane g of 0 .. 3 holds the page of the tile's tokens 16 g .. + 15, loaded a tile ahead of its use.
    const auto pages = [&](int at) {
        const int x = at + 16 * (lane & 3);
        const int id = x < kv_held ? tab[x >> page_log] : -1;
        return (unsigned)id < (unsigned)A.c.n_pages ? id : -1;
    };
    const auto memory = [&](const int8_t* p, int id) {        // this head's of a page
        return p + (((size_t)max(id, 0) * A.c.h_kv + e) << page_log) * D;
    };
    const bool copies = kUnits >= kBlockThreads || w < kUnits / kWave;
    u32x4 held[kPer], held_v[kPer];
    const auto pages_of = [&](int ids, int (&page_k)[kPer], int (&page_v)[kPer]) {
        each<kPer>([&](auto i) {
            const int first = (w * kWave + i * kBlockThreads) * 16;
            page_k[i] = __builtin_amdgcn_readlane(ids, first >> (kDLog + 4) & 3);
            page_v[i] = __builtin_amdgcn_readlane(ids, first >> (kDLog + part_log) << (part_log - 4) & 3);
        });
    };
    const auto load_k = [&](int at, const int (&page_k)[kPer]) {
        const uint32_t off = (16 * tid) & ((D << part_log) - 1);
        each<kPer>([&](auto i) {
            const int8_t* p = memory(A.c.k, page_k[i]) + (at & ((1 << page_log) - 1)) * D + ((i * kBlockThreads * 16) & ((D << part_log) - 1));
            if (copies) held[i] = *reinterpret_cast<const u32x4*>(p + off);
        });
    };
    const auto store_k = [&](int buf) {
        const int u = tid, to = Lds::k_at(u / Lds::kChunks, u % Lds::kChunks) + buf * Lds::kK;
        each<kPer>([&](auto i) {
            if (copies) *reinterpret_cast<u32x4*>(lds + ((to + i * kBlockThreads * 16) ^ (i * 128))) = held[i];      // 32 tokens on: rows 8 on
        });
    };
    const auto load_v = [&](int at, const int (&page_v)[kPer]) {
        const uint32_t y = (16 * tid) & ((D << part_log) - 1), off = y + (page_log == 7 ? y & ~63u : 0u);
        each<kPer>([&](auto i) {
            const uint32_t step = ((i * kBlockThreads * 16) & ((D << part_log) - 1)) << (page_log - part_log);   // more channels
            const int8_t* p = memory(A.c.v, page_v[i]) + (at & ((1 << page_log) - 1)) + step;
            if (copies) held_v[i] = *reinterpret_cast<const u32x4*>(p + off);
        });
    };
    const auto store_v = [&](int buf) {
        const uint32_t u = 16 * tid, y = u & ((D << part_log) - 1);
        const int d = y >> part_log, g = ((u >> (kDLog + part_log)) << (part_log - 4)) + (y >> 4 & ((1 << (part_log - 4)) - 1));
        const int to = Lds::v_at(d, 2 * g) + buf * Lds::kV;
        const int more_d = part_log == 6 ? 128 * (kBlockThreads / 4) : 0, more_t = part_log == 6 ? 0 : 64;
        each<kPer>([&](auto i) {
            // the second piece: channels 128 on, or tokens 32 on
            const int at = (to + i * more_d) ^ (i * more_t);
            if (copies) {
                *reinterpret_cast<f16x8*>(lds + at) = halves8(held_v[i][0], held_v[i][1]);
                *reinterpret_cast<f16x8*>(lds + (at ^ 16)) = halves8(held_v[i][2], held_v[i][3]);
            }
        });
    };
    // Scales of 16 tokens by one thread each. A lost page's tokens get the logarithm of 0.
    float ks = 0.0f, vs = 0.0f;
    const auto load_scale = [&](int ids) {
        if (tid < kBlockTok / 16) {
            ks = A.c.k_scale[(size_t)max(ids, 0) * A.c.h_kv + e];
            vs = A.c.v_scale[(size_t)max(ids, 0) * A.c.h_kv + e];
            if (ids < 0) vs = -1.0f;                          // no scale is negative
        }
    };
    const auto store_scale = [&](int buf) {
        if (tid < kBlockTok / 16) {
            *reinterpret_cast<float2*>(lds + Lds::kSAt + buf * Lds::kS + 8 * tid) =
                make_float2(vs < 0.0f ? 0.0f : ks, vs < 0.0f ? -__builtin_inff() : log2_scale(vs));
        }
    };
    const int k0 = Lds::k_at((n >> 2) * 16 + (n & 3), g), v0 = Lds::v_at(n, 2 * g);

    v4f acc[kM];
#pragma unroll
    for (int m = 0; m < kM; ++m) acc[m] = v4f{0, 0, 0, 0};
    // p' is taken relative to 2^ref; a lane whose row gets one over 2^limit of it moves ref there.
    float ref = 0.0f, limit = -__builtin_inff();
    LaneSum sum;

    int ids = pages(tile(0)), page_k[kPer], page_v[kPer];
    pages_of(ids, page_k, page_v);
    if (nt > 0) {
        load_k(tile(0), page_k);
        load_v(tile(0), page_v);
        load_scale(ids);
        store_k(0);
        store_v(0);
        store_scale(0);
    }
    ids = pages(tile(min(1, max(nt - 1, 0))));
    lds_barrier();
    for (int t = 0; t < nt; ++t) {
        const int buf = t & 1, at = tile(t), next = tile(min(t + 1, nt - 1));
        const int kt = buf * Lds::kK + k0, vt = buf * Lds::kV + v0;      // bits 4 to 7 are k0's and v0's
        pages_of(ids, page_k, page_v);
        load_k(next, page_k);
        load_v(next, page_v);
        load_scale(ids);
        ids = pages(tile(min(t + 2, nt - 1)));
        if (at <= wave_last && (at >= some_lo || at < A.sinks)) {
            const float2 sc = *reinterpret_cast<const float2*>(lds + Lds::kSAt + buf * Lds::kS + 8 * g);
            float p[16], most = -__builtin_inff();            // lane: row n, tokens at + 16 g + y
            const float cs = qc * sc.x, lv = sc.y - ref;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                i32x4 hi = {0, 0, 0, 0}, lw = {0, 0, 0, 0};
#pragma unroll
                for (int c = 0; c < kC; ++c) {
                    const i32x4 k = *reinterpret_cast<const i32x4*>(lds + (kt ^ (64 * c)) + 4 * i * D);
                    hi = __builtin_amdgcn_mfma_i32_16x16x64_i8(k, __builtin_bit_cast(i32x4, qh[c]), hi, 0, 0, 0);
                    lw = __builtin_amdgcn_mfma_i32_16x16x64_i8(k, __builtin_bit_cast(i32x4, ql[c]), lw, 0, 0, 0);
                }
#pragma unroll
                for (int y = 0; y < 4; ++y) p[4 * i + y] = fmaf((float)((hi[y] << 8) + lw[y]), cs, lv);
            }
            if (at < full_lo || at > full_hi) {
                asm volatile("");                             // a branch: most tiles are seen as a whole
                const int j0 = at + 16 * g, from = P == kOwn ? own : A.window > 0 ? pos - A.window + 1 : 0;
                const uint32_t seen = low_bits(pos - j0 + 1) & (low_bits(A.sinks - j0) | ~low_bits(from - j0));
#pragma unroll
                for (int y = 0; y < 16; ++y) p[y] = (seen >> y) & 1 ? p[y] : -__builtin_inff();
            }
#pragma unroll
            for (int y = 0; y < 16; ++y) most = fmaxf(most, p[y]);
            const float top = pair_max32(pair_max16(most));
            if (__ballot(top > limit)) {
                const float mref = limit == -__builtin_inff() ? limit : ref + kLift;
                const float now = fmaxf(mref, top + ref), to = now == -__builtin_inff() ? 0.0f : now - kLift;
                const float f = now == -__builtin_inff() ? 1.0f : __builtin_amdgcn_exp2f(mref - now);
#pragma unroll
                for (int y = 0; y < 16; ++y) p[y] += ref - to;
                most += ref - to;
                ref = to;
                limit = now == -__builtin_inff() ? now : kLift + kLag;
#pragma unroll
                for (int m = 0; m < kM; ++m) acc[m] *= f;
            }
            const float counts = sum.factor(p, 0.0f, most, ref, sc.y);
            f16x8 pf[2];
            float of_tile = 0.0f;
#pragma unroll
            for (int y = 0; y < 16; ++y) {
                const float v = __builtin_amdgcn_exp2f(p[y]);
                of_tile += v;                                 // before its rounding: a small page's p' loses bits by it
                pf[y / 8][y & 7] = (_Float16)v;
            }
            sum.l = fmaf(of_tile, counts, sum.l);
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int m = 0; m < kM; ++m)
                    acc[m] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                        *reinterpret_cast<const f16x8*>(lds + (vt ^ (16 * s)) + 16 * m * 128), pf[s], acc[m], 0, 0, 0);
        }
        store_k(buf ^ 1);
        store_v(buf ^ 1);
        store_scale(buf ^ 1);
        lds_barrier();
    }

    const float m_ref = limit == -__builtin_inff() ? kNone : ref, lse = sum.log2_row(m_ref);
    int thread = tid;
    asm volatile("" : "+v"(thread));                          // the row is worked out again: it does not wait in registers
    const int r = w0 + (thread & 15), qi = r / A.G, head = e * A.G + r - qi * A.G, d0 = 4 * (thread >> 4 & 3);
    if constexpr (P == kShared) {
        const ItemParts<kBlockRows, D> to(A.shared_part, A.n_shared);
        const size_t at = (size_t)block * kBlockRows + (r - r0);
        if (r < rows) {
            if (d0 == 0) *reinterpret_cast<float2*>(to.ml + 2 * at) = make_float2(m_ref, lse);
#pragma unroll
            for (int m = 0; m < kM; ++m) *reinterpret_cast<v4f*>(to.o + at * D + 16 * m + d0) = acc[m];
        }
        return;
    }
    if (kCut && parts > 1) {
        const BlockParts<D> to(A.block_part, A.slots);
        const size_t at = (size_t)blockIdx.x * kBlockRows + (r - r0);
        if (r < rows) {
            if (d0 == 0) *reinterpret_cast<float2*>(to.ml + 2 * at) = make_float2(m_ref, lse);
#pragma unroll
            for (int m = 0; m < kM; ++m) *reinterpret_cast<v4f*>(to.o + at * D + 16 * m + d0) = acc[m];
        }
        return;
    }
    if (P == kOwn && r < rows) {
#pragma unroll
        for (int m = 0; m < kM; ++m) store_row_part(A, s0 + qi, head, 16 * m + d0, acc[m], m_ref, lse);
    } else if (r < rows) {
        constexpr int kN = kM < 8 ? kM : 8;                   // pieces of 4 channels, their gates on the way together
#pragma unroll
        for (int m0 = 0; m0 < kM; m0 += kN) {
            uint2 z[kN];
#pragma unroll
            for (int i = 0; i < kN; ++i) z[i] = load_gate(A, s0 + qi, head, 16 * (m0 + i) + d0);
#pragma unroll
            for (int i = 0; i < kN; ++i) store_out(A, s0 + qi, head, 16 * (m0 + i) + d0, outputs(acc[m0 + i], lse), z[i]);
        }
    }
}

// Every block's outputs are shared out over as many workgroups as there are for each.
template <int D, Tokens P>
__global__ void __launch_bounds__(kJoinThreads) block_join_kernel(AttnArgs A) {
    const Blocks blocks = all_blocks<D, P>(A, threadIdx.x & (kWave - 1));
    if (blocks.parts == 1) return;
    const int n = (int)gridDim.x / blocks.n, k = blockIdx.x % blocks.n, i = blockIdx.x / blocks.n;
    if (i >= n) return;
    const BlockParts<D> parts(A.block_part, A.slots);
    const BlockCut c = parts.cut[k];
    if (c.parts == 1) return;
    const int all = min(kBlockRows, c.rows - c.r0) * (D / 4);
    const auto at = [&](int k) { return (size_t)(c.first + k * c.step) * kBlockRows; };
    join_outputs<D, P>(A, parts.o, parts.ml, 0, c.parts - 1, at, (int)((long long)all * i / n), (int)((long long)all * (i + 1) / n),
                    c.s0, c.e, c.r0);
}

// Sequences of at most kSplitMost (token, head) rows a kv head are split_kernel's in any case, and so are all where the
// batch's rows fill fewer than least_blocks(D) blocks. A block takes the same time with 1 row and with 128, and
// split_kernel that of its 16s: 128 sequences over 4 kv heads of 128, 4,096 tokens each, take with 32, 48 and 64 rows
// 193, 283 and 371 us there and 187, 187 and 194 here, with 512 tokens 32, 43 and 54 to 36, 40 and 42. Few blocks are few
// workgroups, or parts that must be joined: 16, 32 and 64 blocks of one sequence take, at D = 128 behind 16,384 tokens,
// 60, 104 and 186 us there and 44, 61 and 96 here, behind 2,048 tokens 19, 28 and 35 to 28, 30 and 31, and behind none 9,
// 10 and 11 to 15; at D = 256 16 blocks 130, 33 and 15 to 60, 30 and 22, at D = 64 64 blocks 106, 21 and 9 to 69, 23 and 12.
constexpr int kSplitMost = 32;
constexpr int least_blocks(int d) { return 4096 / d; }

Plan plan_of(int d, int h_kv, int G, int T, int max_q, hipStream_t s) {
    Plan p;
    const int n_cu = device_cu_count(s);
    p.n_wg = 2 * n_cu;
    p.slots = d == 256 ? n_cu : 2 * n_cu;
    p.full = (long long)T * G / kBlockRows * h_kv;
    p.max_q = max_q;
    p.block = (long long)max_q * G > kSplitMost && p.full >= least_blocks(d);
    p.cut = p.block && p.full < p.slots;
    return p;
}

template <int D>
size_t split_bytes(const Plan& p) { return (Parts<kSplitRows, D>::bytes(p.n_wg) + 255) / 256 * 256; }
// Also where this batch's blocks stay whole: those of a smaller one, which the workspace has to do for as well, may not.
template <int D>
size_t attn_bytes(const Plan& p) { return split_bytes<D>(p) + (p.block ? BlockParts<D>::bytes(p.slots) : 0); }

template <int D, bool kCut, Tokens P>
hipError_t launch_blocks(AttnArgs& A, long long n, hipStream_t s) {
    static OncePerDevice once;
    const hipError_t ready = allow_lds(once, &block_kernel<D, kCut, P>, BlockLds<D>::kBytes, s);
    if (ready != hipSuccess) return ready;
    A.blocks = (int)n;
    return launch_in_pieces(n, kBlockThreads, [&](long long first, unsigned count) {      // one, of blocks in parts
        A.first = (int)first;
        hipLaunchKernelGGL((block_kernel<D, kCut, P>), dim3(count), dim3(kBlockThreads), BlockLds<D>::kBytes, s, A);
    });
}

// With at most max_q new tokens in each other one, a sequence of the batch has at least these. Where that is more than
// kSplitMost rows all are block_kernel's (also those of a batch whose offsets end before T), and it is the only launch.
int small_of(const AttnArgs& A, const Plan& p) {
    const long long shortest = A.a.T - (long long)(A.a.n_seq - 1) * p.max_q;
    return p.block && shortest * A.G > kSplitMost ? 0 : p.block ? kSplitMost : 0x7fffffff;
}
template <int D, Tokens P>
hipError_t launch_seq_blocks(AttnArgs& A, const Plan& p, hipStream_t s) {
    if (!p.cut) return launch_blocks<D, false, P>(A, p.full + (long long)A.a.n_seq * A.c.h_kv, s);
    // a sequence has at most one block that is not full, and more than kSplitMost rows
    const long long most = A.small == 0 ? A.a.n_seq : std::min((long long)A.a.n_seq, (long long)A.a.T * A.G / kSplitMost);
    const long long blocks = p.full + most * A.c.h_kv;
    A.slots = p.slots;
    A.items = 2 * p.slots;
    A.block_part = A.part + split_bytes<D>(p) / sizeof(float);
    const hipError_t e = launch_blocks<D, true, P>(A, std::max(blocks, (long long)A.items), s);
    if (e == hipSuccess) hipLaunchKernelGGL((block_join_kernel<D, P>), dim3((unsigned)(2 * p.n_wg)), dim3(kJoinThreads), 0, s, A);
    return e;
}

template <int D>
hipError_t launch_attn(AttnArgs& A, const Plan& p, hipStream_t s) {
    const int n_wg = p.n_wg;
    A.small = small_of(A, p);
    // tiles: at most those of a whole table for each block of rows, and n_wg - 1 and a workgroup's share more in sums
    const long long row_blocks = (long long)A.a.T * A.G / kSplitRows + A.a.n_seq;
    const long long tiles = ((long long)A.a.width << A.c.page_log) / kSplitTok<D> + 1;
    A.narrow = row_blocks < (1ll << 31) / tiles / A.c.h_kv / 2 - n_wg;
    if (p.block) {
        const hipError_t e = launch_seq_blocks<D, kAll>(A, p, s);
        if (e != hipSuccess) return e;
        if (A.small == 0) return hipGetLastError();
    }
    const unsigned lds = kSplitWaves * kSplitRows * (D + 4 + 2 + 1) * sizeof(float) + D / 64 * 2 * kWave * sizeof(uint4);
    hipLaunchKernelGGL((split_kernel<D>), dim3((unsigned)n_wg), dim3(kSplitThreads), lds, s, A);
    if (n_wg > 1) hipLaunchKernelGGL((join_kernel<D>), dim3((unsigned)n_wg - 1), dim3(kJoinThreads), 0, s, A, n_wg);
    return hipGetLastError();
}

}  // namespace

Plan attn_plan(int d, int h_kv, int G, int T, int max_q, hipStream_t s) { return plan_of(d, h_kv, G, T, max_q, s); }
size_t attn_bytes(int d, const Plan& p) { return d == 64 ? attn_bytes<64>(p) : d == 128 ? attn_bytes<128>(p) : attn_bytes<256>(p); }
int attn_small(const AttnArgs& A, const Plan& p) { return small_of(A, p); }
hipError_t launch_own_blocks(AttnArgs& A, const Plan& p, hipStream_t s) {
    const hipError_t e = A.c.d == 64 ? launch_seq_blocks<64, kOwn>(A, p, s)
                         : A.c.d == 128 ? launch_seq_blocks<128, kOwn>(A, p, s) : launch_seq_blocks<256, kOwn>(A, p, s);
    return e == hipSuccess ? hipGetLastError() : e;
}
hipError_t launch_shared_blocks(AttnArgs& A, int n_wg, hipStream_t s) {
    A.slots = n_wg;
    switch (A.c.d) {
        case 64: return launch_blocks<64, false, kShared>(A, A.n_shared, s);
        case 128: return launch_blocks<128, false, kShared>(A, A.n_shared, s);
        default: return launch_blocks<256, false, kShared>(A, A.n_shared, s);
    }
}

// The blocks of the batch are numbered in 31 bits.
bool attn_shape_ok(const Kv8& c, int n_seq, int T, int max_q, int h_q) {
    return n_seq > 0 && n_seq <= 65535 && T >= 0 && max_q >= 0 && (T == 0 || max_q > 0) && h_q > 0 && h_q % c.h_kv == 0 &&
           h_q <= 65536 && (long long)T * h_q <= 1ll << 37;
}
bool make_attn(const ix_kv8* cache, int n_seq, int T, int max_q, const int32_t* cu, const int32_t* kv_len, const int32_t* table, int width,
               int h_q, float scale, AttnArgs* A) {
    if (!make_kv8(cache, &A->c) || !make_batch(n_seq, T, cu, kv_len, table, width, &A->a)) return false;
    if (!attn_shape_ok(A->c, n_seq, T, max_q, h_q)) return false;
    A->scale2 = scale * kLog2e;
    A->h_q = h_q;
    A->G = h_q / A->c.h_kv;
    return true;
}
bool make_operands(const ix_rows* q, const ix_rows* gate, uint16_t* o, void* workspace, size_t bytes, size_t need, AttnArgs* A) {
    const long long row = (long long)A->h_q * A->c.d;
    if (!rows_ok(q, row) || (gate && !rows_ok(gate, row)) || !o || !ptr_aligned(o, 2)) return false;
    if (!workspace || !ptr_aligned(workspace, 256) || bytes < need) return false;
    A->q = q->p;
    A->q_stride = q->stride;
    if (gate) {
        A->gate = gate->p;
        A->gate_stride = gate->stride;
    }
    A->o = o;
    A->part = static_cast<float*>(workspace);
    return true;
}

}  // namespace ixg

extern "C" {

size_t ix_kv8_attn_workspace_size(const ix_kv8* cache, int n_seq, int total_T, int max_q, int h_q) {
    using namespace ixg;
    Kv8 c;
    if (!make_kv8(cache, &c) || !attn_shape_ok(c, n_seq, total_T, max_q, h_q)) return 0;
    return attn_bytes(c.d, plan_of(c.d, c.h_kv, h_q / c.h_kv, total_T, max_q, nullptr));
}

hipError_t ix_kv8_attn(const ix_kv8* cache, int n_seq, int total_T, int max_q, const int32_t* cu_seqlens,
                       const int32_t* kv_len, const int32_t* table, int width, const ix_rows* q, int h_q, float scale,
                       int window, int sinks, const ix_rows* gate, uint16_t* o, void* workspace, size_t workspace_bytes,
                       hipStream_t s) {
    using namespace ixg;
    AttnArgs A{};
    if (!make_attn(cache, n_seq, total_T, max_q, cu_seqlens, kv_len, table, width, h_q, scale, &A)) return hipErrorInvalidValue;
    if (window < 0 || window > 1 << 30 || sinks < 0) return hipErrorInvalidValue;
    if (total_T == 0) return hipSuccess;                      // of tensors without elements, whose addresses may be 0
    const Plan p = plan_of(A.c.d, A.c.h_kv, A.G, total_T, max_q, s);
    if (!make_operands(q, gate, o, workspace, workspace_bytes, attn_bytes(A.c.d, p), &A)) return hipErrorInvalidValue;
    A.window = window;
    A.sinks = sinks;
    switch (A.c.d) {
        case 64: return launch_attn<64>(A, p, s);
        case 128: return launch_attn<128>(A, p, s);
        default: return launch_attn<256>(A, p, s);
    }
}

}  // extern "C"
