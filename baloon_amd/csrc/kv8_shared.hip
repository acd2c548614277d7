// kv8_shared.hip -- attention over the paged 8-bit cache of a batch whose sequences have their first tokens in common.
//
// A row's softmax over all its tokens is put together of that over the shared ones and that over its own (kv8_attn.h, Joined):
// with partial results (m, l, o), p taken relative to 2^m, o = sum_i o_i 2^(m_i - m) / sum_i l_i 2^(m_i - m). So the rows of all of
// a group's sequences go over the shared tokens together, those of each over its own, and gather_kernel puts the partial results
// together. few_kernel takes 16 rows a workgroup: each sequence's own tokens, and the shared ones of groups of few rows, all of
// these in one launch; block_kernel (kv8_attn.hip) takes 128: the shared tokens of groups of many rows, and prompts.
#include "kv8_attn.h"

namespace ixg {
namespace {

constexpr int kThreads = 256, kWaves = kThreads / kWave;
template <int D>
constexpr int kTokOf = D == 256 ? 32 : 64;

// The groups in the lanes of a wave, if there are up to 64.
struct Groups {
    Group g;
    int first, last;
};
__device__ __forceinline__ Groups groups_in_lanes(const AttnArgs& A, int lane) {
    Groups out{};
    if (A.n_groups > kWave || lane >= A.n_groups) return out;
    out.g = group_at(A, lane);
    out.first = group_first(A, lane);
    out.last = group_first(A, lane + 1);
    return out;
}
// The first own token of sequence b, a lane's own.
__device__ __forceinline__ int first_own(const AttnArgs& A, const Groups& groups, int b) {
    int from = 0;
    if (A.n_groups <= kWave) {
        for (int x = 0; x < A.n_groups; ++x)
            from = b >= lane_of(groups.first, x) && b < lane_of(groups.last, x) ? lane_of(groups.g.kv, x) : from;
        return from;
    }
    int lo = 0, n = A.n_groups;                               // the last group that begins at b or before
    while (n > 1) {
        const int half = n / 2;
        const bool right = group_first(A, lo + half) <= b;
        lo += right ? half : 0;
        n = right ? n - half : half;
    }
    return b >= group_first(A, lo) && b < group_first(A, lo + 1) ? group_at(A, lo).kv : 0;
}

// What few_kernel takes: the groups, where they have few rows, and behind them the sequences of few rows.
struct Unit {
    int s0, rows;             // rows s0 G .. of a kv head, in blocks of 16; 0: nothing to do
    int t0, nt;               // its tiles (one at least)
    int first, kv;            // position of row 0 (of a group far behind its tokens), and tokens
};
template <int D>
__device__ __forceinline__ Unit unit_at(const AttnArgs& A, const Groups& groups, int u) {
    constexpr int kTok = kTokOf<D>;
    const int n_groups = A.few ? A.n_groups : 0;
    Unit out{};
    if (u < n_groups) {
        const Group g = group_at(A, u);
        out = Unit{g.s0, g.rows, 0, g.kv / kTok, 1 << 30, g.kv};
    } else if (u - n_groups < A.a.n_seq) {
        const int b = u - n_groups, s0 = A.a.start(b), q = max(A.a.start(b + 1) - s0, 0), kv = max(A.a.kv_len[b], 0);
        const int held = (int)min((long long)kv, (long long)A.a.width << A.c.page_log);
        const int t0 = first_own(A, groups, b) / kTok;
        out = Unit{s0, (long long)q * A.G <= A.small ? q * A.G : 0, t0, max(held / kTok + (held % kTok != 0) - t0, 1), kv - q, held};
    }
    return out;
}
__device__ __forceinline__ int blocks_of(const Unit& u) { return (u.rows + kSplitRows - 1) / kSplitRows; }
__device__ __forceinline__ Unit unit_of_lane(const Unit& u, int l) {
    return Unit{lane_of(u.s0, l), lane_of(u.rows, l), lane_of(u.t0, l), lane_of(u.nt, l), lane_of(u.first, l), lane_of(u.kv, l)};
}

// A unit's blocks are taken in parts of up to `chunk` tiles: as few as leave at most `rounds` items for each workgroup. Item
// ((blocks and parts of the units before it) + block * parts + part) * h_kv + head. A piece of work is never two units', however
// short: a workgroup's way to its first tile is longer than several of them (64 sequences of up to 1,000 own tokens behind 8,190
// shared ones took split_kernel, whose shares are cut at one length, 16 us; drafts of 37 sequences of up to 500 took it 25).
struct FewCuts {
    int chunk, units;
    __device__ __forceinline__ int parts(const Unit& u) const { return (u.nt + chunk - 1) / chunk; }
};
// The items of `segments` blocks: at most this.
__host__ __device__ inline long long few_items(long long segments, int n_wg) {
    const long long rounds = segments / n_wg + 1;
    return (rounds * n_wg - segments < n_wg / 4 ? rounds + 1 : rounds) * n_wg;
}
template <int D>
__device__ __forceinline__ FewCuts few_cuts(const AttnArgs& A, const Groups& groups, int n_wg, int lane) {
    FewCuts out;
    out.units = (A.few ? A.n_groups : 0) + A.a.n_seq;
    long long tiles = 0, segments = 0;
    for (int u0 = 0; u0 < out.units; u0 += kWave) {
        const Unit u = unit_at<D>(A, groups, u0 + lane);
        tiles += (long long)blocks_of(u) * u.nt;
        segments += blocks_of(u);
    }
    tiles = lane_of(wave_scan_int(tiles), kWave - 1) * A.c.h_kv;
    segments = lane_of(wave_scan_int(segments), kWave - 1) * A.c.h_kv;
    const long long room = few_items(segments, n_wg) - segments;
    out.chunk = (int)min(max((tiles + room - 1) / room, (long long)kWaves), 0x7fffffffll);
    return out;
}

// What block_kernel and gather_kernel ask of a sequence, by a workgroup that does nothing else.
template <int D>
__device__ __forceinline__ void write_plan(const AttnArgs& A, const Groups& groups, const FewCuts& cuts, int tid) {
    const int lane = tid & (kWave - 1), n_groups = A.few ? A.n_groups : 0;
    for (int b = tid; b < A.a.n_seq; b += kThreads) A.seq[b] = SeqPlan{};
    __syncthreads();
    if (tid >= kWave) return;
    const Cuts blocks = A.few ? Cuts{1} : cuts_of<D>(A, A.slots, lane);
    int base = 0;
    for (int g0 = 0; g0 < A.n_groups; g0 += kWave) {
        const Group g = group_at(A, g0 + lane);
        const int first = g.rows ? group_first(A, g0 + lane) : 0, last = g.rows ? group_first(A, g0 + lane + 1) : 0;
        const Unit u{g.s0, g.rows, 0, g.kv / kTokOf<D>, 0, 0};
        const int parts = A.few ? cuts.parts(u) : blocks.parts(g), items = (A.few ? blocks_of(u) : Cuts::blocks(g)) * parts;
        const int before = wave_scan_int(items) - items;
        unsigned long long todo = __ballot(g.rows > 0);
        while (todo) {                                        // all lanes for one group's sequences
            const int l = __builtin_ctzll(todo);
            todo &= todo - 1;
            const int item = base + lane_of(before, l), s0 = lane_of(g.s0, l), n = lane_of(parts, l);
            for (int b = lane_of(first, l) + lane; b < lane_of(last, l); b += kWave) {
                A.seq[b].shared_item = item;
                A.seq[b].s0 = s0;
                A.seq[b].shared_parts = n;
            }
        }
        base += lane_of(before + items, kWave - 1);
    }
    base = A.few ? base : 0;
    for (int u0 = n_groups; u0 < cuts.units; u0 += kWave) {
        const Unit u = unit_at<D>(A, groups, u0 + lane);
        const int parts = cuts.parts(u), items = blocks_of(u) * parts, before = wave_scan_int(items) - items, b = u0 - n_groups + lane;
        if (b < A.a.n_seq) {
            A.seq[b].from = u.t0 * kTokOf<D>;
            A.seq[b].item = base + before;
            A.seq[b].parts = parts;
        }
        base += lane_of(before + items, kWave - 1);
    }
}

// An item is 16 rows of a unit over a part of its tiles. A wave takes a tile of kTok tokens at a time by itself, all in registers,
// with the next one's loads under way; products and the layout of P are those of split_kernel.
template <int D>
__global__ void __launch_bounds__(kThreads, 2) few_kernel(AttnArgs A_) {
    constexpr int kC = D / 64, kM = D / 16, kPitch = D + 4, kTok = kTokOf<D>, kS = kTok / 16;
    typedef typename std::conditional<kS == 4, uint4, uint2>::type Codes;     // 4 S values of a channel
    extern __shared__ float lds[];
    uint4* lo_q = reinterpret_cast<uint4*>(lds);              // [kC][hi, lo][lane]
    uint32_t* lo_qm = reinterpret_cast<uint32_t*>(lo_q + kC * 2 * kWave);     // [kC][16]
    float* lo_o = lds;                                        // behind the tiles: [waves][16][kPitch]
    float* lo_ml = lds + kWaves * kSplitRows * kPitch;        // [waves][16][2]
    const int n_wg = gridDim.x - 1;
    FewCuts cuts;
    {
        const AttnArgs& A = args_again();
        const Groups groups = groups_in_lanes(A, threadIdx.x & (kWave - 1));
        cuts = few_cuts<D>(A, groups, n_wg, threadIdx.x & (kWave - 1));
        if ((int)blockIdx.x == n_wg) {
            write_plan<D>(A, groups, cuts, threadIdx.x);
            return;
        }
    }
    for (int item = blockIdx.x;; item += n_wg) {
        int tid = threadIdx.x;
        asm volatile("" : "+v"(tid));                         // worked out again for each item: not kept over the main loop
        const int lane = tid & (kWave - 1), w = __builtin_amdgcn_readfirstlane(tid / kWave);
        const int n = lane & 15, g = lane >> 4, mine = 4 * kS * g, keys = 4 * kS * (n >> 2);
        const AttnArgs& A = args_again();
        const int h_kv = A.c.h_kv, page_log = A.c.page_log, n_pages = A.c.n_pages, e = item % h_kv;
        // its unit, block and part
        Unit it;
        int table_row = -1, r0 = 0, t = 0, t1 = 0;
        {
            const Groups groups = groups_in_lanes(A, lane);
            const int n_groups = A.few ? A.n_groups : 0;
            int left = item / h_kv;
            for (int u0 = 0; u0 < cuts.units; u0 += kWave) {
                const Unit u = unit_at<D>(A, groups, u0 + lane);
                const int p = cuts.parts(u), count = blocks_of(u) * p, incl = wave_scan_int(count);
                const unsigned long long hit = __ballot(incl > left);
                if (hit) {
                    const int l = __builtin_amdgcn_readfirstlane(__builtin_ctzll(hit));
                    const int parts = lane_of(p, l), in = left - lane_of(incl - count, l), part = in % parts;
                    it = unit_of_lane(u, l);
                    table_row = u0 + l < n_groups ? group_first(A, u0 + l) : u0 + l - n_groups;
                    r0 = in / parts * kSplitRows;
                    t = it.t0 + (int)((long long)it.nt * part / parts) + w;
                    t1 = it.t0 + (int)((long long)it.nt * (part + 1) / parts);
                    break;
                }
                left -= lane_of(incl, kWave - 1);
            }
        }
        if (table_row < 0) return;
        const int n_rows = it.rows - r0, kv = it.kv;
        const int32_t* tab = A.a.table + (size_t)table_row * A.a.width;
        const int8_t *kb = A.c.k + ((size_t)e << page_log) * D, *vb = A.c.v + ((size_t)e << page_log) * D;
        const float *ksb = A.c.k_scale + e, *vsb = A.c.v_scale + e;
        int step = 16 << page_log;                            // of 16 channels
        asm volatile("" : "+v"(ksb), "+v"(vsb), "+v"(kb), "+v"(vb), "+v"(step));           // not in scalar registers, which are few
        const uint32_t page_bytes = (uint32_t)(h_kv << page_log) * D;
        // What is loaded of a tile behind the last is the last's again, and not used.
        const auto page_of = [&](int t, int off) {
            const int j = min(t, t1 - 1) * kTok + off, id = j < kv ? tab[j >> page_log] : -1;
            return (unsigned)id < (unsigned)n_pages ? id : -1;
        };
        const auto slot_of = [&](int t, int off) { return (min(t, t1 - 1) * kTok + off) & ((1 << page_log) - 1); };
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
        int pv = page_of(t, mine), pk_next = page_of(t + kWaves, keys), pv_next = page_of(t + kWaves, mine);
        // q: wave c takes channels 64 c + 16 g .. + 15 of every row (row n its lanes'), as two int8 of 16 bits
        uint4 raw[2] = {};
        if (w < kC) {
            const int rc = min(r0 + n, it.rows - 1), qi = rc / A.G;
            const uint16_t* qp = A.q + (long long)(it.s0 + qi) * A.q_stride + (size_t)(e * A.G + rc - qi * A.G) * D + 64 * w + 16 * g;
            raw[0] = load_row8(qp);
            raw[1] = load_row8(qp + 8);
        }
        load_k(t, page_of(t, keys));
        {
            const int8_t* p = values_at(t, pv);
#pragma unroll
            for (int m = 0; m < kM; ++m, p += step) vr[m] = *reinterpret_cast<const Codes*>(p);
        }
        float ks = ksb[(size_t)max(pv, 0) * h_kv], vs = vsb[(size_t)max(pv, 0) * h_kv];
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
        const float qc = qm * (1.0f / 32639.0f) * A.scale2;
        if (w < kC) {
            split_q(raw[0], raw[1], qm > 1e-33f ? 32639.0f / qm : 0.0f);
            lo_q[2 * w * kWave + lane] = raw[0];
            lo_q[(2 * w + 1) * kWave + lane] = raw[1];
        }
        const int pos = it.first + (r0 + n) / A.G, full = it.first + r0 / A.G - kTok + 1;       // tiles that start there or before are seen whole
        lds_barrier();

        v4f acc[kM];
        float mref = -__builtin_inff();
        LaneSum sum;
#pragma unroll
        for (int m = 0; m < kM; ++m) acc[m] = v4f{0, 0, 0, 0};
        for (; t < t1; t += kWaves) {
            asm volatile("" ::: "memory");                    // q is read from LDS again: there are no registers to keep it
            const float lv = log2_scale(vs), cs = qc * ks;
            const bool lost = pv < 0;
            const int at = t * kTok;
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
                for (int y = 0; y < 4; ++y) p[4 * i + y] = fmaf((float)((h[y] << 8) + lw[y]), cs, lv);
            }
            __builtin_amdgcn_sched_barrier(0);
            load_k(t + kWaves, pk_next);
            ks = ksb[(size_t)max(pv_next, 0) * h_kv];
            vs = vsb[(size_t)max(pv_next, 0) * h_kv];
            if (at > full || __ballot(lost)) {
                asm volatile("");                             // a branch: most tiles are seen as a whole
                const uint32_t seen = lost ? 0 : low_bits(pos - at - mine + 1);
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
            float of_tile = 0.0f;
#pragma unroll
            for (int y = 0; y < 4 * kS; ++y) {
                const float v = __builtin_amdgcn_exp2f(p[y] - ref);
                of_tile += v;                                 // before its rounding: a small page's p' loses bits by it
                pf[y / 8][y & 7] = (_Float16)v;
            }
            sum.l = fmaf(of_tile, counts, sum.l);
            pv = pv_next;
            const int8_t* vp = values_at(t + kWaves, pv);
            pk_next = page_of(t + 2 * kWaves, keys);
            pv_next = page_of(t + 2 * kWaves, mine);
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
#pragma unroll
                for (int m = m0; m < m0 + 4; ++m, vp += step) vr[m] = *reinterpret_cast<const Codes*>(vp);
                __builtin_amdgcn_sched_barrier(0);
            }
        }

        // the four waves' parts together
        const ItemParts<kSplitRows, D> parts(args_again().item_part, args_again().n_items);
        const float m = mref == -__builtin_inff() ? kNone : mref - kLift, lse = sum.log2_row(m);
        lds_barrier();                                        // q has been read
        if (g == 0) {
            lo_ml[(w * kSplitRows + n) * 2] = m;
            lo_ml[(w * kSplitRows + n) * 2 + 1] = lse;
        }
#pragma unroll
        for (int y = 0; y < kM; ++y) *reinterpret_cast<v4f*>(lo_o + (w * kSplitRows + n) * kPitch + 16 * y + 4 * g) = acc[y];
        lds_barrier();
        for (int i = tid; i < kSplitRows * D / 4; i += kThreads) {
            const int row = i / (D / 4), d = i % (D / 4) * 4;
            if (row >= n_rows) break;
            Joined to;
#pragma unroll
            for (int k = 0; k < kWaves; ++k) to.meet_m(lo_ml[(k * kSplitRows + row) * 2]);
#pragma unroll
            for (int k = 0; k < kWaves; ++k) to.meet_sum(lo_ml[(k * kSplitRows + row) * 2], lo_ml[(k * kSplitRows + row) * 2 + 1]);
#pragma unroll
            for (int k = 0; k < kWaves; ++k)
                to.add(lo_ml[(k * kSplitRows + row) * 2], lo_ml[(k * kSplitRows + row) * 2 + 1],
                       *reinterpret_cast<const v4f*>(lo_o + (k * kSplitRows + row) * kPitch + d));
            *reinterpret_cast<v4f*>(parts.o + ((size_t)item * kSplitRows + row) * D + d) = to.o;
            if (d == 0) *reinterpret_cast<float2*>(parts.ml + ((size_t)item * kSplitRows + row) * 2) = make_float2(to.m, to.log2_sum());
        }
        lds_barrier();                                        // the next item's q goes there
    }
}

// Puts each row's partial results together and writes it: a workgroup takes up to 256 outputs (in fours) of 16 rows of a sequence and
// head. The 16s of sequence b are numbered from start G / 16 + b on, with gaps. kRows: the blocks of groups.
template <int D, int kRows>
__global__ void __launch_bounds__(kThreads) gather_kernel(AttnArgs A, int first) {
    constexpr int kPer = kSplitRows * (D / 4) / kThreads;     // workgroups of a block
    const int tid = threadIdx.x, lane = tid & (kWave - 1), h_kv = A.c.h_kv;
    const int all = first + (int)blockIdx.x, piece = all % kPer, e = all / kPer % h_kv, j = all / kPer / h_kv;
    const auto key = [&](int b) { return (int)((long long)A.a.start(b) * A.G / kSplitRows) + b; };
    const int b = wave_search(A.a.n_seq, j, lane, key);
    const int s0 = A.a.start(b), rows = max(A.a.start(b + 1) - s0, 0) * A.G, rb = j - key(b), r0 = rb * kSplitRows;
    if (rb < 0 || r0 >= rows) return;                         // rb < 0: before the first sequence's rows
    const int row = (piece * kThreads + tid) / (D / 4), d = tid % (D / 4) * 4, r = r0 + row;
    if (r >= rows) return;
    const int qi = r / A.G, t = s0 + qi, h = e * A.G + r - qi * A.G;
    const uint2 z = load_gate(A, t, h, d);
    const SeqPlan plan = A.seq[b];
    Joined sum;
    const auto add = [&](const auto& parts, int block, int rows_of, int first_item, int n, int in) {
        size_t at = ((size_t)(first_item + block * n) * h_kv + e) * rows_of + in;
#pragma unroll 8
        for (int k = 0; k < n; ++k, at += (size_t)h_kv * rows_of)
            sum.more(parts.ml[2 * at], parts.ml[2 * at + 1], *reinterpret_cast<const v4f*>(parts.o + at * D + d));
    };
    const ItemParts<kSplitRows, D> few(A.item_part, A.n_items);
    if (rows <= A.small) {
        add(few, rb, kSplitRows, plan.item, plan.parts, row);
    } else {
        const size_t at = (size_t)t * A.h_q + h;
        sum.more(A.row_ml[2 * at], A.row_ml[2 * at + 1], *reinterpret_cast<const v4f*>(A.row_o + at * D + d));
    }
    if (plan.shared_parts > 0) {
        const int of_group = (t - plan.s0) * A.G + r - qi * A.G, block = of_group / kRows, in = of_group - block * kRows;
        if constexpr (kRows == kSplitRows) add(few, block, kRows, plan.shared_item, plan.shared_parts, in);
        else add(ItemParts<kRows, D>(A.shared_part, A.n_shared), block, kRows, plan.shared_item, plan.shared_parts, in);
    }
    store_out(A, t, h, d, outputs(sum.o, sum.log2_sum()), z);
}

// The workspace: what block_kernel needs over the sequences' own tokens, the plan, few_kernel's items, and, where block_kernel takes
// any, partial results of the rows and of its items over the shared tokens.
struct SharedPlan {
    Plan own;
    bool few;                 // groups' rows are few_kernel's
    int n_wg;                 // workgroups of block_kernel that the chip holds
    long long n_items, n_shared;
    size_t seq, items, shared, row_o, row_ml, bytes;
};
// Groups of up to this many rows a kv head in the mean are few_kernel's.
constexpr int kFewRows = 32;
SharedPlan shared_plan(int d, int h_kv, int G, int n_seq, int T, int max_q, int n_groups, hipStream_t s) {
    SharedPlan p;
    p.own = attn_plan(d, h_kv, G, T, max_q, s);
    const long long rows = (long long)T * G, nonempty = std::min(n_seq, T);
    p.few = rows <= (long long)kFewRows * n_groups;
    p.n_wg = d == 256 ? p.own.n_wg / 2 : p.own.n_wg;
    // a sequence or group has at most one block that is not full
    const auto segments = [&](bool few) { return (rows / kSplitRows + nonempty + (few ? rows / kSplitRows + n_groups : 0)) * h_kv; };
    const auto blocks = [&] {
        const long long n = (rows / kBlockRows + n_groups) * h_kv;
        return n < p.n_wg / 2 ? p.n_wg : (n + p.n_wg - 1) / p.n_wg * p.n_wg + p.n_wg;
    };
    p.n_items = few_items(segments(p.few), p.own.n_wg - 1);
    p.n_shared = p.few ? 0 : blocks();
    const auto up = [](size_t n) { return (n + 255) / 256 * 256; };
    const auto item_bytes = [&](long long n, int block) { return up((size_t)n * block * (d + 2) * sizeof(float)); };
    p.seq = attn_bytes(d, p.own);
    p.items = p.seq + up(n_seq * sizeof(SeqPlan));
    // room as for groups of many rows and of few: a smaller batch's may be either
    p.shared = p.items + item_bytes(few_items(segments(true), p.own.n_wg - 1), kSplitRows);
    p.row_o = p.shared + item_bytes(blocks(), kBlockRows);
    p.row_ml = p.row_o + (p.own.block ? up((size_t)rows * h_kv * d * sizeof(float)) : 0);
    p.bytes = p.row_ml + (p.own.block ? up((size_t)rows * h_kv * 2 * sizeof(float)) : 0);
    // workgroups and items are numbered in 31 bits; a batch beyond that has more outputs than the GPU has memory
    if (segments(true) > 1 << 28 || (rows / kSplitRows + n_seq) * h_kv * (kSplitRows * (d / 4) / kThreads) > 0x7fffffff) p.bytes = 0;
    return p;
}

template <int D>
hipError_t launch_shared(AttnArgs& A, const SharedPlan& p, hipStream_t s) {
    char* ws = reinterpret_cast<char*>(A.part);
    A.seq = reinterpret_cast<SeqPlan*>(ws + p.seq);
    A.item_part = reinterpret_cast<float*>(ws + p.items);
    A.shared_part = reinterpret_cast<float*>(ws + p.shared);
    A.row_o = reinterpret_cast<float*>(ws + p.row_o);
    A.row_ml = reinterpret_cast<float*>(ws + p.row_ml);
    A.n_items = (int)p.n_items;
    A.n_shared = (int)p.n_shared;
    A.few = p.few;
    A.slots = p.n_wg;
    A.small = attn_small(A, p.own);
    constexpr unsigned lds = kWaves * kSplitRows * (D + 4 + 2) * sizeof(float);
    static OncePerDevice once;
    hipError_t e = allow_lds(once, &few_kernel<D>, lds, s);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((few_kernel<D>), dim3((unsigned)p.own.n_wg), dim3(kThreads), lds, s, A);
    e = hipGetLastError();
    if (e == hipSuccess && !p.few) e = launch_shared_blocks(A, p.n_wg, s);
    if (e == hipSuccess && p.own.block) e = launch_own_blocks(A, p.own, s);
    if (e != hipSuccess) return e;
    constexpr int kPer = kSplitRows * (D / 4) / kThreads;
    const long long segments = (long long)A.a.T * A.G / kSplitRows + A.a.n_seq;
    return launch_in_pieces(segments * A.c.h_kv * kPer, kThreads, [&](long long first, unsigned n) {
        if (p.few) hipLaunchKernelGGL((gather_kernel<D, kSplitRows>), dim3(n), dim3(kThreads), 0, s, A, (int)first);
        else hipLaunchKernelGGL((gather_kernel<D, kBlockRows>), dim3(n), dim3(kThreads), 0, s, A, (int)first);
    });
}

}  // namespace
}  // namespace ixg

extern "C" {

size_t ix_kv8_attn_shared_workspace_size(const ix_kv8* cache, int n_seq, int total_T, int max_q, int n_groups, int h_q) {
    using namespace ixg;
    Kv8 c;
    if (!make_kv8(cache, &c) || !attn_shape_ok(c, n_seq, total_T, max_q, h_q) || n_groups < 0 || n_groups > 65535) return 0;
    if (n_groups == 0) return ix_kv8_attn_workspace_size(cache, n_seq, total_T, max_q, h_q);
    return shared_plan(c.d, c.h_kv, h_q / c.h_kv, n_seq, total_T, max_q, n_groups, nullptr).bytes;
}

hipError_t ix_kv8_attn_shared(const ix_kv8* cache, int n_seq, int total_T, int max_q, const int32_t* cu_seqlens, const int32_t* kv_len,
                              const int32_t* table, int width, int n_groups, const int32_t* groups, const int32_t* shared_len,
                              const ix_rows* q, int h_q, float scale, const ix_rows* gate, uint16_t* o, void* workspace,
                              size_t workspace_bytes, hipStream_t s) {
    using namespace ixg;
    if (n_groups == 0)
        return ix_kv8_attn(cache, n_seq, total_T, max_q, cu_seqlens, kv_len, table, width, q, h_q, scale, 0, 0, gate, o, workspace,
                           workspace_bytes, s);
    AttnArgs A{};
    if (!make_attn(cache, n_seq, total_T, max_q, cu_seqlens, kv_len, table, width, h_q, scale, &A)) return hipErrorInvalidValue;
    if (n_groups < 0 || n_groups > 65535 || !groups || !shared_len || !ptr_aligned(groups, 4) || !ptr_aligned(shared_len, 4))
        return hipErrorInvalidValue;
    if (total_T == 0) return hipSuccess;                      // of tensors without elements, whose addresses may be 0
    const SharedPlan p = shared_plan(A.c.d, A.c.h_kv, A.G, n_seq, total_T, max_q, n_groups, s);
    if (!p.bytes || !make_operands(q, gate, o, workspace, workspace_bytes, p.bytes, &A)) return hipErrorInvalidValue;
    A.groups = groups;
    A.shared = shared_len;
    A.n_groups = n_groups;
    switch (A.c.d) {
        case 64: return launch_shared<64>(A, p, s);
        case 128: return launch_shared<128>(A, p, s);
        default: return launch_shared<256>(A, p, s);
    }
}

}  // extern "C"
