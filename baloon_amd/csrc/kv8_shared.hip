// kv8_shared.hip -- attention over the paged 8-bit cache of a batch whose sequences have their first tokens in common.
//
// A row's softmax over all its tokens is put together of that over the shared ones and that over its own (kv8_attn.h, Joined):
// with partial results (m, l, o), p taken relative to 2^m, o = sum_i o_i 2^(m_i - m) / sum_i l_i 2^(m_i - m). So the rows of all of
// a group's sequences go over the shared tokens together (shared_kernel), those of each over its own (split_kernel and
// block_kernel of kv8_attn.hip), and gather_kernel puts the partial results together: three launches for single tokens.
#include "kv8_attn.h"

namespace ixg {
namespace {

constexpr int kThreads = 256, kWaves = kThreads / kWave;
constexpr int kGrain = 64;            // shared tokens are taken in whole 64s; what is left over is each sequence's own

// A group's rows, and the tokens that are taken together.
struct Group {
    int s0, rows, kv;
};
__device__ __forceinline__ int group_first(const AttnArgs& A, int g) { return min(max(A.groups[g], 0), A.a.n_seq); }
__device__ __forceinline__ Group group_at(const AttnArgs& A, int g) {
    Group out{0, 0, 0};
    if (g >= A.n_groups) return out;
    const int first = group_first(A, g), last = group_first(A, g + 1), n = A.shared[g];
    out.s0 = A.a.start(first);
    const int tokens = A.a.start(last) - out.s0;
    if (tokens > 0 && last - first > 1 && (long long)tokens * A.G <= 1 << 30) {
        out.rows = tokens * A.G;
        out.kv = (int)min((long long)max(n, 0), (long long)A.a.width << A.c.page_log) / kGrain * kGrain;
    }
    if (out.kv == 0) out.rows = 0;
    return out;
}

// The blocks of kRows rows of all groups and heads are taken in parts of about as many tiles each, so that there are at most
// `rounds` items for each workgroup: group g has parts_of(kv) for each of its blocks, and item
// ((blocks and parts of the groups before it) + block * parts + part) * h_kv + head.
template <int kRows, int kTok>
struct Cuts {
    int chunk;                // tiles
    static __device__ __forceinline__ int blocks(const Group& g) { return (g.rows + kRows - 1) / kRows; }
    __device__ __forceinline__ int parts(const Group& g) const { return g.rows ? (g.kv / kTok + chunk - 1) / chunk : 0; }
};
constexpr int kLeastChunk = kWaves;   // a tile for each wave
template <int kRows, int kTok>
__device__ __forceinline__ Cuts<kRows, kTok> cuts_of(const AttnArgs& A, int n_wg, int lane) {
    typedef Cuts<kRows, kTok> C;
    long long tiles = 0, blocks = 0;
    for (int g0 = 0; g0 < A.n_groups; g0 += kWave) {
        const Group g = group_at(A, g0 + lane);
        tiles += (long long)C::blocks(g) * (g.kv / kTok);
        blocks += C::blocks(g);
    }
    tiles = lane_of(wave_scan_int(tiles), kWave - 1) * A.c.h_kv;
    blocks = lane_of(wave_scan_int(blocks), kWave - 1) * A.c.h_kv;
    long long room = (blocks / n_wg + 1) * n_wg - blocks;     // items that can be more than one a block
    if (room < n_wg / 4) room += n_wg;
    C out;
    out.chunk = (int)min(max((tiles + room - 1) / room, (long long)kLeastChunk), 0x7fffffffll);
    return out;
}

// What the other launches ask of a sequence's group. One workgroup of shared_kernel's launch does nothing else.
template <int kRows, int kTok>
__device__ __forceinline__ void write_plan(const AttnArgs& A, const Cuts<kRows, kTok>& cuts, int tid) {
    const int lane = tid & (kWave - 1);
    SeqPlan* plan = A.seq;
    for (int b = tid; b < A.a.n_seq; b += kThreads) plan[b] = SeqPlan{0, 0, 0, 0};
    __syncthreads();
    if (tid >= kWave) return;
    int base = 0;
    for (int g0 = 0; g0 < A.n_groups; g0 += kWave) {
        const Group g = group_at(A, g0 + lane);
        const int items = cuts.blocks(g) * cuts.parts(g), incl = wave_scan_int(items);
        const int first = g.rows ? group_first(A, g0 + lane) : 0, last = g.rows ? group_first(A, g0 + lane + 1) : 0;
        unsigned long long todo = __ballot(g.rows > 0);
        while (todo) {                                        // all lanes for one group's sequences
            const int l = __builtin_ctzll(todo);
            todo &= todo - 1;
            const SeqPlan s{lane_of(g.kv, l), base + lane_of(incl - items, l), lane_of(g.s0, l), lane_of(cuts.parts(g), l)};
            for (int b = lane_of(first, l) + lane; b < lane_of(last, l); b += kWave) plan[b] = s;
        }
        base += lane_of(incl, kWave - 1);
    }
}

// Partial results of the items: sums [item][kRows][D], then (m, lse) [item][kRows][2].
template <int kRows, int D>
struct ItemParts {
    float *o, *ml;
    __device__ __forceinline__ explicit ItemParts(const AttnArgs& A) : o(A.item_part), ml(A.item_part + (size_t)A.n_items * kRows * D) {}
};

// Tokens of a tile: as many as leave registers for the next one's keys.
template <int D, int kG>
constexpr int kTokOf = D == 256 || (D == 128 && kG > 1) ? 32 : 64;

// A workgroup of 4 waves takes an item: kRows = 16 kG rows of one group and kv head over a part of the shared tokens, each wave
// its own tiles of kTok tokens for all the rows. Keys and values come from memory into the wave's registers, where they serve kG
// products; the products and the layout of P are those of split_kernel.
template <int D, int kG>
__global__ void __launch_bounds__(kThreads, 2) shared_kernel(AttnArgs A_) {
    constexpr int kC = D / 64, kM = D / 16, kPitch = D + 4, kTok = kTokOf<D, kG>, kS = kTok / 16, kRows = kG * kSplitRows;
    typedef typename std::conditional<kS == 4, uint4, uint2>::type Codes;     // 4 S values of a channel
    extern __shared__ float lds[];
    uint4* lo_q = reinterpret_cast<uint4*>(lds);              // [kG][kC][hi, lo][lane]
    uint32_t* lo_qm = reinterpret_cast<uint32_t*>(lo_q + kG * kC * 2 * kWave);              // [kG][waves][16]
    float* lo_o = lds;                                        // behind the tiles: [waves][16][kPitch]
    float* lo_ml = lds + kWaves * kSplitRows * kPitch;        // [waves][16][2]
    const int n_wg = gridDim.x - 1;
    Cuts<kRows, kTok> cuts;
    {
        const AttnArgs& A = args_again();
        cuts = cuts_of<kRows, kTok>(A, n_wg, threadIdx.x & (kWave - 1));
        if ((int)blockIdx.x == n_wg) {
            write_plan(A, cuts, threadIdx.x);
            return;
        }
    }
    for (int item = blockIdx.x;; item += n_wg) {
        int tid = threadIdx.x;
        asm volatile("" : "+v"(tid));                         // worked out again for each item: not kept over the main loop
        const int lane = tid & (kWave - 1), w = __builtin_amdgcn_readfirstlane(tid / kWave);
        const int n = lane & 15, g = lane >> 4, mine = 4 * kS * g, keys = 4 * kS * (n >> 2);
        const AttnArgs& A = args_again();
        const int h_kv = A.c.h_kv, page_log = A.c.page_log, n_pages = A.c.n_pages;
        // its group, block and part
        const int e = item % h_kv;
        int left = item / h_kv;
        int gi = -1, rb = 0, part = 0, n_parts = 1;
        Group gr{};
        for (int g0 = 0; g0 < A.n_groups; g0 += kWave) {
            const Group x = group_at(A, g0 + lane);
            const int p = cuts.parts(x), count = cuts.blocks(x) * p, incl = wave_scan_int(count);
            const unsigned long long hit = __ballot(incl > left);
            if (hit) {
                const int l = __builtin_amdgcn_readfirstlane(__builtin_ctzll(hit));
                gi = g0 + l;
                n_parts = lane_of(p, l);
                const int in = (int)(left - lane_of(incl - count, l));
                rb = in / n_parts;
                part = in - rb * n_parts;
                gr = Group{lane_of(x.s0, l), lane_of(x.rows, l), lane_of(x.kv, l)};
                break;
            }
            left -= lane_of(incl, kWave - 1);
        }
        if (gi < 0) return;
        const int all = gr.kv / kTok, t0 = (int)((long long)all * part / n_parts), t1 = (int)((long long)all * (part + 1) / n_parts);
        const int r0 = rb * kRows, n_rows = gr.rows - r0;
        const int32_t* tab = A.a.table + (size_t)group_first(A, gi) * A.a.width;
        const int8_t *kb = A.c.k + ((size_t)e << page_log) * D, *vb = A.c.v + ((size_t)e << page_log) * D;
        const float *ksb = A.c.k_scale + e, *vsb = A.c.v_scale + e;
        int step = 16 << page_log;                            // of 16 channels
        asm volatile("" : "+v"(ksb), "+v"(vsb), "+v"(kb), "+v"(vb), "+v"(step));           // not in scalar registers, which are few
        const uint32_t page_bytes = (uint32_t)(h_kv << page_log) * D;
        const auto page_of = [&](int t, int off) {
            const int id = tab[(min(t, t1 - 1) * kTok + off) >> page_log];        // t0 < t1: a group with blocks has tiles
            return (unsigned)id < (unsigned)n_pages ? id : -1;
        };
        const auto slot_of = [&](int t, int off) { return (min(t, t1 - 1) * kTok + off) & ((1 << page_log) - 1); };
        // Loads of a tile behind the last are the last's again, and not used.
        uint4 kr[kS][kC];
        Codes vr[kM];
        const auto load_k = [&](int t, int page) {
            const int8_t* p = kb + (size_t)max(page, 0) * page_bytes + (slot_of(t, keys) + (n & 3)) * D + 16 * g;
#pragma unroll
            for (int i = 0; i < kS; ++i)
#pragma unroll
                for (int c = 0; c < kC; ++c) kr[i][c] = *reinterpret_cast<const uint4*>(p + 4 * i * D + 64 * c);
        };
        const auto load_v = [&](int t, int page) {
            const int8_t* p = vb + (size_t)max(page, 0) * page_bytes + (n << page_log) + slot_of(t, mine);
#pragma unroll
            for (int m = 0; m < kM; ++m, p += step) vr[m] = *reinterpret_cast<const Codes*>(p);
        };
        int t = t0 + w;
        int pk = page_of(t, keys), pv = page_of(t, mine);
        float ks = 0.0f, vs = 0.0f;
        const auto load_scales = [&] {
            ks = ksb[(size_t)max(pv, 0) * h_kv];
            vs = vsb[(size_t)max(pv, 0) * h_kv];
        };
        // q: wave c takes channels 64 c + 16 g .. + 15 of every row (row n its lanes'), as two int8 of 16 bits
        uint4 raw[kG][2] = {};
        if (w < kC) {
#pragma unroll
            for (int x = 0; x < kG; ++x) {
                const int rc = min(r0 + x * kSplitRows + n, gr.rows - 1), qi = rc / A.G;
                const uint16_t* qp = A.q + (long long)(gr.s0 + qi) * A.q_stride + (size_t)(e * A.G + rc - qi * A.G) * D + 64 * w + 16 * g;
                raw[x][0] = load_row8(qp);
                raw[x][1] = load_row8(qp + 8);
            }
#pragma unroll
            for (int x = 0; x < kG; ++x) {
                u16x2 mb = max_abs_bits(max_abs_bits(u16x2{0, 0}, raw[x][0]), raw[x][1]);
                uint32_t mu = max((uint32_t)mb[0], (uint32_t)mb[1]);
                mu = max(mu, (uint32_t)__shfl_xor((int)mu, 16, kWave));
                mu = max(mu, (uint32_t)__shfl_xor((int)mu, 32, kWave));
                if (g == 0) lo_qm[(x * kWaves + w) * kSplitRows + n] = mu;
            }
        }
        load_k(t, pk);
        load_scales();
        lds_barrier();
        float qc[kG];
#pragma unroll
        for (int x = 0; x < kG; ++x) {
            uint32_t mu = lo_qm[x * kWaves * kSplitRows + n];
#pragma unroll
            for (int c = 1; c < kC; ++c) mu = max(mu, lo_qm[(x * kWaves + c) * kSplitRows + n]);
            const float qm = __uint_as_float(mu << 16);       // a row that is not finite gets scores that are none
            qc[x] = qm * (1.0f / 32639.0f) * A.scale2;
            if (w < kC) {
                split_q(raw[x][0], raw[x][1], qm > 1e-33f ? 32639.0f / qm : 0.0f);
                lo_q[((x * kC + w) * 2) * kWave + lane] = raw[x][0];
                lo_q[((x * kC + w) * 2 + 1) * kWave + lane] = raw[x][1];
            }
        }
        lds_barrier();

        v4f acc[kG][kM];
        float mref[kG];
        LaneSum sum[kG];
#pragma unroll
        for (int x = 0; x < kG; ++x) {
            mref[x] = -__builtin_inff();
#pragma unroll
            for (int m = 0; m < kM; ++m) acc[x][m] = v4f{0, 0, 0, 0};
        }
        for (; t < t1; t += kWaves) {
            asm volatile("" ::: "memory");                    // q is read from LDS again: there are no registers to keep it
            const float lv = log2_scale(vs);
            float p[kG][4 * kS], most[kG], top[kG];
#pragma unroll
            for (int x = 0; x < kG; ++x) {
                const uint4* lq = lo_q + 2 * kC * kWave * x + lane;
                const float cs = qc[x] * ks;
#pragma unroll
                for (int i = 0; i < kS; ++i) {
                    i32x4 h = {0, 0, 0, 0}, lw = {0, 0, 0, 0};
#pragma unroll
                    for (int c = 0; c < kC; ++c) {
                        const i32x4 k = __builtin_bit_cast(i32x4, kr[i][c]);
                        h = __builtin_amdgcn_mfma_i32_16x16x64_i8(k, __builtin_bit_cast(i32x4, lq[2 * c * kWave]), h, 0, 0, 0);
                        lw = __builtin_amdgcn_mfma_i32_16x16x64_i8(k, __builtin_bit_cast(i32x4, lq[(2 * c + 1) * kWave]), lw, 0, 0, 0);
                    }
#pragma unroll
                    for (int y = 0; y < 4; ++y) p[x][4 * i + y] = fmaf((float)((h[y] << 8) + lw[y]), cs, lv);
                }
                if (kG > 1) __builtin_amdgcn_sched_barrier(0);                            // one block's q at a time
            }
            const bool lost = pv < 0;
            __builtin_amdgcn_sched_barrier(0);
            load_v(t, pv);
            pk = page_of(t + kWaves, keys);
            pv = page_of(t + kWaves, mine);
            __builtin_amdgcn_sched_barrier(0);
            if (__ballot(lost)) {
                asm volatile("");                             // a branch: hardly ever
#pragma unroll
                for (int x = 0; x < kG; ++x)
#pragma unroll
                    for (int y = 0; y < 4 * kS; ++y) p[x][y] = lost ? -__builtin_inff() : p[x][y];
            }
            bool over = false;
#pragma unroll
            for (int x = 0; x < kG; ++x) {
                most[x] = p[x][0];
#pragma unroll
                for (int y = 1; y < 4 * kS; ++y) most[x] = fmaxf(most[x], p[x][y]);
                top[x] = pair_max32(pair_max16(most[x]));
                over = over || top[x] > mref[x] + kLag;
            }
            if (__ballot(over)) {
                asm volatile("");                             // a branch: at the first tiles, then seldom
#pragma unroll
                for (int x = 0; x < kG; ++x) {
                    const float now = fmaxf(mref[x], top[x]);
                    const float f = now == -__builtin_inff() ? 1.0f : __builtin_amdgcn_exp2f(mref[x] - now);
                    mref[x] = now;
#pragma unroll
                    for (int m = 0; m < kM; ++m) acc[x][m] *= f;
                }
            }
            float ref[kG], counts[kG];
            bool usual = true;
#pragma unroll
            for (int x = 0; x < kG; ++x) {
                ref[x] = mref[x] == -__builtin_inff() ? 0.0f : mref[x] - kLift;
                usual = sum[x].usual(most[x] - ref[x], ref[x], lv, &counts[x]) && usual;
            }
            if (__ballot(!usual)) {
                asm volatile("");                             // a branch: at a lane's first tokens, then hardly ever
#pragma unroll
                for (int x = 0; x < kG; ++x) counts[x] = sum[x].factor(p[x], ref[x], most[x] - ref[x], ref[x], lv);
            }
            f16x8 pf[kG][kS / 2];
#pragma unroll
            for (int x = 0; x < kG; ++x) {
                float of_tile = 0.0f;
#pragma unroll
                for (int y = 0; y < 4 * kS; ++y) {
                    const float v = __builtin_amdgcn_exp2f(p[x][y] - ref[x]);
                    of_tile += v;                             // before its rounding: a small page's p' loses bits by it
                    pf[x][y / 8][y & 7] = (_Float16)v;
                }
                sum[x].l = fmaf(of_tile, counts[x], sum[x].l);
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int m = 0; m < kM; ++m) {
                const f16x8 v = halves8(vr[m].x, vr[m].y);
#pragma unroll
                for (int x = 0; x < kG; ++x) acc[x][m] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, pf[x][0], acc[x][m], 0, 0, 0);
                if constexpr (kS == 4) {
                    const f16x8 u = halves8(vr[m].z, vr[m].w);
#pragma unroll
                    for (int x = 0; x < kG; ++x) acc[x][m] = __builtin_amdgcn_mfma_f32_16x16x32_f16(u, pf[x][1], acc[x][m], 0, 0, 0);
                }
                if (m % 4 == 3) __builtin_amdgcn_sched_barrier(0);
                if (m == kM / 2 - 1) {                        // half of the values' registers are free for the next keys
                    load_k(t + kWaves, pk);
                    load_scales();
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
        }

        // the four waves' parts together, 16 rows at a time
        const ItemParts<kRows, D> parts(args_again());
        lds_barrier();                                        // q has been read
#pragma unroll
        for (int x = 0; x < kG; ++x) {
            const float m = mref[x] == -__builtin_inff() ? kNone : mref[x] - kLift, lse = sum[x].log2_row(m);
            if (g == 0) {
                lo_ml[(w * kSplitRows + n) * 2] = m;
                lo_ml[(w * kSplitRows + n) * 2 + 1] = lse;
            }
#pragma unroll
            for (int y = 0; y < kM; ++y) *reinterpret_cast<v4f*>(lo_o + (w * kSplitRows + n) * kPitch + 16 * y + 4 * g) = acc[x][y];
            lds_barrier();
            for (int i = tid; i < kSplitRows * D / 4; i += kThreads) {
                const int row = i / (D / 4), d = i % (D / 4) * 4, r = x * kSplitRows + row;
                if (r >= n_rows) break;
                Joined to;
#pragma unroll
                for (int k = 0; k < kWaves; ++k) to.meet_m(lo_ml[(k * kSplitRows + row) * 2]);
#pragma unroll
                for (int k = 0; k < kWaves; ++k) to.meet_sum(lo_ml[(k * kSplitRows + row) * 2], lo_ml[(k * kSplitRows + row) * 2 + 1]);
#pragma unroll
                for (int k = 0; k < kWaves; ++k)
                    to.add(lo_ml[(k * kSplitRows + row) * 2], lo_ml[(k * kSplitRows + row) * 2 + 1],
                           *reinterpret_cast<const v4f*>(lo_o + (k * kSplitRows + row) * kPitch + d));
                *reinterpret_cast<v4f*>(parts.o + ((size_t)item * kRows + r) * D + d) = to.o;
                if (d == 0) *reinterpret_cast<float2*>(parts.ml + ((size_t)item * kRows + r) * 2) = make_float2(to.m, to.log2_sum());
            }
            lds_barrier();                                    // lo_o and lo_ml are free again, and lo_q and lo_qm
        }
    }
}

// Puts each row's partial results together and writes it: a workgroup takes up to 256 outputs (in fours) of a segment of 16 rows
// of a sequence and head, numbered as split_kernel's are but for gaps: those of sequence b are from start G / 16 + b on.
template <int D, int kRows>
__global__ void __launch_bounds__(kThreads) gather_kernel(AttnArgs A, int small, int n_own, int first) {
    constexpr int kPer = kSplitRows * (D / 4) / kThreads;     // workgroups of a segment
    const int tid = threadIdx.x, lane = tid & (kWave - 1);
    const int all = first + (int)blockIdx.x, piece = all % kPer, e = all / kPer % A.c.h_kv, j = all / kPer / A.c.h_kv;
    const auto key = [&](int b) { return (int)((long long)A.a.start(b) * A.G / kSplitRows) + b; };
    const int b = wave_search(A.a.n_seq, j, lane, key);
    const int s0 = A.a.start(b), rows = max(A.a.start(b + 1) - s0, 0) * A.G, r0 = (j - key(b)) * kSplitRows;
    if (r0 < 0 || r0 >= rows) return;                         // r0 < 0: before the first sequence's rows
    const int row = (piece * kThreads + tid) / (D / 4), d = tid % (D / 4) * 4, r = r0 + row;
    if (r >= rows) return;
    const int qi = r / A.G, t = s0 + qi, h = e * A.G + r - qi * A.G;
    const uint2 z = load_gate(A, t, h, d);
    const SeqPlan plan = A.seq[b];
    OwnCut cut{-1, 0, 0, 0};
    if (rows <= small) cut = A.cuts[((size_t)s0 * A.G + r0) * A.c.h_kv + e];
    Joined sum;
    if (cut.first < 0) {
        const size_t at = (size_t)t * A.h_q + h;
        sum.more(A.row_ml[2 * at], A.row_ml[2 * at + 1], *reinterpret_cast<const v4f*>(A.row_o + at * D + d));
    } else {
        const float* ml = A.part + (size_t)2 * n_own * kSplitRows * D;       // split_kernel's parts
#pragma unroll 4
        for (int k = cut.first; k <= cut.last; ++k) {
            const size_t at = (size_t)(k == cut.first ? cut.slot : 2 * k) * kSplitRows + row;
            sum.more(ml[2 * at], ml[2 * at + 1], *reinterpret_cast<const v4f*>(A.part + at * D + d));
        }
    }
    if (plan.parts > 0) {
        const ItemParts<kRows, D> parts(A);
        const int of_group = (t - plan.s0) * A.G + r - qi * A.G, rb = of_group / kRows;
        const size_t item = ((size_t)plan.block + (size_t)rb * plan.parts) * A.c.h_kv + e, step = (size_t)A.c.h_kv * kRows;
        size_t at = item * kRows + (of_group - rb * kRows);
#pragma unroll 8
        for (int k = 0; k < plan.parts; ++k, at += step)
            sum.more(parts.ml[2 * at], parts.ml[2 * at + 1], *reinterpret_cast<const v4f*>(parts.o + at * D + d));
    }
    store_out(A, t, h, d, outputs(sum.o, sum.log2_sum()), z);
}

// The workspace: what the sequences' own tokens need, partial results of rows, the plan, where segments' parts are, and the items'.
struct SharedPlan {
    Plan own;
    int rows, n_wg;           // 16s of rows of a block, and workgroups
    long long items, segments;
    size_t row_o, row_ml, seq, cuts, parts, bytes;
};
SharedPlan shared_plan(int d, int h_kv, int G, int T, int max_q, int n_groups, hipStream_t s) {
    SharedPlan p;
    p.own = attn_plan(d, h_kv, G, T, max_q, s);
    const long long mean = (long long)T * G / n_groups;
    p.rows = mean <= kSplitRows ? 1 : d == 256 ? 2 : 4;
    p.n_wg = p.own.n_wg;
    const auto up = [](size_t n) { return (n + 255) / 256 * 256; };
    const size_t rows = (size_t)T * h_kv * G;
    // blocks, of which a group has at most one that is not full, and those that more parts make (cuts_of)
    const long long blocks = (rows / (16 * p.rows) + (size_t)n_groups * h_kv);
    p.items = blocks + 2ll * p.n_wg;
    p.segments = ((long long)T * G / kSplitRows + 65535) * h_kv;
    p.row_o = attn_bytes(d, p.own);
    p.row_ml = p.row_o + up(rows * d * sizeof(float));
    p.seq = p.row_ml + up(rows * 2 * sizeof(float));
    p.cuts = p.seq + 65536 * sizeof(SeqPlan);
    p.parts = p.cuts + up(rows * sizeof(OwnCut));
    // of the largest items, whatever a smaller batch takes
    p.bytes = p.parts + (rows + 64 * ((size_t)n_groups * h_kv + 2 * p.n_wg)) * (d + 2) * sizeof(float);
    // workgroups and items are numbered in 31 bits; a batch beyond that has more outputs than the GPU has memory
    if (p.items > 0x7fffffff || p.segments * (kSplitRows * (d / 4) / kThreads) > 0x7fffffff) p.bytes = 0;
    return p;
}

template <int D, int kG>
hipError_t launch_shared(AttnArgs& A, const SharedPlan& p, hipStream_t s) {
    constexpr unsigned lds_q = kG * (D / 64 * 2 * kWave * sizeof(uint4) + kWaves * kSplitRows * sizeof(float));
    constexpr unsigned lds_o = kWaves * kSplitRows * (D + 4 + 2) * sizeof(float), lds = lds_q > lds_o ? lds_q : lds_o;
    static OncePerDevice once;
    const hipError_t ready = allow_lds(once, &shared_kernel<D, kG>, lds, s);
    if (ready != hipSuccess) return ready;
    char* ws = reinterpret_cast<char*>(A.part);
    A.n_items = (int)p.items;
    A.item_part = reinterpret_cast<float*>(ws + p.parts);
    A.seq = reinterpret_cast<SeqPlan*>(ws + p.seq);
    A.row_o = reinterpret_cast<float*>(ws + p.row_o);
    A.row_ml = reinterpret_cast<float*>(ws + p.row_ml);
    A.cuts = reinterpret_cast<OwnCut*>(ws + p.cuts);
    hipLaunchKernelGGL((shared_kernel<D, kG>), dim3((unsigned)p.n_wg + 1), dim3(kThreads), lds, s, A);
    hipError_t e = hipGetLastError();
    if (e == hipSuccess) e = launch_own(A, p.own, s);
    if (e != hipSuccess) return e;
    constexpr int kPer = kSplitRows * (D / 4) / kThreads;
    const long long segments = (long long)A.a.T * A.G / kSplitRows + A.a.n_seq;
    return launch_in_pieces(segments * A.c.h_kv * kPer, kThreads, [&](long long first, unsigned n) {
        hipLaunchKernelGGL((gather_kernel<D, kG * kSplitRows>), dim3(n), dim3(kThreads), 0, s, A, A.small, p.own.n_wg, (int)first);
    });
}
template <int D>
hipError_t launch_shared(AttnArgs& A, const SharedPlan& p, hipStream_t s) {
    return p.rows == 1 ? launch_shared<D, 1>(A, p, s) : launch_shared<D, D == 256 ? 2 : 4>(A, p, s);
}

}  // namespace
}  // namespace ixg

extern "C" {

size_t ix_kv8_attn_shared_workspace_size(const ix_kv8* cache, int n_seq, int total_T, int max_q, int n_groups, int h_q) {
    using namespace ixg;
    Kv8 c;
    if (!make_kv8(cache, &c) || !attn_shape_ok(c, n_seq, total_T, max_q, h_q) || n_groups < 0 || n_groups > 65535) return 0;
    if (n_groups == 0) return ix_kv8_attn_workspace_size(cache, n_seq, total_T, max_q, h_q);
    return shared_plan(c.d, c.h_kv, h_q / c.h_kv, total_T, max_q, n_groups, nullptr).bytes;
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
    const SharedPlan p = shared_plan(A.c.d, A.c.h_kv, A.G, total_T, max_q, n_groups, s);
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
