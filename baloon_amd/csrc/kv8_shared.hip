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
template <int D>
constexpr int kTokOf = D == 256 ? 32 : 64;

// Few rows: an item is 16 of them over a part of the shared tokens. A wave takes a tile of kTok tokens at a time by itself, all in
// registers, with the next one's loads under way; products and the layout of P are those of split_kernel.
constexpr float kItemCost = 8.0f;     // tiles in the time of an item's start, its sums and their gathering
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
    Cuts<kSplitRows, kTok> cuts;
    {
        const AttnArgs& A = args_again();
        cuts = cuts_of<kSplitRows, kTok>(A, n_wg, kWaves, kItemCost, threadIdx.x & (kWave - 1));
        if ((int)blockIdx.x == n_wg) {
            write_plan(A, cuts, threadIdx.x, kThreads);
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
        Item<kSplitRows, kTok> it;
        if (!item_at(A, cuts, item, lane, &it)) return;
        const int t1 = it.t1, r0 = it.rb * kSplitRows, n_rows = it.g.rows - r0;
        const int32_t* tab = A.a.table + (size_t)group_first(A, it.group) * A.a.width;
        const int8_t *kb = A.c.k + ((size_t)it.e << page_log) * D, *vb = A.c.v + ((size_t)it.e << page_log) * D;
        const float *ksb = A.c.k_scale + it.e, *vsb = A.c.v_scale + it.e;
        int step = 16 << page_log;                            // of 16 channels
        asm volatile("" : "+v"(ksb), "+v"(vsb), "+v"(kb), "+v"(vb), "+v"(step));           // not in scalar registers, which are few
        const uint32_t page_bytes = (uint32_t)(h_kv << page_log) * D;
        // What is loaded of a tile behind the last is the last's again, and not used.
        const auto page_of = [&](int t, int off) {
            const int id = tab[(min(t, t1 - 1) * kTok + off) >> page_log];
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
        int t = it.t0 + w;
        int pv = page_of(t, mine), pk_next = page_of(t + kWaves, keys), pv_next = page_of(t + kWaves, mine);
        // q: wave c takes channels 64 c + 16 g .. + 15 of every row (row n its lanes'), as two int8 of 16 bits
        uint4 raw[2] = {};
        if (w < kC) {
            const int rc = min(r0 + n, it.g.rows - 1), qi = rc / A.G;
            const uint16_t* qp = A.q + (long long)(it.g.s0 + qi) * A.q_stride + (size_t)(it.e * A.G + rc - qi * A.G) * D + 64 * w + 16 * g;
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
            if (__ballot(lost)) {
                asm volatile("");                             // a branch: hardly ever
#pragma unroll
                for (int y = 0; y < 4 * kS; ++y) p[y] = lost ? -__builtin_inff() : p[y];
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
        const ItemParts<kSplitRows, D> parts(args_again());
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
    int rows, n_wg;           // rows of a block, and workgroups
    long long items;
    size_t row_o, row_ml, seq, cuts, parts, bytes;
};
// Groups of up to 32 rows a kv head in the mean are few_kernel's, others block_kernel's.
constexpr int kFewRows = 32;
SharedPlan shared_plan(int d, int h_kv, int G, int T, int max_q, int n_groups, hipStream_t s) {
    SharedPlan p;
    p.own = attn_plan(d, h_kv, G, T, max_q, s);
    const size_t rows = (size_t)T * h_kv * G;
    // a group has at most one block that is not full
    const auto items = [&](int block, int n_wg) {
        const long long blocks = rows / block + (size_t)n_groups * h_kv;
        return blocks < n_wg / 2 ? n_wg : (blocks + n_wg - 1) / n_wg * n_wg + n_wg;
    };
    p.rows = (long long)T * G <= (long long)kFewRows * n_groups ? kSplitRows : kBlockRows;
    p.n_wg = p.rows == kSplitRows || d != 256 ? p.own.n_wg : p.own.n_wg / 2;
    p.items = items(p.rows, p.n_wg);
    const auto up = [](size_t n) { return (n + 255) / 256 * 256; };
    p.row_o = attn_bytes(d, p.own);
    p.row_ml = p.row_o + up(rows * d * sizeof(float));
    p.seq = p.row_ml + up(rows * 2 * sizeof(float));
    p.cuts = p.seq + 65536 * sizeof(SeqPlan);
    p.parts = p.cuts + up(rows * sizeof(OwnCut));
    // of the largest items, whichever a smaller batch takes
    p.bytes = p.parts + (size_t)items(kBlockRows, p.own.n_wg) * kBlockRows * (d + 2) * sizeof(float);
    // workgroups and items are numbered in 31 bits; a batch beyond that has more outputs than the GPU has memory
    if (items(kSplitRows, p.own.n_wg) > 1 << 30 || ((long long)T * G / kSplitRows + 65535) * h_kv * (kSplitRows * (d / 4) / kThreads) > 0x7fffffff)
        p.bytes = 0;
    return p;
}

template <int D, int kRows>
hipError_t launch_shared(AttnArgs& A, const SharedPlan& p, hipStream_t s) {
    char* ws = reinterpret_cast<char*>(A.part);
    A.n_items = (int)p.items;
    A.item_part = reinterpret_cast<float*>(ws + p.parts);
    A.seq = reinterpret_cast<SeqPlan*>(ws + p.seq);
    A.row_o = reinterpret_cast<float*>(ws + p.row_o);
    A.row_ml = reinterpret_cast<float*>(ws + p.row_ml);
    A.cuts = reinterpret_cast<OwnCut*>(ws + p.cuts);
    hipError_t e;
    if constexpr (kRows == kBlockRows) {
        e = launch_shared_blocks(A, p.n_wg, s);
    } else {
        constexpr unsigned lds = kWaves * kSplitRows * (D + 4 + 2) * sizeof(float);
        static OncePerDevice once;
        e = allow_lds(once, &few_kernel<D>, lds, s);
        if (e == hipSuccess) {
            hipLaunchKernelGGL((few_kernel<D>), dim3((unsigned)p.n_wg), dim3(kThreads), lds, s, A);
            e = hipGetLastError();
        }
    }
    if (e == hipSuccess) e = launch_own(A, p.own, s);
    if (e != hipSuccess) return e;
    constexpr int kPer = kSplitRows * (D / 4) / kThreads;
    const long long segments = (long long)A.a.T * A.G / kSplitRows + A.a.n_seq;
    return launch_in_pieces(segments * A.c.h_kv * kPer, kThreads, [&](long long first, unsigned n) {
        hipLaunchKernelGGL((gather_kernel<D, kRows>), dim3(n), dim3(kThreads), 0, s, A, A.small, p.own.n_wg, (int)first);
    });
}
template <int D>
hipError_t launch_shared(AttnArgs& A, const SharedPlan& p, hipStream_t s) {
    return p.rows == kSplitRows ? launch_shared<D, kSplitRows>(A, p, s) : launch_shared<D, kBlockRows>(A, p, s);
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
