// kv8_shared.hip -- attention over the paged 8-bit cache of a batch whose sequences have their first tokens in common.
//
// A row's softmax over all its tokens is put together of that over the shared ones and that over its own (kv8_attn.h, Joined):
// with partial results (m, l, o), p taken relative to 2^m, o = sum_i o_i 2^(m_i - m) / sum_i l_i 2^(m_i - m). So the rows of all of
// a group's sequences go over the shared tokens together, those of each over its own, and gather_kernel puts the partial results
// together. few_kernel takes 16 rows a workgroup: each sequence's own tokens, and the shared ones of groups of few rows, all of
// these in one launch; block_kernel (kv8_attn.hip) takes 128: the shared tokens of groups of many rows, and prompts.
#include "kv8_attn.h"
#include "shared_list.h"

namespace ixg {
namespace {

constexpr int kThreads = 256, kWaves = kThreads / kWave;
template <int D>
constexpr int kTokOf = D == 256 ? 32 : 64;
constexpr int few_per_cu(int d) { return d == 256 ? 2 : d == 128 ? 3 : 4; }      // few_kernel's workgroups, by its registers

constexpr int kGrain = 64;            // shared tokens are taken in whole 64s; what is left over is each sequence's own,
constexpr int kFarthest = 1 << 30;    // and so are those from here on: where rows of a group are taken to stand, with room for as many of them

// A group's rows, and the tokens that are taken together.
struct Group {
    int s0, rows, kv;
    int alone;                // blocks of 16 rows of its sequences each for itself, about
};
__device__ __forceinline__ int group_first(const AttnArgs& A, int g) { return min(max(A.groups[g], 0), A.a.n_seq); }
__device__ __forceinline__ Group group_at(const AttnArgs& A, int g) {
    Group out{};
    if (g >= A.n_groups) return out;
    const int first = group_first(A, g), last = group_first(A, g + 1), n = A.shared[g];
    out.s0 = A.a.start(first);
    const int tokens = A.a.start(last) - out.s0;
    if (tokens > 0 && last - first > 1 && (long long)tokens * A.G <= kFarthest) {
        out.rows = tokens * A.G;
        out.alone = (last - first) * (((unsigned)out.rows / (unsigned)(last - first) + kSplitRows - 1) / kSplitRows);
        out.kv = (int)min((long long)min(max(n, 0), kFarthest), (long long)A.a.width << A.c.page_log) / kGrain * kGrain;
    }
    if (out.kv == 0) out.rows = 0;
    return out;
}

// Whether few_kernel takes a group's tokens together: where that is fewer tiles, with 8 more for each block more that it begins.
// Together and not, us: 37 sequences of 16 rows behind 2,049 tokens 38 and 35, 102 behind 208 56 and 48, 89 of 24 behind 75 28 and 22.
template <int D>
__device__ __forceinline__ bool few_shares(const Group& g) {
    const float tiles = (float)(g.kv / kTokOf<D>);
    return (float)g.alone * tiles > (float)((g.rows + kSplitRows - 1) / kSplitRows) * (tiles + 8.0f);
}
// few: those that are not worth it share nothing.
template <int D>
__device__ __forceinline__ Group settled(Group g, bool few) {
    if (few && !few_shares<D>(g)) g.rows = g.kv = 0;
    return g;
}
// The groups in the lanes of a wave, if there are up to 64.
struct Groups {
    Group g;
    int first, last;
    bool few;
};
__device__ __forceinline__ Groups groups_in_lanes(const AttnArgs& A, int lane) {
    Groups out{};
    if (A.n_groups > kWave || lane >= A.n_groups) return out;
    out.g = group_at(A, lane);
    out.first = group_first(A, lane);
    out.last = group_first(A, lane + 1);
    return out;
}

// Many rows: the blocks of 128 rows of all groups and heads are taken in parts of about as many tiles each: group g has parts(g)
// for each of its blocks, item ((blocks and parts of the groups before it) + block * parts + part) * h_kv + head.
struct Cuts {
    int chunk;                // tiles
    static __device__ __forceinline__ int blocks(const Group& g) { return (g.rows + kBlockRows - 1) / kBlockRows; }
    __device__ __forceinline__ int parts(const Group& g) const { return g.rows ? (g.kv / kBlockTok + chunk - 1) / chunk : 0; }
};
// The items are at most A.n_shared. Up to 64 groups lane p - 1 knows the time of the longest group's tiles in p parts, beyond
// that the room for items is filled.
template <int D>
__device__ __forceinline__ Cuts cuts_of(const AttnArgs& A, const Groups& groups, int n_wg, int lane) {
    Cuts out;
    long long tiles = 0, blocks = 0;
    int most = 0;
    Group g{};
    for (int g0 = 0; g0 < A.n_groups; g0 += kWave) {
        g = A.n_groups <= kWave ? groups.g : group_at(A, g0 + lane);
        tiles += (long long)Cuts::blocks(g) * (g.kv / kBlockTok);
        blocks += Cuts::blocks(g);
        most = max(most, g.kv / kBlockTok);
    }
    tiles = lane_of(wave_scan_int(tiles), kWave - 1) * A.c.h_kv;
    blocks = lane_of(wave_scan_int(blocks), kWave - 1) * A.c.h_kv;
    most = wave_max_int(most);
    const int room = A.n_shared - (int)blocks;                // parts beyond one a block
    if (A.n_groups > kWave || room < n_wg / 8) {
        out.chunk = room < n_wg / 8 ? max(most, 1) : (int)min(max((tiles + room - 1) / room, (long long)kLeastPart), 0x7fffffffll);
        return out;
    }
    const int chunk = max((most + lane) / (lane + 1), kLeastPart), t = g.kv / kBlockTok;
    const float inv = 1.0f / (float)chunk;
    int items = 0;                                            // at most 64 a block, of which there are at most A.n_shared
    for (int x = 0; x < A.n_groups; ++x) {
        const int tx = lane_of(t, x), full = (int)((float)tx * inv);      // or one less or more: at most 64
        items += lane_of(Cuts::blocks(g), x) * (full + (tx > full * chunk));
    }
    items *= A.c.h_kv;
    const float cost = items <= A.n_shared ? (float)((items + n_wg - 1) / n_wg) * ((float)chunk + kPartCost<D>) : __builtin_inff();
    const int best = -wave_max_int(-__float_as_int(cost));    // numbers >= 0 are in the order of their bits
    out.chunk = lane_of(chunk, __builtin_amdgcn_readfirstlane(__builtin_ctzll(__ballot(__float_as_int(cost) == best))));
    return out;
}

// The first own token of sequence b, a lane's own.
template <int D>
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
    return b >= group_first(A, lo) && b < group_first(A, lo + 1) ? settled<D>(group_at(A, lo), groups.few).kv : 0;
}

// What few_kernel takes: the groups, where block_kernel does not, and behind them the sequences of few rows.
struct Unit {
    int s0, rows;             // rows s0 G .. of a kv head, in blocks of 16; 0: nothing to do
    int t0, nt;               // its tiles (one at least)
    int first, kv;            // position of row 0 (of a group far behind its tokens), and tokens
};
template <int D>
__device__ __forceinline__ Unit unit_at(const AttnArgs& A, const Groups& groups, int n_groups, int u) {
    constexpr int kTok = kTokOf<D>;
    Unit out{};
    if (u < n_groups) {
        const Group g = A.n_groups <= kWave ? groups.g : settled<D>(group_at(A, u), groups.few);       // the lane's own: these units are the first 64
        out = Unit{g.s0, g.rows, 0, g.kv / kTok, kFarthest, g.kv};
    } else if (u - n_groups < A.a.n_seq) {
        const int b = u - n_groups, s0 = A.a.start(b), q = max(A.a.start(b + 1) - s0, 0), kv = max(A.a.kv_len[b], 0);
        const int held = (int)min((long long)kv, (long long)A.a.width << A.c.page_log);
        const int t0 = first_own<D>(A, groups, b) / kTok;
        out = Unit{s0, (long long)q * A.G <= A.small ? q * A.G : 0, t0, max(held / kTok + (held % kTok != 0) - t0, 1), kv - q, held};
    }
    return out;
}
__device__ __forceinline__ int blocks_of(const Unit& u) { return (u.rows + kSplitRows - 1) / kSplitRows; }

// A unit's blocks are taken in parts of up to `chunk` tiles: as few as leave at most `rounds` items for each workgroup. Item
// ((blocks and parts of the units before it) + block * parts + part) * h_kv + head. A piece of work is never two units', however
// short: a workgroup's way to its first tile is longer than several of them (64 sequences of up to 1,000 own tokens behind 8,190
// shared ones took split_kernel, whose shares are cut at one length, 16 us; drafts of 37 sequences of up to 500 took it 25).
struct FewCuts {
    int chunk, units, n_groups;           // groups among the units
    __device__ __forceinline__ int parts(const Unit& u) const { return (u.nt + chunk - 1) / chunk; }
};
// The items of `segments` blocks (below 2^29): at most this.
__host__ __device__ inline int few_items(int segments, int n_wg) {
    const int rounds = (int)((unsigned)segments / (unsigned)n_wg) + 1;
    return (rounds * n_wg - segments < n_wg / 4 ? rounds + 1 : rounds) * n_wg;
}
// Where groups have up to kFewRows rows a kv head in the mean, they are few_kernel's without a question (but see below), else where
// all of them have up to kFewTiles tiles of 16 rows: block_kernel takes a tile in half the time, but has 14 us before its first and for its partial results, of
// which 3 remain where it finds nothing to do. us there and here: 8 sequences of 16 heads over 2 of 256 behind 1,000 tokens (64 rows)
// 30 and 16, 16 of them 32 and 18; 64 behind 1,024, 4,096 and 8,190 (2,000, 8,200 and 16,400 tiles) 40, 44, 49 and 28, 41, 56; 128 of 20
// over 4 of 128 behind 1,024, 2,048 and 4,096 (2,600, 5,100 and 10,200) 53, 54, 62 and 42, 45, 61.
//
// The mean says little where one group has most of the rows (of a captured call's groups many can be empty). So the device chooses
// also where one group of all rows over a whole table would have over twice kFewTiles: 2 us where block_kernel then has nothing
// to do (24 groups of 4 sequences over a table that wide 56 and 58). One group beside 63 empty ones with few_kernel alone and with
// the choice, us: 64 sequences of 16 heads over 2 of 256 behind 16,384 tokens (34,800 such tiles) 92 and 59, behind 8,192 (18,400, where there
// is none) 56, 48 as the only group; 128 behind 4,096 and 16,384 (20,500, 69,600) 88, 280 and 61, 86; 200 of 32 over 8 of 128
// behind 16,384 (105,600) 199 and 122.
constexpr int kFewRows = 64, kFewTiles = 10000;
// The first units, worked out once and kept in LDS, and the sums of all waves.
constexpr int kKept = 512;
struct Kept {
    int unit[6][kKept];
    float tiles[kWaves];
    int segments[kWaves];
    FewCuts cuts;                         // and what the main loop has no registers for
    int item, rows;
    int2 found[kWaves];                   // where a wave found its last item: the 64 units, and the items before them (for one head)
};
// Whether the groups are few_kernel's, which settles what they share: where it has few tiles, or no more than as blocks of 128, which take
// the time of kFewRows however few of them are rows. Of few tiles those that it would not share count less: they are no items of
// their own. us as blocks of 128 and so: 37 sequences of 16 rows, 8 heads of 128, behind 2,049 and 4,096 tokens (9,500 and 19,000
// tiles) 41, 48 and 36, 53; 64 of 16 and of 32 rows, 2 heads of 256, behind 2,048 (8,200 and 16,400) 49, 56 and 42, 75.
template <int D>
__device__ __forceinline__ bool few_take(const AttnArgs& A, const Groups& groups, int lane) {
    if (!A.many) return true;
    float tiles = 0.0f, more = 0.0f;                          // more: than as blocks of 128
    for (int g0 = 0; g0 < A.n_groups; g0 += kWave) {
        const Group g = A.n_groups <= kWave ? groups.g : group_at(A, g0 + lane);
        const bool shares = few_shares<D>(g);
        const int blocks = shares ? (g.rows + kSplitRows - 1) / kSplitRows : g.alone, t = g.kv / kTokOf<D>;
        tiles += (shares ? 1.0f : D == 256 ? 0.8f : 0.6f) * (float)blocks * (float)t;
        more += (float)(blocks - (g.rows + kBlockRows - 1) / kBlockRows * (kFewRows / kSplitRows)) * (float)t;
    }
    return __builtin_amdgcn_readfirstlane((int)(wave_sum(tiles) * (float)A.c.h_kv <= (float)kFewTiles || wave_sum(more) <= 0.0f));
}
template <int D>
__device__ __forceinline__ FewCuts few_cuts(const AttnArgs& A, Groups& groups, Kept* kept, int n_wg, int tid) {
    FewCuts out;
    const int lane = tid & (kWave - 1);
    groups.few = few_take<D>(A, groups, lane);
    groups.g = settled<D>(groups.g, groups.few);
    out.n_groups = groups.few ? A.n_groups : 0;
    out.units = out.n_groups + A.a.n_seq;
    float tiles = 0.0f;
    int segments = 0;
    for (int u0 = tid - lane; u0 < out.units; u0 += kThreads) {
        const Unit u = unit_at<D>(A, groups, out.n_groups, u0 + lane);
        if (u0 + lane < kKept) {
            const int x[6] = {u.s0, u.rows, u.t0, u.nt, u.first, u.kv};
#pragma unroll
            for (int i = 0; i < 6; ++i) kept->unit[i][u0 + lane] = x[i];
        }
        tiles += (float)blocks_of(u) * (float)u.nt;
        segments += blocks_of(u);
    }
    tiles = wave_sum(tiles);
    segments = wave_scan_int(segments);
    if (lane == kWave - 1) {
        kept->tiles[tid / kWave] = tiles;
        kept->segments[tid / kWave] = segments;
    }
    __syncthreads();
    tiles = 0.0f, segments = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        tiles += kept->tiles[w];
        segments += kept->segments[w];
    }
    // chunk * room >= tiles: at most `room` items more than blocks. The sums' roundings are under 2^-16 of them.
    segments *= A.c.h_kv;
    const float room = (float)(few_items(segments, n_wg) - segments), chunk = tiles * (float)A.c.h_kv * (1.0f + 0x1p-14f) / room;
    out.chunk = __builtin_amdgcn_readfirstlane(max((int)fminf(ceilf(chunk), 0x1p30f), kWaves));
    return out;
}
template <int D>
__device__ __forceinline__ Unit kept_unit(const AttnArgs& A, const Kept* kept, int u, const FewCuts& cuts, int lane) {
    if (cuts.units > kKept && (u | (kWave - 1)) >= kKept) {   // the same for the wave
        Groups groups = groups_in_lanes(A, lane);
        groups.few = cuts.n_groups > 0;
        groups.g = settled<D>(groups.g, groups.few);
        return unit_at<D>(A, groups, cuts.n_groups, u);
    }
    Unit out{};
    if (u < cuts.units)
        out = Unit{kept->unit[0][u], kept->unit[1][u], kept->unit[2][u], kept->unit[3][u], kept->unit[4][u], kept->unit[5][u]};
    return out;
}

// An item: rows r0 .. r0 + n_rows - 1 of a unit and head e, over tiles t0 .. t1 - 1.
struct Piece {
    int table_row, e, s0, rows, r0, first, kv, t0, t1;
};
template <int D>
__device__ __forceinline__ bool piece_at(const AttnArgs& A, Kept* kept, const FewCuts& cuts, int item, int w, int lane, Piece* out) {
    const int2 from = kept->found[w];                         // a workgroup's items ascend
    int left = item / A.c.h_kv - taken(from.y);
    for (int u0 = taken(from.x); u0 < cuts.units; u0 += kWave) {
        const Unit u = kept_unit<D>(A, kept, u0 + lane, cuts, lane);
        const int p = cuts.parts(u), count = blocks_of(u) * p, incl = wave_scan_int(count);
        const unsigned long long hit = __ballot(incl > left);
        if (hit) {
            if (lane == 0) kept->found[w] = make_int2(u0, item / A.c.h_kv - left);
            const int l = __builtin_amdgcn_readfirstlane(__builtin_ctzll(hit));
            const int parts = lane_of(p, l), in = left - lane_of(incl - count, l), rb = in / parts, part = in - rb * parts;
            const int t0 = lane_of(u.t0, l), nt = lane_of(u.nt, l), each = nt / parts, more = nt - each * parts;
            const int row = u0 + l < cuts.n_groups ? group_first(A, u0 + l) : u0 + l - cuts.n_groups;
            *out = Piece{row, item % A.c.h_kv, lane_of(u.s0, l), lane_of(u.rows, l), rb * kSplitRows, lane_of(u.first, l), lane_of(u.kv, l),
                         t0 + part * each + min(part, more), t0 + (part + 1) * each + min(part + 1, more)};
            return true;
        }
        left -= lane_of(incl, kWave - 1);
    }
    return false;
}

// What block_kernel and gather_kernel ask of a sequence, by a wave that does nothing else. A field is written once: the sequences that
// share something are those whose own tokens begin behind the first.
template <int D>
__device__ __forceinline__ void write_plan(const AttnArgs& A, const Groups& groups, const FewCuts& cuts, int lane) {
    const bool few = cuts.n_groups == A.n_groups;
    const Cuts blocks = few ? Cuts{1} : cuts_of<D>(A, groups, A.slots, lane);
    int base = 0;
    for (int g0 = 0; g0 < A.n_groups; g0 += kWave) {
        const Group g = A.n_groups <= kWave ? groups.g : settled<D>(group_at(A, g0 + lane), groups.few);
        const int first = g.rows ? group_first(A, g0 + lane) : 0, last = g.rows ? group_first(A, g0 + lane + 1) : 0;
        const Unit u{g.s0, g.rows, 0, g.kv / kTokOf<D>, 0, 0};
        const int parts = few ? cuts.parts(u) : blocks.parts(g), items = (few ? blocks_of(u) : Cuts::blocks(g)) * parts;
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
                A.seq[b].shared_rows = few ? kSplitRows : kBlockRows;
            }
            if (few) continue;
            const int rows = lane_of(g.rows, l), kv = lane_of(g.kv, l), row = lane_of(first, l);
            const int each = kv / kBlockTok / n, more = kv / kBlockTok - each * n;         // tiles of a part, and parts of one more
            const int listed = items_listed(item, lane_of(items, l), A.n_shared / A.c.h_kv);
            for (int i = lane; i < listed; i += kWave) {
                const int rb = i / n, part = i - rb * n;
                A.shared_items[item + i] = SharedItem{s0, rows, rb * kBlockRows, row, part * each + min(part, more),
                                                      (part + 1) * each + min(part + 1, more), kv, 0};
            }
        }
        base += lane_of(before + items, kWave - 1);
    }
    for (int i = (few ? 0 : list_end(base, A.n_shared / A.c.h_kv)) + lane; A.many && i <= A.n_shared / A.c.h_kv; i += kWave)
        A.shared_items[i].row = -1;
    base = few ? base : 0;
    for (int u0 = cuts.n_groups; u0 < cuts.units; u0 += kWave) {
        const Unit u = unit_at<D>(A, groups, cuts.n_groups, u0 + lane);
        const int parts = cuts.parts(u), items = blocks_of(u) * parts, before = wave_scan_int(items) - items, b = u0 - cuts.n_groups + lane;
        if (b < A.a.n_seq) {
            A.seq[b].from = u.t0 * kTokOf<D>;
            A.seq[b].item = base + before;
            A.seq[b].parts = parts;
            if (u.t0 == 0) A.seq[b].shared_parts = 0;
        }
        base += lane_of(before + items, kWave - 1);
    }
}

// An item is 16 rows of a unit over a part of its tiles. A wave takes a tile of kTok tokens at a time by itself, all in registers,
// with the next one's loads under way; products and the layout of P are those of split_kernel. Every workgroup works out the cuts by
// itself (2.5 us, where a kernel ahead of this one costs a launch); the way to an item's first tile is a chain of three reads, which
// lies under the last item's join. Long own parts are bound by HBM: 96 sequences in groups of 4, 32 heads over 8 of 128, 226 MB
// with the page tables in 49 us, 4.6 TB/s; shorter ones by that chain (64 of up to 1,000 own tokens 17 us, 10 where there is next to nothing to do).
template <int D>
__global__ void __launch_bounds__(kThreads, few_per_cu(D)) few_kernel(AttnArgs A_) {
    constexpr int kC = D / 64, kM = D / 16, kPitch = D + 4, kTok = kTokOf<D>, kS = kTok / 16;
    typedef typename std::conditional<kS == 4, uint4, uint2>::type Codes;     // 4 S values of a channel
    extern __shared__ float lds[];
    uint4* lo_q = reinterpret_cast<uint4*>(lds);              // [kC][hi, lo][lane]
    uint32_t* lo_qm = reinterpret_cast<uint32_t*>(lo_q + kC * 2 * kWave);     // [kC][16]
    float* lo_o = lds;                                        // behind the tiles: [waves][16][kPitch]
    float* lo_ml = lds + kWaves * kSplitRows * kPitch;        // [waves][16][2]
    Kept* kept = reinterpret_cast<Kept*>(lds + kWaves * kSplitRows * (kPitch + 2));
    const int n_wg = gridDim.x - 1;
    {
        // The argument's cache lines, asked for at once: else each is waited for where it is first used.
        const int* line = reinterpret_cast<const int*>(&args_again());
        static_assert(sizeof(AttnArgs) > 256 && sizeof(AttnArgs) <= 320);
        asm volatile("" ::"s"(line[0]), "s"(line[16]), "s"(line[32]), "s"(line[48]), "s"(line[64]));
        const AttnArgs& A = args_again();
        Groups groups = groups_in_lanes(A, threadIdx.x & (kWave - 1));
        const FewCuts cuts = few_cuts<D>(A, groups, kept, n_wg, threadIdx.x);
        if ((int)blockIdx.x == n_wg) {
            if (threadIdx.x < kWave) write_plan<D>(A, groups, cuts, threadIdx.x);
            return;
        }
        kept->cuts = cuts;                                    // by all waves the same
        if (threadIdx.x < kWaves) kept->found[threadIdx.x] = make_int2(0, 0);
        __syncthreads();
    }
    // The sums of an item, for rows n: of 2^(kLift - mref) p' v / vs, and of p; and what is left to do for it.
    v4f acc[kM];
    float mref;
    LaneSum sum;
    bool open = false;
    for (int item = blockIdx.x;; item += n_wg) {
        // The next item's first loads are on their way while the last one's waves are joined.
        int tid = threadIdx.x;
        asm volatile("" : "+v"(tid));                         // worked out again for each item: not kept over the main loop
        const int lane = tid & (kWave - 1), w = __builtin_amdgcn_readfirstlane(tid / kWave);
        const int n = lane & 15, g = lane >> 4, mine = 4 * kS * g, keys = 4 * kS * (n >> 2);
        const AttnArgs& A = args_again();
        const int h_kv = A.c.h_kv, page_log = A.c.page_log, n_pages = A.c.n_pages;
        Piece it{};
        const bool any = item < A.n_items && piece_at<D>(A, kept, FewCuts{taken(kept->cuts.chunk), taken(kept->cuts.units), taken(kept->cuts.n_groups)}, item, w, lane, &it);
        if (!any && !open) return;
        const int e = it.e, r0 = it.r0, kv = it.kv, t1 = it.t1;
        int t = it.t0 + w;
        const int32_t* tab = A.a.table + (size_t)it.table_row * A.a.width;
        const int step = 16 << page_log;                      // of 16 channels
        const uint32_t page_bytes = (uint32_t)(h_kv << page_log) * D, head = (uint32_t)(e << page_log) * D;      // both below 2^31
        // What is loaded of a tile behind the last is the last's again, and not used.
        const auto page_of = [&](int t, int off) {
            const int j = min(t, t1 - 1) * kTok + off, id = j < kv ? tab[j >> page_log] : -1;
            return (unsigned)id < (unsigned)n_pages ? id : -1;
        };
        const auto slot_of = [&](int t, int off) { return (min(t, t1 - 1) * kTok + off) & ((1 << page_log) - 1); };
        uint4 kr[kS][kC];
        Codes vr[kM];
        const auto load_k = [&](int t, int page) {
            const int8_t* p = args_again().c.k + head + (size_t)max(page, 0) * page_bytes + (slot_of(t, keys) + (n & 3)) * D + 16 * g;
#pragma unroll
            for (int i = 0; i < kS; ++i)
#pragma unroll
                for (int c = 0; c < kC; ++c) kr[i][c] = *reinterpret_cast<const uint4*>(p + 4 * i * D + 64 * c);
        };
        const auto values_at = [&](int t, int page) {
            return args_again().c.v + head + (size_t)max(page, 0) * page_bytes + (n << page_log) + slot_of(t, mine);
        };
        int pv = -1, pk_next = -1, pv_next = -1;
        float ks = 0.0f, vs = 0.0f;
        const auto load_scales = [&](int page) {
            const size_t at = (size_t)max(page, 0) * h_kv + e;
            ks = args_again().c.k_scale[at];
            vs = args_again().c.v_scale[at];
        };
        // q: wave c takes channels 64 c + 16 g .. + 15 of every row (row n its lanes'), as two int8 of 16 bits
        uint4 raw[2] = {};
        if (any) pv = page_of(t, mine), pk_next = page_of(t + kWaves, keys), pv_next = page_of(t + kWaves, mine);
        if (any && w < kC) {
            const int rc = min(r0 + n, it.rows - 1), qi = rc / A.G;
            const uint16_t* qp = A.q + (long long)(it.s0 + qi) * A.q_stride + (size_t)(e * A.G + rc - qi * A.G) * D + 64 * w + 16 * g;
            raw[0] = load_row8(qp);
            raw[1] = load_row8(qp + 8);
        }
        if (any) {
            load_k(t, page_of(t, keys));
            const int8_t* p = values_at(t, pv);
#pragma unroll
            for (int m = 0; m < kM; ++m, p += step) vr[m] = *reinterpret_cast<const Codes*>(p);
            load_scales(pv);
        }
        if (open) {                                      // the four waves' parts of the last item together
            const ItemParts<kSplitRows, D> parts(args_again().item_part, args_again().n_items);
            const float m = mref == -__builtin_inff() ? kNone : mref - kLift, lse = sum.log2_row(m);
            const int x_item = taken(kept->item), x_rows = taken(kept->rows);
            lds_barrier();                                    // q has been read
            if (g == 0) {
                lo_ml[(w * kSplitRows + n) * 2] = m;
                lo_ml[(w * kSplitRows + n) * 2 + 1] = lse;
            }
#pragma unroll
            for (int y = 0; y < kM; ++y) *reinterpret_cast<v4f*>(lo_o + (w * kSplitRows + n) * kPitch + 16 * y + 4 * g) = acc[y];
            lds_barrier();
            for (int i = tid; i < kSplitRows * D / 4; i += kThreads) {
                const int row = i / (D / 4), d = i % (D / 4) * 4;
                if (row >= x_rows) break;
                Joined to;
#pragma unroll
                for (int k = 0; k < kWaves; ++k) to.meet_m(lo_ml[(k * kSplitRows + row) * 2]);
#pragma unroll
                for (int k = 0; k < kWaves; ++k) to.meet_sum(lo_ml[(k * kSplitRows + row) * 2], lo_ml[(k * kSplitRows + row) * 2 + 1]);
#pragma unroll
                for (int k = 0; k < kWaves; ++k)
                    to.add(lo_ml[(k * kSplitRows + row) * 2], lo_ml[(k * kSplitRows + row) * 2 + 1],
                           *reinterpret_cast<const v4f*>(lo_o + (k * kSplitRows + row) * kPitch + d));
                *reinterpret_cast<v4f*>(parts.o + ((size_t)x_item * kSplitRows + row) * D + d) = to.o;
                if (d == 0) *reinterpret_cast<float2*>(parts.ml + ((size_t)x_item * kSplitRows + row) * 2) = make_float2(to.m, to.log2_sum());
            }
            lds_barrier();                                    // the next item's q goes there
        }
        if (!any) return;
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

        mref = -__builtin_inff(), sum = LaneSum{};
        kept->item = item, kept->rows = it.rows - r0;         // by all waves the same, behind the last item's
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
            load_scales(pv_next);
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

        open = true;
    }
}

// Puts each row's partial results together and writes it, bound by reading them (34 MB of 64 sequences' 1,024 rows of 256 behind
// 8,190 shared tokens in 8.8 us; 4.4 of 96 rows in few parts): a wave takes 64 outputs (in fours) of a token or, kWays, a workgroup's four
// waves every fourth of their results each.
constexpr int kOutputs = kWave;
template <int D, bool kWays>
__global__ void __launch_bounds__(kThreads) gather_kernel(AttnArgs A, int first) {
    __shared__ v4f lo_o[kThreads];
    __shared__ float2 lo_ml[kThreads];
    const int tid = threadIdx.x, lane = tid & (kWave - 1), w = __builtin_amdgcn_readfirstlane(tid / kWave), h_kv = A.c.h_kv;
    const int per = (A.h_q * (D / 4) + kOutputs - 1) / kOutputs;         // waves of a token
    const long long all = ((long long)first + blockIdx.x) * (kWays ? 1 : kWaves) + (kWays ? 0 : w);
    if (all >= (long long)A.a.T * per) return;                // all threads with kWays, which alone have a barrier
    const int t = __builtin_amdgcn_readfirstlane(all >> 32 == 0 ? (int)((unsigned)all / (unsigned)per) : (int)(all / per));
    const int out = (int)(all - (long long)t * per) * kOutputs + lane;
    const int b = wave_search(A.a.n_seq, t, lane, [&](int i) { return A.a.start(i); });
    const int s0 = A.a.start(b), end = A.a.start(b + 1);
    if (t < s0 || t >= end || end - s0 > A.max_q) return;     // of no sequence, or of one that has no partial results
    const bool any = out < A.h_q * (D / 4);
    const int h = any ? out / (D / 4) : 0, d = out % (D / 4) * 4, e = h / A.G, in_token = h - e * A.G, rows = (end - s0) * A.G;
    const SeqPlan plan = A.seq[b];
    uint2 z = make_uint2(0, 0);
    if (!kWays || w == 0) z = load_gate(A, t, h, d);
    Joined sum;
    const int way = kWays ? w : 0, step = kWays ? kWaves : 1;
    const auto add = [&](const auto& parts, int room, int rows_of, int first, int n, int in, int from) {
        if (first < 0 || first > room / h_kv - n) return;     // only where sequences or groups overlap, which is not allowed
        size_t at = ((size_t)(first + from) * h_kv + e) * rows_of + in;
#pragma unroll 8
        for (int k = from; k < n; k += step, at += (size_t)step * h_kv * rows_of)
            sum.more(parts.ml[2 * at], parts.ml[2 * at + 1], *reinterpret_cast<const v4f*>(parts.o + at * D + d));
    };
    const ItemParts<kSplitRows, D> few(A.item_part, A.n_items);
    int own = 1;
    if (rows <= A.small) {
        const int r = (t - s0) * A.G + in_token, rb = r / kSplitRows;
        own = plan.parts;
        add(few, A.n_items, kSplitRows, plan.item + rb * own, own, r - rb * kSplitRows, way);
    } else if (way == 0) {
        const size_t at = (size_t)t * A.h_q + h;
        sum.more(A.row_ml[2 * at], A.row_ml[2 * at + 1], *reinterpret_cast<const v4f*>(A.row_o + at * D + d));
    }
    if (plan.shared_parts > 0) {
        const int r = (t - plan.s0) * A.G + in_token, n = plan.shared_rows, block = r / n, in = r - block * n;
        const int from = kWays ? (way - own) & (kWaves - 1) : 0;
        const int first = plan.shared_item + block * plan.shared_parts;
        if (n == kSplitRows) add(few, A.n_items, kSplitRows, first, plan.shared_parts, in, from);
        else add(ItemParts<kBlockRows, D>(A.shared_part, A.n_shared), A.n_shared, kBlockRows, first, plan.shared_parts, in, from);
    }
    if constexpr (kWays) {
        lo_o[tid] = sum.o;
        lo_ml[tid] = make_float2(sum.m, sum.log2_sum());
        __syncthreads();
        if (w > 0) return;
#pragma unroll
        for (int x = 1; x < kWaves; ++x) sum.more(lo_ml[tid + x * kWave].x, lo_ml[tid + x * kWave].y, lo_o[tid + x * kWave]);
    }
    if (any) store_out(A, t, h, d, outputs(sum.o, sum.log2_sum()), z);
}

// The workspace: what block_kernel needs over the sequences' own tokens, the plan, few_kernel's items, and, where block_kernel takes
// any, partial results of the rows and of its items over the shared tokens.
struct SharedPlan {
    Plan own;
    bool many;                // groups' rows may be block_kernel's
    int n_wg, few_wg;         // workgroups of block_kernel and of few_kernel that the chip holds
    long long n_items, n_shared;
    size_t seq, items, shared, shared_items, row_o, row_ml, bytes;
};
SharedPlan shared_plan(int d, int h_kv, int G, int n_seq, int T, int max_q, int n_groups, long long table_tokens, hipStream_t s) {
    SharedPlan p;
    p.own = attn_plan(d, h_kv, G, T, max_q, s);
    const long long rows = (long long)T * G, nonempty = std::min(n_seq, T);
    const double tiles = (double)((rows + kSplitRows - 1) / kSplitRows) * (double)(table_tokens / (d == 256 ? kTokOf<256> : kTokOf<128>)) * h_kv;
    p.many = rows > (long long)kFewRows * n_groups || (rows > kFewRows && tiles > 2.0 * kFewTiles);
    p.n_wg = d == 256 ? p.own.n_wg / 2 : p.own.n_wg;
    // a sequence or group has at most one block that is not full; a group with rows to share has two sequences or more, and a token;
    // the groups may be few_kernel's
    const long long with_rows = std::min({n_groups, n_seq / 2, T});
    const long long segments = (2 * (rows / kSplitRows) + nonempty + with_rows) * h_kv, blocks = (rows / kBlockRows + with_rows) * h_kv;
    p.few_wg = p.own.n_wg / 2 * few_per_cu(d);
    p.n_items = segments > 1 << 28 ? 0 : few_items((int)segments, p.few_wg - 1);
    p.n_shared = blocks < p.n_wg / 2 ? p.n_wg : (blocks + p.n_wg - 1) / p.n_wg * p.n_wg + p.n_wg;
    const auto up = [](size_t n) { return (n + 255) / 256 * 256; };
    const auto item_bytes = [&](long long n, int block) { return up((size_t)n * block * (d + 2) * sizeof(float)); };
    p.seq = attn_bytes(d, p.own);
    p.items = p.seq + up(n_seq * sizeof(SeqPlan));
    p.shared = p.items + item_bytes(p.n_items, kSplitRows);
    p.shared_items = p.shared + item_bytes(p.n_shared, kBlockRows);
    p.row_o = p.shared_items + up((p.n_shared / h_kv + 1) * sizeof(SharedItem));
    p.row_ml = p.row_o + (p.own.block ? up((size_t)rows * h_kv * d * sizeof(float)) : 0);
    p.bytes = p.row_ml + (p.own.block ? up((size_t)rows * h_kv * 2 * sizeof(float)) : 0);
    // workgroups and items are numbered in 31 bits; a batch beyond that has more outputs than the GPU has memory
    if (segments > 1 << 28 || rows * h_kv * d / 256 > 1 << 30) p.bytes = 0;
    return p;
}

template <int D>
hipError_t launch_shared(AttnArgs& A, const SharedPlan& p, hipStream_t s) {
    char* ws = reinterpret_cast<char*>(A.part);
    A.seq = reinterpret_cast<SeqPlan*>(ws + p.seq);
    A.item_part = reinterpret_cast<float*>(ws + p.items);
    A.shared_part = reinterpret_cast<float*>(ws + p.shared);
    A.shared_items = reinterpret_cast<SharedItem*>(ws + p.shared_items);
    A.row_o = reinterpret_cast<float*>(ws + p.row_o);
    A.row_ml = reinterpret_cast<float*>(ws + p.row_ml);
    A.n_items = (int)p.n_items;
    A.n_shared = (int)p.n_shared;
    A.many = p.many;
    A.max_q = p.own.max_q;
    A.slots = p.n_wg;
    A.small = attn_small(A, p.own);
    constexpr unsigned lds = kWaves * kSplitRows * (D + 4 + 2) * sizeof(float) + sizeof(Kept);
    static OncePerDevice once;
    hipError_t e = allow_lds(once, &few_kernel<D>, lds, s);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((few_kernel<D>), dim3((unsigned)p.few_wg), dim3(kThreads), lds, s, A);
    e = hipGetLastError();
    if (e == hipSuccess && p.many) e = launch_shared_blocks(A, p.n_wg, s);
    if (e == hipSuccess && p.own.block) e = launch_own_blocks(A, p.own, s);
    if (e != hipSuccess) return e;
    const auto gather = [&](auto ways) {
        const long long waves = (long long)A.a.T * ((A.h_q * (D / 4) + kOutputs - 1) / kOutputs);
        return launch_in_pieces(ways ? waves : (waves + kWaves - 1) / kWaves, kThreads, [&](long long first, unsigned n) {
            hipLaunchKernelGGL((gather_kernel<D, ways>), dim3(n), dim3(kThreads), 0, s, A, (int)first);
        });
    };
    // Four waves for each output where the chip holds as many at once: 64 tokens of 16 heads of 256 9.1 us against 11.3 with one;
    // 148 drafted ones of 32 of 128 8.8 against 6.9.
    const bool ways = (long long)A.a.T * A.h_q * D <= (long long)p.own.n_wg * 1024;
    return ways ? gather(std::true_type{}) : gather(std::false_type{});
}

}  // namespace
}  // namespace ixg

extern "C" {

size_t ix_kv8_attn_shared_workspace_size(const ix_kv8* cache, int n_seq, int total_T, int max_q, int n_groups, int h_q) {
    using namespace ixg;
    Kv8 c;
    if (!make_kv8(cache, &c) || !attn_shape_ok(c, n_seq, total_T, max_q, h_q) || n_groups < 0 || n_groups > 65535) return 0;
    if (n_groups == 0) return ix_kv8_attn_workspace_size(cache, n_seq, total_T, max_q, h_q);
    return shared_plan(c.d, c.h_kv, h_q / c.h_kv, n_seq, total_T, max_q, n_groups, 0, nullptr).bytes;      // whatever the tables
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
    const SharedPlan p = shared_plan(A.c.d, A.c.h_kv, A.G, n_seq, total_T, max_q, n_groups, (long long)width << A.c.page_log, s);
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
