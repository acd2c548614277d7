// kv8.h -- the paged key/value cache in 8 bits (ix_kv8, include/ix_gdn.h): its checks on the host and the
// lookups its kernels share.
#pragma once
#include "gdn_common.h"

namespace ixg {

struct Kv8 {
    int8_t *k, *v;
    float *k_scale, *v_scale;
    int n_pages, page, page_log, h_kv, d;
};

// A batch: packed rows of new tokens and the sequences' pages.
struct Batch {
    const int32_t *cu, *kv_len, *table;
    int n_seq, T, width;
    __device__ __forceinline__ int start(int b) const { return min(max(cu[b], 0), T); }
    // Page id of page p of sequence b, or -1 where there is none.
    __device__ __forceinline__ int page_at(int b, int p, int n_pages) const {
        const int id = p < width ? table[(size_t)b * width + p] : -1;
        return (unsigned)id < (unsigned)n_pages ? id : -1;
    }
};

inline bool ptr_aligned(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

inline bool make_kv8(const ix_kv8* c, Kv8* out) {
    if (!c || c->n_pages <= 0 || c->h_kv <= 0 || c->h_kv > 1024) return false;
    if (c->page != 16 && c->page != 32 && c->page != 64 && c->page != 128) return false;
    if (c->d != 64 && c->d != 128 && c->d != 256) return false;
    if (!c->k || !c->v || !c->k_scale || !c->v_scale || !ptr_aligned(c->k, 16) || !ptr_aligned(c->v, 16) ||
        !ptr_aligned(c->k_scale, 4) || !ptr_aligned(c->v_scale, 4))
        return false;
    *out = Kv8{c->k, c->v, c->k_scale, c->v_scale, c->n_pages, c->page, __builtin_ctz((unsigned)c->page), c->h_kv, c->d};
    return true;
}

inline bool make_batch(int n_seq, int T, const int32_t* cu, const int32_t* kv_len, const int32_t* table, int width, Batch* out) {
    if (n_seq <= 0 || n_seq > 65535 || T < 0 || width <= 0 || !cu || !kv_len || !table) return false;
    if (!ptr_aligned(cu, 4) || !ptr_aligned(kv_len, 4) || !ptr_aligned(table, 4)) return false;
    *out = Batch{cu, kv_len, table, n_seq, T, width};
    return true;
}

inline bool rows_ok(const ix_rows* r, long long least) {
    return r && r->p && ptr_aligned(r->p, 2) && r->stride >= least;
}

// 8 values of a row, bf16, at any 2-byte address (the target reads and writes words unaligned).
__device__ __forceinline__ uint4 load_row8(const uint16_t* p) {
    uint4 x;
    __builtin_memcpy(&x, p, sizeof(x));
    return x;
}

// The last b in [0, n) with key(b) <= j, or 0 where there is none, for a key that does not fall: each step the wave's
// lanes try 64 places (one load's latency for 64 sequences, two for 4,096). The same in every lane.
template <class Key>
__device__ __forceinline__ int wave_search(int n, int j, int lane, Key key) {
    int lo = 0;
    while (n > 1) {
        const int step = (n + kWave - 1) / kWave, at = lane * step;
        const bool below = at < n && (lane == 0 || key(lo + at) <= j);
        const int last = __popcll(__ballot(below)) - 1;
        lo += last * step;
        n = min(step, n - last * step);
    }
    return __builtin_amdgcn_readfirstlane(lo);
}

}  // namespace ixg
