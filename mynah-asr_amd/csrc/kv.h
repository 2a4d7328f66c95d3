// kv.h — what the paged-cache kernels (kv_append.hip, kv_attention.hip, kv_prompt.hip)
// share: the tables of a call, and which keys a row sees. Plain integer arithmetic,
// for the host (workspace sizes) and the device.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "launch.h"

#define KV_HD __host__ __device__ __forceinline__

enum { KV_F32 = 0, KV_F16 = 1, KV_BF16 = 2 };   // cache elements

// The pool and the tables of one call (mynah_asr_hip_kv_cache, _kv_batch).
struct KvTables {
    void *k, *v;
    const int *row_start, *len, *pages;
    int n_pages, page, Hk;        // page: slots of one
    int nseq, rows, max_pages;
};

// One sequence: its rows r0 .. r0 + n - 1, and L keys, the rows' own among
// them. Whatever the tables hold, 0 <= r0, r0 + n <= rows and 0 <= L <= 2^30.
struct KvSeq {
    int r0, n, L;
};
__device__ __forceinline__ KvSeq kv_seq(const KvTables &t, int b) {
    // (both within the rows before they are subtracted: 2^31 - 1 and -2^31 are 1 apart in 32 bits)
    const int r0 = min(max(t.row_start[b], 0), t.rows), r1 = min(max(t.row_start[b + 1], r0), t.rows);
    return {r0, r1 - r0, min(max(t.len[b], 0), 1 << 30)};
}

// Row of the pool (head_dim elements each) that holds key j of sequence b for
// head h; KV_NONE where the table names no page of the pool. j is in [0,
// max_pages * page). The pool's rows are fewer than 2^32 - 1 (checked on the host).
constexpr uint32_t KV_NONE = 0xffffffffu;
__device__ __forceinline__ uint32_t kv_slot(const KvTables &t, int b, int j, int h) {
    const int lp = j / t.page;
    const int pg = t.pages[(size_t)b * t.max_pages + lp];
    return (unsigned)pg < (unsigned)t.n_pages ? ((uint32_t)pg * t.Hk + h) * t.page + (j - lp * t.page) : KV_NONE;
}

// The keys that rows between two positions see, as a list of aligned blocks of
// KB keys: the ns blocks that the first keys lie in, then blocks first .. of
// the window. (One run of blocks from 0 where the two meet.)
struct KvSpan {
    int ns, first, cnt;
    KV_HD int block(int e) const { return e < ns ? e : first + e - ns; }
};
// lo: the first row's window start; hi: the last key that the last row sees (-1: none)
template <int KB>
KV_HD KvSpan kv_span(int lo, int hi, int sinks) {
    const int nb = hi < 0 ? 0 : hi / KB + 1;
    int first = lo / KB, ns = ((sinks < lo ? sinks : lo) + KB - 1) / KB;
    if (first <= ns) first = ns = 0;
    if (ns > nb) ns = nb;
    return {ns, first, ns + (nb > first ? nb - first : 0)};
}

// What a tile of a sequence's rows sees. Rows are (token, query head of the K/V
// head): row r is head r % G of token r / G, tile rt holds RT of them.
struct KvTile {
    KvSeq s;
    int live;                 // its rows; <= 0: none, and the rest is not set
    int lo0, hi0, lo1, hi1;   // the first and the last row's window start and last key
    KvSpan sp;
};
__device__ __forceinline__ int kv_last(const KvTables &t, const KvAttend &a, const KvSeq &s, int tok) {
    const int64_t cap = (int64_t)t.max_pages * t.page;
    const int top = (int)min((int64_t)min(s.L, a.max_len), cap) - 1;
    return a.causal ? min(s.L - s.n + tok, top) : top;
}
__device__ __forceinline__ int kv_first(const KvAttend &a, const KvSeq &s, int tok) {
    return a.window ? max(s.L - s.n + tok - a.window + 1, 0) : 0;
}
// a sequence's rows that are computed
__device__ __forceinline__ int kv_rows(const KvAttend &a, const KvSeq &s) { return min(s.n, a.max_new) * a.G; }
template <int RT, int KB>
__device__ __forceinline__ KvTile kv_tile(const KvTables &t, const KvAttend &a, int b, int rt) {
    KvTile T;
    T.s = kv_seq(t, b);
    T.live = min(kv_rows(a, T.s) - rt * RT, RT);
    if (T.live <= 0) return T;
    const int i0 = rt * RT / a.G, i1 = (rt * RT + T.live - 1) / a.G;
    T.lo0 = kv_first(a, T.s, i0);
    T.lo1 = kv_first(a, T.s, i1);
    T.hi0 = kv_last(t, a, T.s, i0);
    T.hi1 = kv_last(t, a, T.s, i1);
    T.sp = kv_span<KB>(T.lo0, T.hi1, a.sinks);
    return T;
}
