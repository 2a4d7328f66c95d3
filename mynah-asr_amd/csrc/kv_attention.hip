// kv_attention.hip — attention of new rows over a paged cache.
//
//   out = sum_j softmax_j(scale q . k_j) v_j over the keys j that a row sees
//
// with causal order, a sliding window and first keys that stay visible decided by
// position (kv.h). The G query heads that share a K/V head are rows of one
// product, as are a sequence's new rows: tile rows r = token * G + head, 16 NR a tile.
//
// One workgroup = four waves = one chunk of the keys that a sequence's rows see, for
// one K/V head. The keys are a list of blocks of 64 (kv_span); a wave takes every
// fourth of the chunk's. It reads K and V once, from memory to registers, and
// keeps a running maximum, sum and context of its own; the waves' are joined in
// LDS, the chunks' by k_kv_join (one chunk is written at once). The chunk's size
// depends on the number of blocks the rows see alone, so a row's bits do not
// depend on the other sequences of the call.
//
// What bounds it: memory. 48 requests of 500 to 9000 keys, 32 heads on 8 of 128, f16
// (636 MB): 130 us, 4.9 TB/s, 7 of them the join; one of 131072 keys, 64 heads on 8,
// bf16 (537 MB): 104 us, 5.2 TB/s. A large read takes 5.4 TB/s. One request of 200
// keys: 7.3 us, a chain of memory round trips. 32 keys a step at three waves a SIMD
// are faster than 64 at two (129 and 141 us) and 32 at four, which spill (157).
//
// Products: S^T = K Q^T and O^T = V^T P^T (lane l, c = l & 15, g = l >> 4: A row
// c, B column c, D rows 4g + e, column c). f32 caches: the f32 MFMA 16x16x4, slot g;
// 16-bit ones: the 16x16x32 MFMA of their type, slots 8g + j, on q and probabilities
// in terms (kv_terms.h). S^T leaves lane (c, g) with keys 4g + e of query row c, and
// the second product is free to take its keys in that order: probabilities never
// leave their lane. It is free in the order of features too, so a lane loads runs of
// 16 bytes of a value row, and pairs the rows' elements by byte permutes.
#include <hip/hip_runtime.h>
#include <math.h>

#include "kv.h"
#include "kv_terms.h"
#include "launch.h"
#include "product.h"

namespace {

constexpr int NW = 4, NTH = 64 * NW;
constexpr int KB = 64;      // keys of a block

// Blocks a wave takes in one chunk of a tile that sees `cnt`. Up to 512 keys are one
// chunk: the join would cost more than its second block. Long lists have longer chunks
// (fewer partial results to join).
KV_HD int wave_blocks(int cnt) { return cnt <= NW ? 1 : cnt <= 2 * NW ? 2 : cnt <= 256 ? 1 : cnt <= 1024 ? 2 : 4; }
KV_HD int chunk_blocks(int cnt) { return NW * wave_blocks(cnt); }
KV_HD int chunks_of(int cnt) { return cnt <= 0 ? 1 : (cnt + chunk_blocks(cnt) - 1) / chunk_blocks(cnt); }

// most chunks of a tile that sees up to n blocks
int most_chunks(int n) {
    int m = chunks_of(n);
    if (n > 256) m = m > chunks_of(256) ? m : chunks_of(256);
    if (n > 1024) m = m > chunks_of(1024) ? m : chunks_of(1024);
    return m;
}

struct StepArgs {
    KvTables t;
    KvAttend a;
    float *part;   // partial contexts [workgroup][R][DK], then their maxima and sums [workgroup][R][2]
    int nch, R;    // chunks of a sequence's keys (at most), rows of a partial result
};

__device__ __forceinline__ f4 mfma4(float a, float b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }
__device__ __forceinline__ float max_g(float x) {   // over the four lanes of a query row
    x = fmaxf(x, __shfl_xor(x, 16, 64));
    return fmaxf(x, __shfl_xor(x, 32, 64));
}
__device__ __forceinline__ float sum_g(float x) {
    x += __shfl_xor(x, 16, 64);
    return x + __shfl_xor(x, 32, 64);
}

// BYTES from p
template <int BYTES> __device__ __forceinline__ void load_run(const void *p, uint32_t (&x)[BYTES / 4]) {
    if constexpr (BYTES % 16 == 0) {
#pragma unroll
        for (int i = 0; i < BYTES / 16; i++) {
            const uint4 v = ((const uint4 *)p)[i];
            x[4 * i] = v.x, x[4 * i + 1] = v.y, x[4 * i + 2] = v.z, x[4 * i + 3] = v.w;
        }
    } else {
        const uint2 v = *(const uint2 *)p;
        x[0] = v.x, x[1] = v.y;
    }
}

// The two products of a wave on one kind of cache. Both take and give the f32
// scores s[tile of 16 keys], keys 4 g + e of query row c in lane (c, g). The query
// rows, which the workgroup's waves share, lie in LDS as fragments of 64 x 16 bytes;
// put_q has each wave form its part of them.
template <typename T, int DK> struct Wave {   // 16 bits
    using X = KvTerms<T>;
    typedef typename X::v8 v8;
    static constexpr int NB = 2;                   // key tiles at a time
    static constexpr int NU = DK / 32, VE = DK / 16, QF = NU * X::N;
    static constexpr float TOP = X::N == 2 ? 14.0f : 0.0f;   // probabilities reach 2^TOP
    float sc;
    __device__ __forceinline__ void put_q(const float *qp, float f, bool live, int g, int w, uint4 *ql) {
        float x[NU][8], mx = 0.0f;
#pragma unroll
        for (int u = 0; u < NU; u++) {
            *(f4 *)&x[u][0] = *(const f4 *)(qp + 32 * u + 8 * g);
            *(f4 *)&x[u][4] = *(const f4 *)(qp + 32 * u + 8 * g + 4);
#pragma unroll
            for (int j = 0; j < 8; j++) {
                x[u][j] = live ? x[u][j] * f : 0.0f;
                mx = fmaxf(mx, fabsf(x[u][j]));
            }
        }
        const int e = X::shift(max_g(mx));
        sc = ldexpf(1.0f, -e);
#pragma unroll
        for (int u = 0; u < NU; u++) {
            if (u % NW != w) continue;
#pragma unroll
            for (int j = 0; j < 8; j++) x[u][j] = ldexpf(x[u][j], e);
            v8 q[X::N];
            X::split(x[u], q);
#pragma unroll
            for (int i = 0; i < X::N; i++) ql[64 * (X::N * u + i)] = __builtin_bit_cast(uint4, q[i]);
        }
    }
    __device__ __forceinline__ void scores(const uint4 *ql, const uint32_t (&k)[NB][NU][4], f4 (&s)[NB]) const {
#pragma unroll
        for (int n = 0; n < NB; n++) s[n] = f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int u = 0; u < NU; u++)
#pragma unroll
            for (int i = 0; i < X::N; i++) {
                const v8 q = __builtin_bit_cast(v8, ql[64 * (X::N * u + i)]);
#pragma unroll
                for (int n = 0; n < NB; n++)
                    s[n] = X::mfma16(__builtin_bit_cast(v8, uint4{k[n][u][0], k[n][u][1], k[n][u][2], k[n][u][3]}), q, s[n]);
            }
#pragma unroll
        for (int n = 0; n < NB; n++) s[n] *= sc;
    }
    // o[i][e] += V^T P^T: feature VE (4 g + x) + e of the context in element x
    template <int NR>
    static __device__ __forceinline__ void context(const uint32_t (&v)[NB][4][VE / 2], const f4 (&p)[NR][NB],
                                                   f4 (&o)[NR][VE]) {
#pragma unroll
        for (int n = 0; n < NB; n += 2) {
            // slots 8 g + j: keys 4 g + j of tile n, then of tile n + 1
            v8 pt[NR][X::N];
#pragma unroll
            for (int i = 0; i < NR; i++) {
                const float pf[8] = {p[i][n][0],     p[i][n][1],     p[i][n][2],     p[i][n][3],
                                     p[i][n + 1][0], p[i][n + 1][1], p[i][n + 1][2], p[i][n + 1][3]};
                X::split(pf, pt[i]);
            }
#pragma unroll
            for (int e = 0; e < VE; e++) {
                uint32_t a[4];
#pragma unroll
                for (int y = 0; y < 4; y++) {
                    const int k = n + y / 2, r = 2 * (y & 1);
                    a[y] = __builtin_amdgcn_perm(v[k][r + 1][e / 2], v[k][r][e / 2], e & 1 ? 0x07060302u : 0x05040100u);
                }
                const v8 av = __builtin_bit_cast(v8, uint4{a[0], a[1], a[2], a[3]});
#pragma unroll
                for (int x = 0; x < X::N; x++)
#pragma unroll
                    for (int i = 0; i < NR; i++) o[i][e] = X::mfma16(av, pt[i][x], o[i][e]);
            }
        }
    }
    // the elements that are not finite, set to 0; whether there are any
    static __device__ __forceinline__ bool clean(uint32_t &x) {
        const bool l = kv_odd_lo<T>(x), h = kv_odd_hi<T>(x);
        x = (l ? 0u : x & 0xffffu) | (h ? 0u : x & 0xffff0000u);
        return l || h;
    }
};
template <int DK> struct Wave<float, DK> {
    static constexpr int NB = 1;
    static constexpr int NU = DK / 16, VE = DK / 16, QF = NU;
    static constexpr float TOP = 0.0f;
    __device__ __forceinline__ void put_q(const float *qp, float f, bool live, int g, int w, uint4 *ql) {
#pragma unroll
        for (int u = 0; u < NU; u++) {
            if (u % NW != w) continue;
            const f4 x = *(const f4 *)(qp + 16 * u + 4 * g);
            ql[64 * u] = __builtin_bit_cast(uint4, live ? x * f : f4{0.0f, 0.0f, 0.0f, 0.0f});
        }
    }
    __device__ __forceinline__ void scores(const uint4 *ql, const uint32_t (&k)[NB][NU][4], f4 (&s)[NB]) const {
#pragma unroll
        for (int n = 0; n < NB; n++) s[n] = f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int u = 0; u < NU; u++) {
            const f4 q = __builtin_bit_cast(f4, ql[64 * u]);
#pragma unroll
            for (int j = 0; j < 4; j++)
#pragma unroll
                for (int n = 0; n < NB; n++) s[n] = mfma4(__uint_as_float(k[n][u][j]), q[j], s[n]);
        }
    }
    template <int NR>
    static __device__ __forceinline__ void context(const uint32_t (&v)[NB][4][VE], const f4 (&p)[NR][NB],
                                                   f4 (&o)[NR][VE]) {
#pragma unroll
        for (int n = 0; n < NB; n++)
#pragma unroll
            for (int x = 0; x < 4; x++)
#pragma unroll
                for (int e = 0; e < VE; e++)
#pragma unroll
                    for (int i = 0; i < NR; i++) o[i][e] = mfma4(__uint_as_float(v[n][x][e]), p[i][n][x], o[i][e]);
    }
    static __device__ __forceinline__ bool clean(uint32_t &x) {
        const bool odd = !(fabsf(__uint_as_float(x)) < INFINITY);
        x = odd ? 0u : x;
        return odd;
    }
};

__device__ __attribute__((aligned(16))) const float kv_zeros[128] = {};

template <typename T, int DK, int NR>
__global__ __launch_bounds__(NTH, NR == 1 ? 3 : 2) void k_kv_step(const StepArgs A) {
    using W = Wave<T, DK>;
    constexpr int RT = 16 * NR;
    constexpr int EL = 16 / sizeof(T);       // features of a 16-byte load
    constexpr int NB = W::NB, NU = W::NU, VE = W::VE;
    constexpr int VB = VE * sizeof(T);       // bytes of a value row, per lane
    constexpr int OS = DK + 4;
    __shared__ uint32_t slots[NW][KB];
    __shared__ float mls[NW][RT][2];
    // q's fragments, then the waves' contexts
    __shared__ __attribute__((aligned(16))) float os[NW][RT][OS];
    static_assert(NR * W::QF * 1024 <= sizeof os, "q in LDS");
    uint4 *ql = (uint4 *)os + (threadIdx.x & 63);
    const KvTables &t = A.t;
    const KvAttend &a = A.a;
    const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, g = lane >> 4;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    int at = blockIdx.x;
    const int h = at % t.Hk;
    at /= t.Hk;
    const int ch = at % A.nch, b = at / A.nch;
    const KvTile tl = kv_tile<RT, KB>(A.t, A.a, b, 0);
    if (tl.live <= 0) return;
    const int nch = chunks_of(tl.sp.cnt), e0 = ch * chunk_blocks(tl.sp.cnt);
    if (ch >= nch) return;

    // This wave's blocks, in parts of NB tiles of 16 keys. The first part's loads are on
    // their way before q is looked at; the next part's keys are loaded once the scores
    // have let go of their registers, its values once the context has.
    const int e1 = min(e0 + chunk_blocks(tl.sp.cnt), tl.sp.cnt);
    const bool alike = tl.lo0 == tl.lo1 && tl.hi0 == tl.hi1;   // every row sees the same keys
    uint32_t kr[NB][NU][4], vr[NB][4][VB / 4];
    int j0 = 0;
    uint64_t some = 0, all = 0;   // of the block's keys, those that some row sees, and every row
    auto page_of = [&](int e) {   // (past the last block: the last one's again)
        const int j = min(tl.sp.block(min(e, e1 - 1)) * KB + lane, tl.hi1);
        return t.pages[(size_t)b * t.max_pages + j / t.page];
    };
    int pg = 0;                   // of block e's keys
    auto look = [&](int e) {      // where the block's keys lie
        j0 = tl.sp.block(e) * KB;
        const int jl = j0 + lane;
        const bool in = jl <= tl.hi1 && (unsigned)pg < (unsigned)t.n_pages;
        const bool seen = in && (jl >= tl.lo0 || jl < a.sinks);
        some = __ballot(seen);
        all = __ballot(in && jl <= tl.hi0 && (jl >= tl.lo1 || jl < a.sinks));
        wave_lds_order();   // the reads of the last block's slots
        slots[w][lane] = seen ? ((uint32_t)pg * t.Hk + h) * t.page + jl % t.page : KV_NONE;
        wave_lds_order();
        pg = page_of(e + NW);
    };
    auto part = [&](uint64_t m, int n0) { return (uint32_t)(m >> (16 * n0)) & (uint32_t)((1ull << (16 * NB)) - 1); };
    auto fetch_k = [&](int n0) {
#pragma unroll
        for (int n = 0; n < NB; n++) {
            const uint32_t at_k = slots[w][16 * (n0 + n) + c];
            const T *kp = (const T *)t.k + (size_t)(at_k == KV_NONE ? 0 : at_k) * DK + EL * g;
#pragma unroll
            for (int u = 0; u < NU; u++) load_run<16>(kp + 4 * EL * u, kr[n][u]);
        }
    };
    auto fetch_v = [&](int n0) {
#pragma unroll
        for (int n = 0; n < NB; n++)
#pragma unroll
            for (int x = 0; x < 4; x++) {
                const uint32_t at_v = slots[w][16 * (n0 + n) + 4 * g + x];
                // (a key that no row sees: its probability 0 times 0)
                const T *vp = at_v == KV_NONE ? (const T *)kv_zeros : (const T *)t.v + (size_t)at_v * DK;
                load_run<VB>(vp + VE * c, vr[n][x]);
            }
    };
    // the next part that a row sees keys of, from (e, n0) on; false: there is none
    auto seek = [&](int &e, int &n0) {
        for (;;) {
            if (n0 == 0) {
                if (e >= e1) return false;
                look(e);
            }
            if (part(some, n0)) return true;
            n0 += NB;
            if (n0 == KB / 16) n0 = 0, e += NW;
        }
    };
    int e = e0 + w, n0 = 0;
    if (e < e1) pg = page_of(e);
    bool more = seek(e, n0);
    if (more) {
        fetch_k(n0);
        fetch_v(n0);
    }

    // this lane's query rows (one of each sixteen), times scale and log2(e)
    int lo[NR], hi[NR];
    W wv[NR];
    float m[NR], l[NR];
    f4 o[NR][VE];
#pragma unroll
    for (int i = 0; i < NR; i++) {
        const int r = min(16 * i + c, tl.live - 1), tok = r / a.G;
        lo[i] = kv_first(a, tl.s, tok);
        hi[i] = kv_last(t, a, tl.s, tok);
        wv[i].put_q(a.q + (int64_t)(tl.s.r0 + tok) * a.ldq + (h * a.G + r % a.G) * DK, a.scale * 1.4426950408889634f,
                    16 * i + c < tl.live, g, w, ql + 64 * W::QF * i);
        m[i] = -INFINITY;
        l[i] = 0.0f;
#pragma unroll
        for (int x = 0; x < VE; x++) o[i][x] = f4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    __syncthreads();

    while (more) {
        f4 s[NR][NB];
#pragma unroll
        for (int i = 0; i < NR; i++) wv[i].scores(ql + 64 * W::QF * i, kr, s[i]);
        const uint32_t m_some = part(some, n0), m_all = part(all, n0);
        const int jp = j0 + 16 * n0;   // the part's first key
        n0 += NB;
        if (n0 == KB / 16) n0 = 0, e += NW;
        more = seek(e, n0);
        if (more) fetch_k(n0);
        bool odd = false;
        if (m_all != part(~0ull, 0)) {
            const uint32_t see = m_some >> (4 * g);
#pragma unroll
            for (int n = 0; n < NB; n++)
#pragma unroll
                for (int x = 0; x < 4; x++) {
                    const int j = jp + 16 * n + 4 * g + x;
                    const bool in = see >> (16 * n + x) & 1;
#pragma unroll
                    for (int i = 0; i < NR; i++)
                        s[i][n][x] = in && j <= hi[i] && (j >= lo[i] || j < a.sinks) ? s[i][n][x] : -INFINITY;
                }
            // A value that only some rows see meets the others' probability 0, which
            // hides it unless it is not finite: such an element counts as 0 in the
            // product and is added afterwards to the rows that see it.
            if (!alike) {
#pragma unroll
                for (int n = 0; n < NB; n++)
#pragma unroll
                    for (int x = 0; x < 4; x++)
#pragma unroll
                        for (int y = 0; y < VB / 4; y++) odd |= W::clean(vr[n][x][y]);
            }
        }
#pragma unroll
        for (int i = 0; i < NR; i++) {
            float mx = -INFINITY;
#pragma unroll
            for (int n = 0; n < NB; n++)
#pragma unroll
                for (int x = 0; x < 4; x++) mx = fmaxf(mx, s[i][n][x]);
            const float mn = fmaxf(m[i], max_g(mx)), mz = mn == -INFINITY ? 0.0f : mn;
            const float al = __builtin_amdgcn_exp2f(m[i] - mz);
            m[i] = mn;
            l[i] *= al;
#pragma unroll
            for (int n = 0; n < NB; n++)
#pragma unroll
                for (int x = 0; x < 4; x++) {
                    s[i][n][x] = __builtin_amdgcn_exp2f(s[i][n][x] - mz + W::TOP);
                    l[i] += s[i][n][x];
                }
#pragma unroll
            for (int x = 0; x < VE; x++) o[i][x] *= al;
        }
        W::template context<NR>(vr, s, o);
        if (__any(odd)) {
            for (int jj = 0; jj < 16 * NB; jj++) {
                const int j = jp + jj;
                if (!(m_some >> jj & 1)) continue;
                const T *vp = (const T *)t.v + (size_t)kv_slot(t, b, j, h) * DK;
#pragma unroll
                for (int i = 0; i < NR; i++) {
                    if (j > hi[i] || (j < lo[i] && j >= a.sinks)) continue;
#pragma unroll
                    for (int x = 0; x < 4; x++)
#pragma unroll
                        for (int y = 0; y < VE; y++) {
                            const float v = (float)vp[VE * (4 * g + x) + y];
                            if (!(fabsf(v) < INFINITY)) o[i][y][x] += v;
                        }
                }
            }
        }
        if (more) fetch_v(n0);
    }

    // join the waves
#pragma unroll
    for (int i = 0; i < NR; i++) {
        l[i] = sum_g(l[i]);
        if (g == 0) mls[w][16 * i + c][0] = m[i], mls[w][16 * i + c][1] = l[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NR; i++) {
        const int row = 16 * i + c;
        float mb = -INFINITY;
#pragma unroll
        for (int k = 0; k < NW; k++) mb = fmaxf(mb, mls[k][row][0]);
        const float mz = mb == -INFINITY ? 0.0f : mb, f = __builtin_amdgcn_exp2f(m[i] - mz);
        float lb = 0.0f;
#pragma unroll
        for (int k = 0; k < NW; k++) lb += mls[k][row][1] * __builtin_amdgcn_exp2f(mls[k][row][0] - mz);
#pragma unroll
        for (int x = 0; x < 4; x++)
#pragma unroll
            for (int y = 0; y < VE; y += 4) {
                f4 u;
#pragma unroll
                for (int z = 0; z < 4; z++) u[z] = o[i][y + z][x] * f;
                *(f4 *)(&os[w][row][VE * (4 * g + x) + y]) = u;
            }
        if (w == 0 && g == 0 && nch > 1 && row < tl.live) {
            float *ml = A.part + (size_t)gridDim.x * A.R * DK + ((size_t)blockIdx.x * A.R + row) * 2;
            ml[0] = mb;
            ml[1] = lb;
        }
    }
    __syncthreads();
    for (int i = tid; i < tl.live * (DK / 4); i += NTH) {
        const int row = i / (DK / 4), d = 4 * (i % (DK / 4));
        f4 u = *(const f4 *)&os[0][row][d];
#pragma unroll
        for (int k = 1; k < NW; k++) u += *(const f4 *)&os[k][row][d];
        if (nch > 1) {
            *(f4 *)(A.part + ((size_t)blockIdx.x * A.R + row) * DK + d) = u;
            continue;
        }
        float ms = -INFINITY, ls = 0.0f;
#pragma unroll
        for (int k = 0; k < NW; k++) ms = fmaxf(ms, mls[k][row][0]);
        ms = ms == -INFINITY ? 0.0f : ms;
#pragma unroll
        for (int k = 0; k < NW; k++) ls += mls[k][row][1] * __builtin_amdgcn_exp2f(mls[k][row][0] - ms);
        const float inv = ls == 0.0f ? 0.0f : 1.0f / ls;
        *(f4 *)(a.out + (int64_t)(tl.s.r0 + row / a.G) * a.ldo + (h * a.G + row % a.G) * DK + d) = u * inv;
    }
}

// The chunks of a row, joined in their order: out = sum_c 2^(m_c - M) O_c / sum_c
// 2^(m_c - M) l_c. One workgroup a row and K/V head; NG groups of lanes take every
// NG-th chunk, then the groups are added in order.
template <int DK, int NR>
__global__ __launch_bounds__(NTH) void k_kv_join(const StepArgs A) {
    constexpr int RT = 16 * NR, LN = DK / 4, NG = NTH / LN;
    __shared__ float red[NW];
    __shared__ __attribute__((aligned(16))) float os[NG][DK];
    __shared__ float ls[NG];
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, row = blockIdx.y;
    const int h = blockIdx.x % A.t.Hk, b = blockIdx.x / A.t.Hk;
    const KvTile tl = kv_tile<RT, KB>(A.t, A.a, b, 0);
    if (row >= tl.live) return;
    const int nch = chunks_of(tl.sp.cnt);
    if (nch <= 1) return;
    // chunk i's workgroup: (b nch_max + i) Hk + h
    const size_t wg0 = (size_t)b * A.nch * A.t.Hk + h;
    const size_t wgs = (size_t)A.t.nseq * A.nch * A.t.Hk;
    const float *ml = A.part + wgs * A.R * DK;
    auto slot = [&](int i) { return (wg0 + (size_t)i * A.t.Hk) * A.R + row; };
    // the first contexts are on their way while the maximum is found
    constexpr int U = 4;
    const int gi = tid / LN, d = 4 * (tid % LN);
    f4 x[U];
    float2 y[U];
    auto fetch = [&](int i0) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const size_t s = slot(min(i0 + NG * u, nch - 1));
            x[u] = *(const f4 *)(A.part + s * DK + d);
            y[u] = *(const float2 *)(ml + 2 * s);
        }
    };
    fetch(gi);
    float m = -INFINITY;
    for (int i = tid; i < nch; i += NTH) m = fmaxf(m, ml[2 * slot(i)]);
    m = wave_max<64>(m);
    if (lane == 0) red[w] = m;
    __syncthreads();
    m = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    const float mz = m == -INFINITY ? 0.0f : m;
    f4 o = {0.0f, 0.0f, 0.0f, 0.0f};
    float l = 0.0f;
    for (int i0 = gi; i0 < nch; i0 += NG * U) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const bool in = i0 + NG * u < nch;
            const float f = in ? __builtin_amdgcn_exp2f(y[u].x - mz) : 0.0f;
            l += in ? f * y[u].y : 0.0f;
            o += in ? f * x[u] : f4{0.0f, 0.0f, 0.0f, 0.0f};
        }
        if (i0 + NG * U < nch) fetch(i0 + NG * U);
    }
    *(f4 *)&os[gi][d] = o;
    if (d == 0) ls[gi] = l;
    __syncthreads();
    if (gi == 0) {
#pragma unroll
        for (int i = 1; i < NG; i++) {
            o += *(const f4 *)&os[i][d];
            l += ls[i];
        }
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        *(f4 *)(A.a.out + (int64_t)(tl.s.r0 + row / A.a.G) * A.a.ldo + (h * A.a.G + row % A.a.G) * DK + d) = o * inv;
    }
}

// The launch's sizes: sixteens of rows in a tile (17 to 32 rows in one tile read the keys once: two requests
// of 30000 keys, 8 rows, 32 heads on 8, f16, 64 us, in two tiles 73; 16 of 2000, 5 rows, 41 and 48),
// chunks of a sequence's keys, rows of a partial result.
struct Plan {
    int nr, nch, R;
    int64_t wgs;
};
Plan plan_of(int nseq, int Hk, int page, int max_pages, const KvAttend &a) {
    Plan p;
    p.R = a.max_new * a.G;   // (at most 32)
    p.nr = p.R > 16 ? 2 : 1;
    const int64_t cap = (int64_t)max_pages * page;
    const int keys = (int)(a.max_len < cap ? a.max_len : cap), all = (keys + KB - 1) / KB;
    int64_t blocks = all;
    if (a.window) {
        // (a sequence's rows reach max_new - 1 keys further; each end of each part may cut a block)
        const int64_t win = ((int64_t)a.window + a.max_new + KB - 1) / KB + 1, sink = ((int64_t)a.sinks + KB - 1) / KB + 1;
        if (win + sink < blocks) blocks = win + sink;
    }
    p.nch = most_chunks((int)blocks);
    p.wgs = (int64_t)nseq * p.nch * Hk;
    return p;
}

}  // namespace

int64_t mh_kv_attention_ws(int nseq, int rows, int Hk, int page, int max_pages, int type, int dk, const KvAttend &a) {
    if ((int64_t)a.max_new * a.G >= 1 << 30) return -1;
    if (mh_kv_prompt(a)) return mh_kv_prompt_ws(nseq, rows, Hk, page, max_pages, type, dk, a);
    const Plan p = plan_of(nseq, Hk, page, max_pages, a);
    if (p.wgs >= 1 << 24) return -1;   // (a launch holds less than 2^32 threads)
    return p.nch > 1 ? p.wgs * p.R * (dk + 2) : 0;
}

hipError_t mh_launch_kv_attention(const KvTables &t, int type, int dk, const KvAttend &a, float *ws, hipStream_t st) {
    if (mh_kv_prompt(a)) return mh_launch_kv_prompt(t, type, dk, a, ws, st);
    const Plan p = plan_of(t.nseq, t.Hk, t.page, t.max_pages, a);
    const StepArgs A{t, a, ws, p.nch, p.R};
    auto go = [&](auto step, auto join) {
        hipLaunchKernelGGL(step, dim3((unsigned)p.wgs), dim3(NTH), 0, st, A);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess || p.nch <= 1) return e;
        hipLaunchKernelGGL(join, dim3((unsigned)((int64_t)t.nseq * t.Hk), p.R), dim3(NTH), 0, st, A);
        return hipGetLastError();
    };
#define KV_GO(T, DK) (p.nr == 1 ? go(k_kv_step<T, DK, 1>, k_kv_join<DK, 1>) : go(k_kv_step<T, DK, 2>, k_kv_join<DK, 2>))
    if (dk == 128) return type == KV_F32 ? KV_GO(float, 128) : type == KV_F16 ? KV_GO(_Float16, 128) : KV_GO(__bf16, 128);
    return type == KV_F32 ? KV_GO(float, 64) : type == KV_F16 ? KV_GO(_Float16, 64) : KV_GO(__bf16, 64);
#undef KV_GO
}
