// kv_prompt.hip — attention over a paged cache for many new rows of a sequence
// (prompts, and parts of them). The mathematics and the visibility of keys are
// kv_attention.hip's.
//
// One workgroup = four waves = 128 rows of one K/V head (token * G + head), 32 a
// wave, over all the keys they see or one chunk of them; tiles of 64 keys (f32
// caches: 32). K and V tiles go from the cache's pages to LDS as they lie
// (global_load_lds, two slots: the next tile's copies run while this one's products
// do), rows swizzled so that the reads below meet no bank twice.
//
// Products, S^T = K Q^T and O^T = V^T P^T (lane l, c = l & 31, hf = l >> 5: A row c,
// B column c, D rows 8 (e / 4) + 4 hf + e % 4, column c): a lane holds the scores of
// one query row, half of a tile's keys, and its probabilities are the second
// product's B operand as they lie, which is free to take its keys in that order.
// The 32x32x16 MFMA of 16-bit types, slots 8 hf + j; value rows come transposed from
// LDS (ds_read_b64_tr_b16); q and probabilities in terms (kv_terms.h; for f16 a q row scaled
// by a power of two, probabilities below 2^14).
//   f32 caches: a tile is taken apart into three bf16 planes in LDS, exactly (8 bits
//   each); six of the nine products of terms, all but those below 2^-24 of the whole.
//   The copies of the next tile run into the one f32 slot while the planes are in use.
//   (The 32x32x2 f32 MFMA takes 2.7 times as long: four prompts with a window of 512,
//   8 heads, 214 us, then 128.)
// Statistics, in powers of two: a row's reference m follows its maximum only when that
// is 2^6 above it, so the context is seldom rescaled; p = 2^(s - m + TOP), TOP 8 for f16,
// whose small probabilities would be subnormal without it, else 0.
// Sums: over thousands of keys that score alike, the roundings of one long f32 sum go the same way (relative
// error 3e-5 at 8k keys, 1e-4 at 32k). So a tile's probabilities are summed as a tree, and each FOLD tiles
// apart: the chains are at most 128 steps (l) and 512 (o), then one for each part. The whole's context waits
// in the rows of the result (or the partial result). That costs 1% of one prompt of 8192 rows, f16 (with 32
// tiles a part 4%), 1% of eight ragged bf16 prompts with heads of 64, 4% of one f32 prompt of 4096 with these.
//
// What bounds it: the card's power. One prompt of 8192 rows, 32 heads on 8 of 128, f16: 1020 to
// 1030 us, 1.05 PFLOP/s of MFMAs issued (a large product of the library: 1.2). As first built
// (1042 us) it took 824 on zeros, 10% less without its softmax, 11% without its copies. 32 rows a
// wave hold q's terms, the context and a tile's fragments in 256 registers, two waves a SIMD, and
// not all fits: 3 to 20 vector registers a lane and some 90 to 170 scalar ones are spilled. One wave
// a SIMD needs no spill and takes 11 to 19% longer on 16-bit caches (f32, one prompt of 4096, 8 heads: 7%
// less; four with a window: 39% longer). Heads of 64 (eight bf16 prompts of 100 to 4000 rows, 16 heads on 4) have half
// the MFMAs for a probability and are bound by the VALU: 168 registers, three waves, up to 4 spilled,
// 242 -> 230 us then, now 234 (f16, one prompt of 4096, 32 heads: 0.7% slower). What a masked tile needs of a row is
// formed there (one bf16 prompt of 4096, 32 heads of 128: 388 -> 374).
#include <hip/hip_runtime.h>
#include <math.h>

#include <type_traits>

#include "kv.h"
#include "kv_terms.h"
#include "launch.h"
#include "product.h"

namespace {

constexpr int NW = 4, NTH = 64 * NW;
constexpr int RT = 32 * NW;   // rows of a tile
template <typename T> constexpr int KB = sizeof(T) == 4 ? 32 : 64;   // keys of a tile
// Tiles that are summed before they join the whole (even). MFMAs that follow each other into one sum:
// 8 a tile for f16, 12 for bf16 and f32.
template <typename T> constexpr int FOLD = std::is_same_v<T, _Float16> ? 64 : 32;
typedef short s4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) void lds_void;
typedef __attribute__((address_space(3))) s4 lds_s4;
typedef __attribute__((address_space(1))) const void glob_void;

struct PromptArgs {
    KvTables t;
    KvAttend a;
    float *part;         // partial contexts [workgroup][RT][DK], then their references and sums [workgroup][RT][2]
    int ntile, nch, ct;  // tiles (at most), chunks of a tile's keys (at most), key tiles of a chunk
};

// the larger of the two halves' values, in both
__device__ __forceinline__ float max_halves(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// The sequence and its row tile that tile number `at` of the call is. Tiles are numbered
// in rounds: the last of each sequence (in causal order its longest), then the
// last but one of each that has two, and so on, so that no long one starts late. With
// T_b tiles in sequence b, sum_b min(T_b, k) of them come before round k. false: there
// are fewer. Every thread of the workgroup takes part; lds: NW + 2 words, free again
// after the workgroup's next barrier.
__device__ __forceinline__ int wave_sum_i(int x) {
    auto step = [&](auto ctrl) { x += __builtin_amdgcn_update_dpp(0, x, decltype(ctrl)::value, 0xF, 0xF, false); };
    step(std::integral_constant<int, 0xB1>{});    // (the steps of wave_sum)
    step(std::integral_constant<int, 0x4E>{});
    step(std::integral_constant<int, 0x141>{});
    step(std::integral_constant<int, 0x140>{});
    auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    x = r[0] + r[1];
    r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    return r[0] + r[1];
}
__device__ __forceinline__ int block_sum(int x, int *lds) {
    x = wave_sum_i(x);
    __syncthreads();
    if (threadIdx.x % 64 == 0) lds[threadIdx.x / 64] = x;
    __syncthreads();
    return lds[0] + lds[1] + lds[2] + lds[3];
}
__device__ __forceinline__ bool find_tile(const KvTables &t, const KvAttend &a, int at, int *lds, int &b, int &rt) {
    int *hit = lds + NW;
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    auto tiles = [&](int s) { return s < t.nseq ? (kv_rows(a, kv_seq(t, s)) + RT - 1) / RT : 0; };
    if (t.nseq == 1) {
        b = 0;
        rt = tiles(0) - 1 - at;
        return rt >= 0;
    }
    // up to 64 sequences: each wave by itself, a sequence a lane
    const bool few = t.nseq <= 64;
    const int mine = tiles(few ? lane : tid);   // (the others, if there are more, are read again each time)
    auto before = [&](int k) {
        if (few) return wave_sum_i(min(mine, k));
        int x = min(mine, k);
        for (int s = tid + NTH; s < t.nseq; s += NTH) x += min(tiles(s), k);
        return block_sum(x, lds);
    };
    // the round: the largest k with before(k) <= at
    int k = 0, top = (int)(((int64_t)a.max_new * a.G + RT - 1) / RT), base = 0;
    while (k < top) {
        const int mid = k + (top - k + 1) / 2, n = before(mid);
        if (n <= at) k = mid, base = n;
        else top = mid - 1;
    }
    // in it, the sequences that have more than k tiles, in order
    at -= base;
    if (few) {
        const uint64_t have = __ballot(mine > k);
        const uint64_t here = __ballot(mine > k && __popcll(have & ((1ull << lane) - 1)) == at);
        if (!here) return false;
        b = __ffsll((unsigned long long)here) - 1;
        rt = __shfl(mine, b, 64) - 1 - k;
        return true;
    }
    for (int s0 = 0; s0 < t.nseq; s0 += NTH) {
        const int n = s0 ? tiles(s0 + tid) : mine;
        const uint64_t have = __ballot(n > k);
        __syncthreads();
        if (lane == 0) lds[w] = __popcll(have);
        if (tid == 0) hit[0] = -1;
        __syncthreads();
        int rank = __popcll(have & ((1ull << lane) - 1));
        for (int i = 0; i < w; i++) rank += lds[i];
        if (n > k && rank == at) hit[0] = s0 + tid, hit[1] = n - 1 - k;
        at -= lds[0] + lds[1] + lds[2] + lds[3];
        __syncthreads();
        if (hit[0] >= 0) {
            b = hit[0];
            rt = hit[1];
            return true;
        }
    }
    return false;
}

// A wave's operands and products on one kind of cache. at_k, at_v: where this lane's
// first pieces of a K and a V tile lie; other rows of a tile that a lane reads differ by
// a constant number of rows whose swizzle differs by a constant xor.
template <typename T, int DK> struct Ops {   // 16 bits
    using X = KvTerms<T>;
    typedef typename X::v8 v8;
    static constexpr int KS = DK / 16, DT = DK / 32, ROW = DK * 2;
    static constexpr float TOP = X::N == 2 ? 8.0f : 0.0f;
    // K fragments of the next half are read ahead where q's terms leave the registers
    static constexpr bool AHEAD = X::N * KS <= 16;
    // of any 16 rows that follow each other one piece each, and of any four the four
    // pieces that follow each other, lie in all 64 banks
    static __device__ __forceinline__ int swz(int row) {
        return DK == 128 ? (row & 3) * 4 + (row >> 2 & 3) : (row >> 1 & 1) * 4 + (row >> 2 & 3);
    }
    // feature of element x of context tile d
    static __device__ __forceinline__ int feature(int d, int x, int hf) { return 32 * d + 8 * (x / 4) + 4 * hf + x % 4; }
    v8 q[KS][X::N];
    float sc;   // what turns a sum of products into a score, in powers of two
    int at_k, at_v;
    __device__ __forceinline__ void init(const float *qp, float f, bool live, int lane) {
        const int c = lane & 31, hf = lane >> 5, vrow = 4 * hf + (lane & 15) / 4;
        at_k = c * ROW + (hf ^ swz(c)) * 16;
        at_v = vrow * ROW + ((2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) ^ swz(vrow)) * 16 + 8 * (lane & 1);
        float x[KS][8], mx = 0.0f;
#pragma unroll
        for (int s = 0; s < KS; s++) {
            *(f4 *)&x[s][0] = *(const f4 *)(qp + 16 * s + 8 * hf);
            *(f4 *)&x[s][4] = *(const f4 *)(qp + 16 * s + 8 * hf + 4);
#pragma unroll
            for (int j = 0; j < 8; j++) {
                x[s][j] = live ? x[s][j] * f : 0.0f;
                mx = fmaxf(mx, fabsf(x[s][j]));
            }
        }
        const int e = X::shift(max_halves(mx));
        sc = ldexpf(1.0f, -e);
#pragma unroll
        for (int s = 0; s < KS; s++) {
#pragma unroll
            for (int j = 0; j < 8; j++) x[s][j] = ldexpf(x[s][j], e);
            X::split(x[s], q[s]);
        }
    }
    // The products of a tile around `soft`, which turns half n's scores into
    // probabilities. kt, vt: the tile; ka, va: at_k, at_v.
    template <typename F>
    __device__ __forceinline__ void tile(const uint8_t *kt, const uint8_t *vt, int ka, int va, f16v (&o)[DT], F soft) const {
        auto k_frag = [&](int n, int u) { return *(const v8 *)(kt + 32 * n * ROW + (ka ^ 32 * u)); };
        auto v_frag = [&](int n, int g, int d) {   // slots 8 hf + j: keys 32 n + 16 g + 4 hf + j, from j = 4 on 8 further
            s4 v[2];
#pragma unroll
            for (int y = 0; y < 2; y++)
                v[y] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                    (lds_s4 *)(vt + (32 * n + 16 * g + 8 * y) * ROW + (va ^ (64 * d + 32 * y))));
            return __builtin_bit_cast(v8, __builtin_shufflevector(v[0], v[1], 0, 1, 2, 3, 4, 5, 6, 7));
        };
        v8 kf[KS], vf[2][DT];
        if constexpr (AHEAD) {
#pragma unroll
            for (int u = 0; u < KS; u++) kf[u] = k_frag(0, u);
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int n = 0; n < 2; n++) {
            f16v s = zero16();
#pragma unroll
            for (int u = 0; u < KS; u++) {
                if constexpr (!AHEAD) kf[u] = k_frag(n, u);
#pragma unroll
                for (int x = 0; x < X::N; x++) s = X::mfma32(kf[u], q[u][x], s);
            }
            if constexpr (AHEAD) {
#pragma unroll
                for (int g = 0; g < 2; g++)
#pragma unroll
                    for (int d = 0; d < DT; d++) vf[g][d] = v_frag(n, g, d);
                __builtin_amdgcn_sched_barrier(0);
            }
            soft(n, s, sc);
#pragma unroll
            for (int g = 0; g < 2; g++) {
                float p[8];
#pragma unroll
                for (int x = 0; x < 8; x++) p[x] = s[8 * g + x];
                v8 pt[X::N];
                X::split(p, pt);
                if constexpr (AHEAD)
                    if (g == 0 && n == 0) {
#pragma unroll
                        for (int u = 0; u < KS; u++) kf[u] = k_frag(1, u);
                    }
#pragma unroll
                for (int d = 0; d < DT; d++) {
                    if constexpr (!AHEAD) vf[g][d] = v_frag(n, g, d);
#pragma unroll
                    for (int x = 0; x < X::N; x++) o[d] = X::mfma32(vf[g][d], pt[x], o[d]);
                }
            }
        }
    }
    // two packed elements: those that are not finite set to 0; whether there are any
    static __device__ __forceinline__ bool clean(uint32_t &x) {
        const bool l = kv_odd_lo<T>(x), h = kv_odd_hi<T>(x);
        x = (l ? 0u : x & 0xffffu) | (h ? 0u : x & 0xffff0000u);
        return l || h;
    }
};
// f32: bf16's operands, a tile's planes behind each other
template <int DK> struct Ops<float, DK> : Ops<__bf16, DK> {
    using B = Ops<__bf16, DK>;
    using X = typename B::X;
    typedef typename B::v8 v8;
    static constexpr int KS = B::KS, DT = B::DT, ROW = B::ROW, PLANE = KB<float> * ROW;
    // sum += a b, a and b of three terms each
    static __device__ __forceinline__ f16v product(const v8 (&a)[3], const v8 (&b)[3], f16v sum) {
#pragma unroll
        for (int i = 0; i < 3; i++)
#pragma unroll
            for (int j = 0; j < 3 - i; j++) sum = X::mfma32(a[i], b[j], sum);
        return sum;
    }
    template <typename F>
    __device__ __forceinline__ void tile(const uint8_t *kt, const uint8_t *vt, int ka, int va, f16v (&o)[DT], F soft) const {
        f16v s = zero16();
#pragma unroll
        for (int u = 0; u < KS; u++) {
            v8 k[3];
#pragma unroll
            for (int i = 0; i < 3; i++) k[i] = *(const v8 *)(kt + i * PLANE + (ka ^ 32 * u));
            s = product(k, this->q[u], s);
        }
        soft(0, s, 1.0f);
#pragma unroll
        for (int g = 0; g < 2; g++) {
            float p[8];
#pragma unroll
            for (int x = 0; x < 8; x++) p[x] = s[8 * g + x];
            v8 pt[3];
            X::split(p, pt);
#pragma unroll
            for (int d = 0; d < DT; d++) {
                v8 v[3];
#pragma unroll
                for (int i = 0; i < 3; i++) {
                    s4 y[2];
#pragma unroll
                    for (int z = 0; z < 2; z++)
                        y[z] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                            (lds_s4 *)(vt + i * PLANE + (16 * g + 8 * z) * ROW + (va ^ (64 * d + 32 * z))));
                    v[i] = __builtin_bit_cast(v8, __builtin_shufflevector(y[0], y[1], 0, 1, 2, 3, 4, 5, 6, 7));
                }
                o[d] = product(v, pt, o[d]);
            }
        }
    }
    // eight elements into their place in the three planes: 8 bits of each, cut off
    static __device__ __forceinline__ void put(float (&x)[8], uint8_t *at) {
#pragma unroll
        for (int i = 0; i < 3; i++) {
            uint32_t h[4];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const uint32_t a = __float_as_uint(x[2 * j]), b = __float_as_uint(x[2 * j + 1]);
                h[j] = __builtin_amdgcn_perm(b, a, 0x07060302u);
                if (i < 2) {
                    x[2 * j] -= __uint_as_float(a & 0xffff0000u);
                    x[2 * j + 1] -= __uint_as_float(b & 0xffff0000u);
                }
            }
            *(uint4 *)(at + i * PLANE) = uint4{h[0], h[1], h[2], h[3]};
        }
    }
    static __device__ __forceinline__ bool clean(float &x) {
        const bool odd = !(fabsf(x) < INFINITY);
        x = odd ? 0.0f : x;
        return odd;
    }
};

template <typename T, int DK>
__global__ __launch_bounds__(NTH, DK == 64 ? 3 : 2) void k_kv_prompt(const PromptArgs A) {
    using W = Ops<T, DK>;
    constexpr bool F32 = sizeof(T) == 4;
    constexpr int DT = W::DT, KT = KB<T>;
    constexpr int ROW = DK * sizeof(T), CH = ROW / 16;   // bytes of a row of the cache, 16-byte pieces
    constexpr int TB = KT * ROW;                   // bytes of a tile
    constexpr int WR = KT / NW;                    // rows of a tile that a wave copies
    constexpr int RPI = 64 / CH;                   // rows of one copy instruction
    // (Separate arrays, so that reads of one do not wait for copies into another. f32: one slot and
    // the planes; with heads of 128 that is just half of a CU's LDS, so there is no other array.)
    __shared__ __attribute__((aligned(16))) uint8_t k0[TB], k1[F32 ? 16 : TB], v0[TB], v1[F32 ? 16 : TB];
    __shared__ __attribute__((aligned(16))) uint8_t kp[F32 ? 3 * KT * DK * 2 : 16], vp[F32 ? 3 * KT * DK * 2 : 16];
    const KvTables &t = A.t;
    const KvAttend &a = A.a;
    const int tid = threadIdx.x, lane = tid & 63, c = lane & 31, hf = lane >> 5;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    int at = blockIdx.x;
    const int h = at % t.Hk;
    at /= t.Hk;
    int b, rt;
    if (!find_tile(t, a, at % A.ntile, (int *)k0, b, rt)) return;
    b = __builtin_amdgcn_readfirstlane(b);
    rt = __builtin_amdgcn_readfirstlane(rt);
    const KvTile tl = kv_tile<RT, KT>(t, a, b, rt);
    const int ch = at / A.ntile, nch = max((tl.sp.cnt + A.ct - 1) / A.ct, 1);
    if (ch >= nch) return;
    const int e0 = ch * A.ct, e1 = min(e0 + A.ct, tl.sp.cnt);

    // this lane's row: its token and head (formed where they are used: kept, they would cost registers
    // that the products need)
    auto row_of = [&](int &tok, int &head) {
        int ln = lane;
        asm volatile("" : "+v"(ln));
        const int r = rt * RT + min(32 * w + (ln & 31), tl.live - 1);
        tok = r / a.G;
        head = h * a.G + (r - tok * a.G);
    };
    // what the wave's first and last row see (a wave of no rows: nothing)
    const bool idle = 32 * w >= tl.live;
    const int t0 = (rt * RT + min(32 * w, tl.live - 1)) / a.G, t1 = (rt * RT + min(32 * w + 31, tl.live - 1)) / a.G;
    const int wlo0 = kv_first(a, tl.s, t0), wlo1 = kv_first(a, tl.s, t1);
    const int whi0 = kv_last(t, a, tl.s, t0), whi1 = idle ? -1 : kv_last(t, a, tl.s, t1);
    W wv;
    {
        int tok, head;
        row_of(tok, head);
        wv.init(a.q + (int64_t)(tl.s.r0 + tok) * a.ldq + head * DK, a.scale * 1.4426950408889634f, 32 * w + c < tl.live, lane);
    }
    f16v o[DT];
#pragma unroll
    for (int d = 0; d < DT; d++) o[d] = zero16();
    float m = -INFINITY, l = 0.0f;

    // Every FOLD<T> tiles o and l join the whole's context and sum, and start anew. The whole's
    // context lies where the result will: the rows are this wave's own, and their q has
    // been read. Its reference and sum: kept in registers, these two would push others out.
    // (always_inline: of what a call does not inline, o lies in memory.)
    volatile float whole_m, whole_l;
    const bool split = nch > 1;
    auto row_out = [&]() __attribute__((always_inline)) {
        int tok, head;
        row_of(tok, head);
        return split ? A.part + ((size_t)blockIdx.x * RT + 32 * w + c) * DK
                     : a.out + (int64_t)(tl.s.r0 + tok) * a.ldo + head * DK;
    };
    auto add_whole = [&](const float *op) __attribute__((always_inline)) {   // to o and l
        const float mw = whole_m, al = mw == m ? 1.0f : __builtin_amdgcn_exp2f(mw - m);
        l += whole_l * al;
#pragma unroll
        for (int d0 = 0; d0 < DT; d0 += 2) {
            f4 u[2][4];   // (on their way before the first is used)
#pragma unroll
            for (int d = 0; d < 2; d++)
#pragma unroll
                for (int x = 0; x < 4; x++) u[d][x] = *(const f4 *)(op + W::feature(d0 + d, 4 * x, hf));
#pragma unroll
            for (int d = 0; d < 2; d++)
#pragma unroll
                for (int x = 0; x < 16; x++) o[d0 + d][x] += u[d][x / 4][x % 4] * al;
        }
    };
    auto put = [&](float *op, float f) __attribute__((always_inline)) {
#pragma unroll
        for (int d = 0; d < DT; d++)
#pragma unroll
            for (int x = 0; x < 16; x += 4)
                *(f4 *)(op + W::feature(d, x, hf)) = f4{o[d][x], o[d][x + 1], o[d][x + 2], o[d][x + 3]} * f;
    };
    auto fold = [&](int e) __attribute__((always_inline)) {   // after tile e, the last of a part but not of all
        if ((e + 1 - e0) % FOLD<T> || e + 1 == e1) return;
        if (32 * w + c < tl.live) {
            float *op = row_out();
            if (e + 1 - e0 > FOLD<T>) add_whole(op);
            put(op, 1.0f);
        }
        whole_m = m;
        whole_l = l;
        l = 0.0f;
#pragma unroll
        for (int d = 0; d < DT; d++) o[d] = zero16();
    };

    // A lane holds the page of one row of a tile, read from the table a tile ahead and
    // looked at when it is used; wave w copies rows WR w .. of it.
    auto page_of = [&](int e) {
        const int j = min(tl.sp.block(min(e, e1 - 1)) * KT + lane % KT, tl.hi1);
        return t.pages[(size_t)b * t.max_pages + j / t.page];
    };
    // copies tile e; which of its rows there are
    auto copy = [&](int e, int pg, uint8_t *kd, uint8_t *vd) {
        const int j = tl.sp.block(e) * KT + lane % KT;
        const bool have = j <= tl.hi1 && (unsigned)pg < (unsigned)t.n_pages;
        const uint32_t sl = have ? ((uint32_t)pg * t.Hk + h) * t.page + j % t.page : 0;
#pragma unroll
        for (int i = 0; i < WR / RPI; i++) {
            const int rr = WR * w + RPI * i + lane / CH;
            const size_t off = (size_t)(uint32_t)__shfl((int)sl, rr, 64) * ROW + (((lane % CH) ^ (F32 ? 0 : W::swz(rr))) * 16);
            __builtin_amdgcn_global_load_lds((const glob_void *)((const uint8_t *)t.k + off),
                                             (lds_void *)(kd + (WR * w + RPI * i) * ROW), 16, 0, 0);
            __builtin_amdgcn_global_load_lds((const glob_void *)((const uint8_t *)t.v + off),
                                             (lds_void *)(vd + (WR * w + RPI * i) * ROW), 16, 0, 0);
        }
        return (uint64_t)__ballot(have);
    };
    auto whole = [&](uint64_t ok, int j0, int hi_first, int lo_last) -> bool {   // every row sees every key
        return __builtin_amdgcn_readfirstlane(ok == ~0ull && j0 + KT - 1 <= hi_first && (j0 >= lo_last || j0 + KT <= a.sinks));
    };

    // Tile e's products. A value that only some rows see meets the others' probability 0,
    // which hides it unless it is not finite: such an element counts as 0 in the
    // product (and `odd` says that there are any), and is added afterwards to the rows
    // that see it.
    auto tile = [&](int e, uint64_t okw, const uint8_t *kt, const uint8_t *vt, bool odd) {
        const int j0 = tl.sp.block(e) * KT;
        if (j0 > whi1 || (j0 + KT <= wlo0 && j0 >= a.sinks)) return;   // no row of this wave sees any
        // (opaque: the addresses formed from these, kept for every tile, would cost
        // registers that the products need)
        int ka = wv.at_k, va = wv.at_v;
        asm volatile("" : "+v"(ka), "+v"(va));
        const bool every = whole(okw, j0, whi0, wlo1);
        wv.tile(kt, vt, ka, va, o, [&](int n, f16v &s, float sc) {
            if (!every) {
                int tok, head;
                row_of(tok, head);
                const int lo = kv_first(a, tl.s, tok), hi = kv_last(t, a, tl.s, tok);
                const uint32_t mine = (uint32_t)(okw >> (32 * n + 4 * hf));
#pragma unroll
                for (int x = 0; x < 16; x++) {
                    const int jj = 8 * (x / 4) + x % 4, j = j0 + 32 * n + jj + 4 * hf;
                    const bool see = (mine >> jj & 1) && j <= hi && (j >= lo || j < a.sinks);
                    s[x] = see ? s[x] : -INFINITY;
                }
            }
            float mx = s[0];
#pragma unroll
            for (int x = 1; x < 16; x++) mx = fmaxf(mx, s[x]);
            mx = max_halves(mx) * sc;
            const bool up = mx > m + 6.0f;   // (m = -inf: any finite maximum)
            if (__any(up)) {
                const float al = up ? __builtin_amdgcn_exp2f(m - mx) : 1.0f;
                m = up ? mx : m;
                l *= al;
#pragma unroll
                for (int d = 0; d < DT; d++) o[d] *= al;
            }
            const float sub = W::TOP - (m == -INFINITY ? 0.0f : m);
            float sum[8];   // (as a tree: l takes one step for 16 keys)
#pragma unroll
            for (int x = 0; x < 16; x++) s[x] = __builtin_amdgcn_exp2f(fmaf(s[x], sc, sub));
#pragma unroll
            for (int x = 0; x < 8; x++) sum[x] = s[2 * x] + s[2 * x + 1];
            l += ((sum[0] + sum[1]) + (sum[2] + sum[3])) + ((sum[4] + sum[5]) + (sum[6] + sum[7]));
        });
        if (__builtin_expect(odd, 0)) {   // (as likely as not, it would take registers from the products: 3 to 9% slower)
            int tok, head;
            row_of(tok, head);
            const int lo = kv_first(a, tl.s, tok), hi = kv_last(t, a, tl.s, tok);
            for (int jj = 0; jj < KT; jj++) {
                const int j = j0 + jj;
                if (!(okw >> jj & 1) || j > hi || (j < lo && j >= a.sinks)) continue;
                const T *vr = (const T *)t.v + (size_t)kv_slot(t, b, j, h) * DK;
#pragma unroll
                for (int d = 0; d < DT; d++)
#pragma unroll
                    for (int x = 0; x < 16; x++) {
                        const float v = (float)vr[W::feature(d, x, hf)];
                        if (!(fabsf(v) < INFINITY)) o[d][x] += v;
                    }
            }
        }
    };

    if (t.nseq > 64) __syncthreads();   // (find_tile's words lie in k0)
    if (e0 < e1) {
        const auto landed = [] { __builtin_amdgcn_s_waitcnt(0x0f70); };   // vmcnt(0): this wave's copies
        uint64_t ok = copy(e0, page_of(e0), k0, v0);
        int pg = page_of(e0 + 1);
        if constexpr (F32) {
            constexpr int GR = DK / 8;   // groups of eight elements in a row
            for (int e = e0; e < e1; e++) {
                landed();
                __syncthreads();
                const bool all = whole(ok, tl.sp.block(e) * KT, tl.hi0, tl.lo1);
                bool odd = false;
#pragma unroll
                for (int i = 0; i < KT * GR / NTH; i++) {
                    const int row = (tid + NTH * i) / GR, gr = (tid + NTH * i) % GR;
                    const int to = row * W::ROW + (gr ^ W::swz(row)) * 16;
                    float x[8];
                    auto get = [&](const uint8_t *from) {
                        *(f4 *)&x[0] = *(const f4 *)(from + row * ROW + gr * 32);
                        *(f4 *)&x[4] = *(const f4 *)(from + row * ROW + gr * 32 + 16);
                    };
                    get(k0);
                    W::put(x, kp + to);
                    get(v0);
                    if (!all)
#pragma unroll
                        for (int y = 0; y < 8; y++) odd |= W::clean(x[y]);
                    W::put(x, vp + to);
                }
                if (!all) {   // a word of this wave's own rows, which it has read, says what it found
                    odd = __any(odd);
                    if (lane == 0) *(int *)(v0 + (64 * w) / GR * ROW) = odd;
                }
                __syncthreads();
                if (!all) {
                    odd = false;
#pragma unroll
                    for (int i = 0; i < NW; i++) odd |= *(const int *)(v0 + (64 * i) / GR * ROW) != 0;
                    __syncthreads();
                }
                const uint64_t now = ok;
                if (e + 1 < e1) ok = copy(e + 1, pg, k0, v0);
                pg = page_of(e + 2);
                tile(e, now, kp, vp, odd);
                fold(e);
            }
        } else {
            // cleaned in place where it has to be, and the products
            auto turn = [&](int e, uint64_t now, const uint8_t *kt, uint8_t *vt) {
                int odd = 0;
                if (!whole(now, tl.sp.block(e) * KT, tl.hi0, tl.lo1)) {
#pragma unroll
                    for (int i = 0; i < TB / 16 / NTH; i++) {
                        uint4 x = ((uint4 *)vt)[tid + NTH * i];
                        const bool y[4] = {W::clean(x.x), W::clean(x.y), W::clean(x.z), W::clean(x.w)};
                        if (y[0] || y[1] || y[2] || y[3]) {
                            odd = 1;
                            ((uint4 *)vt)[tid + NTH * i] = x;
                        }
                    }
                    odd = __syncthreads_or(odd);
                }
                tile(e, now, kt, vt, odd != 0);
            };
            for (int e = e0;; e += 2) {
                landed();
                __syncthreads();
                uint64_t now = ok;
                if (e + 1 < e1) ok = copy(e + 1, pg, k1, v1);
                pg = page_of(e + 2);
                turn(e, now, k0, v0);
                if (e + 1 >= e1) break;
                landed();
                __syncthreads();
                now = ok;
                if (e + 2 < e1) ok = copy(e + 2, pg, k0, v0);
                pg = page_of(e + 3);
                turn(e + 1, now, k1, v1);
                if (e + 2 >= e1) break;
                fold(e + 1);
            }
        }
    }
    const int r = 32 * w + c;
    if (r >= tl.live) return;
    float *op = row_out();
    if (e1 - e0 > FOLD<T>) add_whole(op);
    l += __shfl_xor(l, 32, 64);
    if (split && hf == 0) {
        float *ml = A.part + (size_t)gridDim.x * RT * DK + 2 * ((size_t)blockIdx.x * RT + r);
        ml[0] = m;
        ml[1] = l;
    }
    put(op, split ? 1.0f : l == 0.0f ? 0.0f : 1.0f / l);
}

// The chunks of a tile's rows, joined in their order, as k_kv_join.
template <typename T, int DK>
__global__ __launch_bounds__(NTH) void k_kv_prompt_join(const PromptArgs A) {
    constexpr int LN = DK / 4, RB = NTH / LN;   // lanes of a row, rows of a workgroup
    int at = blockIdx.x;
    const int h = at % A.t.Hk;
    at /= A.t.Hk;
    __shared__ int lds[NW + 2];
    int b, rt;
    if (!find_tile(A.t, A.a, at, lds, b, rt)) return;
    const KvTile tl = kv_tile<RT, KB<T>>(A.t, A.a, b, rt);
    const int nch = (tl.sp.cnt + A.ct - 1) / A.ct, row = blockIdx.y * RB + threadIdx.x / LN;
    if (nch <= 1 || row >= tl.live) return;
    const int d = 4 * (threadIdx.x % LN);
    const size_t wgs = (size_t)A.t.Hk * A.ntile * A.nch;
    const float *ml = A.part + wgs * RT * DK;
    auto slot = [&](int i) { return (((size_t)i * A.ntile + at) * A.t.Hk + h) * RT + row; };
    float m = -INFINITY;
#pragma unroll 8
    for (int i = 0; i < nch; i++) m = fmaxf(m, ml[2 * slot(i)]);
    const float mz = m == -INFINITY ? 0.0f : m;
    f4 o = {0.0f, 0.0f, 0.0f, 0.0f};
    float l = 0.0f;
    constexpr int U = 4;   // chunks whose loads are on their way at a time
    for (int i0 = 0; i0 < nch; i0 += U) {
        f4 x[U];
        float2 y[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const size_t s = slot(min(i0 + u, nch - 1));
            x[u] = *(const f4 *)(A.part + s * DK + d);
            y[u] = *(const float2 *)(ml + 2 * s);
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (i0 + u >= nch) break;
            const float f = __builtin_amdgcn_exp2f(y[u].x - mz);
            l += f * y[u].y;
            o += f * x[u];
        }
    }
    const int rr = rt * RT + row;
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    *(f4 *)(A.a.out + (int64_t)(tl.s.r0 + rr / A.a.G) * A.a.ldo + (h * A.a.G + rr % A.a.G) * DK + d) = o * inv;
}

// The launch's sizes, from the call's. A tile's keys are split into chunks where that is
// likely to be faster: the longest chunk's tiles, one workgroup a CU or two, and the join of
// the partial results, which grows with the workgroups (units of 0.1 us, measured on heads of 128; heads of
// 64, with half the work a tile and three workgroups a CU, go by the same). Every tile counts as long as
// the longest may be, by max_len and the window. 64-row prompts
// on 64 k keys, 8 heads of 128, f16, unsplit and in as many chunks as 512 places take: 32 of them,
// k = 3, 17 and 26 us, k = 10 32 and 38, k = 40 98 and 94; four of them, k = 3, 14 and 15, k = 6 20
// and 16, k = 40 27 in 8 chunks and 32 in 14. f32, 32 of them on 192 keys 29 and 35.
struct Plan {
    int ntile, nch, ct;
    int64_t wgs;
};
Plan plan_of(int nseq, int rows, int Hk, int page, int max_pages, int type, const KvAttend &a) {
    Plan p;
    const int kb = type == KV_F32 ? KB<float> : KB<__bf16>;
    const int64_t one = type == KV_F32 ? 34 : type == KV_F16 ? 22 : 30;    // a tile, one workgroup a CU
    const int64_t two = type == KV_F32 ? 45 : type == KV_F16 ? 36 : 48;    // two
    const int64_t per = ((int64_t)a.max_new * a.G + RT - 1) / RT;
    const int64_t most = ((int64_t)rows * a.G + RT - 1) / RT + nseq;
    const int64_t ntile = nseq * per < most ? nseq * per : most;
    const int64_t cap = (int64_t)max_pages * page;
    const int64_t keys = a.max_len < cap ? a.max_len : cap;
    int64_t blocks = (keys + kb - 1) / kb;
    if (a.window) {
        // a tile's rows are up to ceil(RT / G) tokens apart; each end of each part may cut a block
        const int64_t toks = (RT + a.G - 1) / a.G + 1;
        const int64_t win = ((int64_t)a.window + toks + kb - 1) / kb + 1, sink = ((int64_t)a.sinks + kb - 1) / kb + 1;
        if (win + sink < blocks) blocks = win + sink;
    }
    if (blocks < 1) blocks = 1;
    const int64_t wgs = ntile * Hk;
    int64_t ct = blocks, best = INT64_MAX;
    for (int64_t n = 1; n == 1 || (n * wgs <= 512 && 2 * n <= blocks + 1); n += 1 + n / 8) {
        const int64_t c = (blocks + n - 1) / n, w = (blocks + c - 1) / c * wgs;
        const int64_t cost = c * (w <= 256 ? one : two) + (c < blocks ? 25 + w * 27 / 200 : 0);
        if (cost < best) best = cost, ct = c;
    }
    p.ntile = ntile < 1 << 30 ? (int)ntile : 1 << 30;
    p.ct = (int)ct;
    p.nch = (int)((blocks + ct - 1) / ct);
    p.wgs = wgs * p.nch;
    return p;
}

}  // namespace

// More rows of a sequence and K/V head than the few-rows form takes in one tile. The whole call takes the
// form of its longest sequence: of 60 single rows on 500 to 100000 keys (32 heads on 8, f16, 855 us) and a part
// of 512 rows (25) in one call, 3060 us. Measured there
// (tiles of 16 side by side) and here: two requests of 30000 keys, 32 heads on 8, f16, 48 rows 115
// and 85 us, 64 of 1000 keys 154 and 81; f32, 16 requests of 2000 keys, 8 heads, 40 rows 113 and 99.
bool mh_kv_prompt(const KvAttend &a) { return (int64_t)a.max_new * a.G > 32; }

int64_t mh_kv_prompt_ws(int nseq, int rows, int Hk, int page, int max_pages, int type, int dk, const KvAttend &a) {
    const Plan p = plan_of(nseq, rows, Hk, page, max_pages, type, a);
    if (p.wgs >= 1 << 24) return -1;   // (a launch holds less than 2^32 threads)
    return p.nch > 1 ? p.wgs * RT * (dk + 2) : 0;
}

hipError_t mh_launch_kv_prompt(const KvTables &t, int type, int dk, const KvAttend &a, float *ws, hipStream_t st) {
    const Plan p = plan_of(t.nseq, t.rows, t.Hk, t.page, t.max_pages, type, a);
    const PromptArgs A{t, a, ws, p.ntile, p.nch, p.ct};
    auto go = [&](auto step, auto join) {
        hipLaunchKernelGGL(step, dim3((unsigned)p.wgs), dim3(NTH), 0, st, A);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess || p.nch <= 1) return e;
        hipLaunchKernelGGL(join, dim3((unsigned)((int64_t)p.ntile * t.Hk), RT / (NTH / (dk / 4))), dim3(NTH), 0, st, A);
        return hipGetLastError();
    };
    if (dk == 128)
        return type == KV_F32 ? go(k_kv_prompt<float, 128>, k_kv_prompt_join<float, 128>)
               : type == KV_F16 ? go(k_kv_prompt<_Float16, 128>, k_kv_prompt_join<_Float16, 128>)
                                : go(k_kv_prompt<__bf16, 128>, k_kv_prompt_join<__bf16, 128>);
    return type == KV_F32 ? go(k_kv_prompt<float, 64>, k_kv_prompt_join<float, 64>)
           : type == KV_F16 ? go(k_kv_prompt<_Float16, 64>, k_kv_prompt_join<_Float16, 64>)
                            : go(k_kv_prompt<__bf16, 64>, k_kv_prompt_join<__bf16, 64>);
}
