// kv_prompt.hip — attention over a paged cache for many new rows of a sequence
// (prompts, and parts of them) on 16-bit caches. The mathematics and the
// visibility of keys are kv_attention.hip's.
//
// One workgroup = four waves = 128 rows of one K/V head (token * G + head), 32 a
// wave, over all the keys they see or one chunk of them; tiles of 64 keys. K and V
// tiles go from the cache's pages to LDS as they lie (global_load_lds, two slots:
// the next tile's copies run while this one's products do), rows swizzled so that
// the 16-byte reads of K and the transposing reads of V meet no bank twice.
//
// Products on the 32x32x16 MFMA of the cache's type (lane l, c = l & 31, hf = l >>
// 5: A row c, B column c, slots 8 hf + j; D rows 8 (e / 4) + 4 hf + e % 4, column c):
//   S^T = K Q^T, O^T = V^T P^T
// so a lane holds the scores of one query row, 32 of a tile's 64 keys, and its
// probabilities are the second product's B operand as they lie (their terms, and q's:
// kv_terms.h; a q row is scaled by a power of two, probabilities stay below 2^14).
// Statistics, in powers of two: a row's reference m follows its maximum only when that
// is 2^6 above it, so the context is seldom rescaled; p = 2^(s - m + 8).
#include <hip/hip_runtime.h>
#include <math.h>

#include "kv.h"
#include "kv_terms.h"
#include "launch.h"
#include "product.h"

namespace {

constexpr int NW = 4, NTH = 64 * NW;
constexpr int RT = 32 * NW;   // rows of a tile
constexpr int KB = 64;        // keys of a tile
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

// The sequence and its row tile that tile number `at` of the call is: tiles are
// numbered sequence by sequence, a sequence's last rows (in causal order the
// longest) first. false: there are fewer. Every thread of the workgroup takes part.
__device__ __forceinline__ bool find_tile(const KvTables &t, const KvAttend &a, int at, int &b, int &rt) {
    __shared__ int sum[NW], hit[2];
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    for (int base = 0, b0 = 0; b0 < t.nseq; b0 += NTH) {
        int n = 0;
        if (b0 + tid < t.nseq) n = (kv_rows(a, kv_seq(t, b0 + tid)) + RT - 1) / RT;
        int x = n;
#pragma unroll
        for (int m = 1; m < 64; m *= 2) {
            const int y = __shfl_up(x, m, 64);
            if (lane >= m) x += y;
        }
        if (lane == 63) sum[w] = x;
        if (tid == 0) hit[0] = -1;
        __syncthreads();
        int before = base + x - n;
        for (int i = 0; i < w; i++) before += sum[i];
        if (at >= before && at < before + n) hit[0] = b0 + tid, hit[1] = n - 1 - (at - before);
        for (int i = 0; i < NW; i++) base += sum[i];
        __syncthreads();
        if (hit[0] >= 0) {
            b = hit[0];
            rt = hit[1];
            return true;
        }
        __syncthreads();
    }
    return false;
}

template <typename T, int DK>
__global__ __launch_bounds__(NTH, 2) void k_kv_prompt(const PromptArgs A) {
    using X = KvTerms<T>;
    typedef typename X::v8 v8;
    constexpr int NT = X::N, KS = DK / 16, DT = DK / 32;
    constexpr int CH = DK / 8;                     // 16-byte pieces of a row
    constexpr int TB = KB * DK * 2;                // bytes of a tile
    constexpr int RPI = 64 / CH;                   // rows of one copy instruction
    __shared__ __attribute__((aligned(16))) uint8_t k0[TB], k1[TB], v0[TB], v1[TB];
    __shared__ __attribute__((aligned(8))) uint16_t valid[2][NW];
    const KvTables &t = A.t;
    const KvAttend &a = A.a;
    const int tid = threadIdx.x, lane = tid & 63, c = lane & 31, hf = lane >> 5;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    int at = blockIdx.x;
    const int h = at % t.Hk;
    at /= t.Hk;
    int b, rt;
    if (!find_tile(t, a, at % A.ntile, b, rt)) return;
    b = __builtin_amdgcn_readfirstlane(b);
    rt = __builtin_amdgcn_readfirstlane(rt);
    const KvTile tl = kv_tile<RT, KB>(t, a, b, rt);
    const int ch = at / A.ntile, nch = max((tl.sp.cnt + A.ct - 1) / A.ct, 1);
    if (ch >= nch) return;
    const int e0 = ch * A.ct, e1 = min(e0 + A.ct, tl.sp.cnt);

    // this lane's row: its keys, and q in terms
    const int r = 32 * w + c, tok = (rt * RT + min(r, tl.live - 1)) / a.G;
    const int head = h * a.G + (rt * RT + min(r, tl.live - 1)) % a.G;
    const int lo = kv_first(a, tl.s, tok), hi = kv_last(t, a, tl.s, tok);
    v8 q[KS][NT];
    float sc;   // what turns a sum of products into a score, in powers of two
    {
        const float *qp = a.q + (int64_t)(tl.s.r0 + tok) * a.ldq + head * DK + 8 * hf;
        const float f = r < tl.live ? a.scale * 1.4426950408889634f : 0.0f;
        float x[KS][8], mx = 0.0f;
#pragma unroll
        for (int s = 0; s < KS; s++) {
            *(f4 *)&x[s][0] = *(const f4 *)(qp + 16 * s);
            *(f4 *)&x[s][4] = *(const f4 *)(qp + 16 * s + 4);
#pragma unroll
            for (int j = 0; j < 8; j++) {
                x[s][j] = r < tl.live ? x[s][j] * f : 0.0f;
                mx = fmaxf(mx, fabsf(x[s][j]));
            }
        }
        mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
        const int e = X::shift(mx);
        sc = ldexpf(1.0f, -e);
#pragma unroll
        for (int s = 0; s < KS; s++) {
#pragma unroll
            for (int j = 0; j < 8; j++) x[s][j] = ldexpf(x[s][j], e);
            X::split(x[s], q[s]);
        }
    }
    f16v o[DT];
#pragma unroll
    for (int d = 0; d < DT; d++) o[d] = zero16();
    float m = -INFINITY, l = 0.0f;

    // A piece of a row lies at its own place with the row's low bits exchanged into it.
    auto swz = [](int row) { return DK == 128 ? row & 15 : (row >> 1) & 7; };
    // Wave w copies rows 16 w .. of a tile; its lanes 0 .. 15 (and again 16 .. ) hold
    // their pages, read from the table a tile ahead and looked at when they are used.
    const int lrow = 16 * w + (lane & 15);
    auto page_of = [&](int e) {
        const int j = min(tl.sp.block(min(e, e1 - 1)) * KB + lrow, tl.hi1);
        return t.pages[(size_t)b * t.max_pages + j / t.page];
    };
    auto copy = [&](int e, int pg, uint8_t *kd, uint8_t *vd, uint16_t *ok) {
        const int j = tl.sp.block(e) * KB + lrow;
        const bool have = j <= tl.hi1 && (unsigned)pg < (unsigned)t.n_pages;
        const uint32_t sl = have ? ((uint32_t)pg * t.Hk + h) * t.page + j % t.page : 0;
        const uint64_t ball = __ballot(have) & 0xffff;
        if (lane == 0) ok[w] = (uint16_t)ball;
#pragma unroll
        for (int i = 0; i < 16 / RPI; i++) {
            const int rr = RPI * i + lane / CH;
            const size_t off = (size_t)(uint32_t)__shfl((int)sl, rr, 64) * (DK * 2) + (((lane % CH) ^ swz(rr)) * 16);
            __builtin_amdgcn_global_load_lds((const glob_void *)((const uint8_t *)t.k + off),
                                             (lds_void *)(kd + (16 * w + RPI * i) * (DK * 2)), 16, 0, 0);
            __builtin_amdgcn_global_load_lds((const glob_void *)((const uint8_t *)t.v + off),
                                             (lds_void *)(vd + (16 * w + RPI * i) * (DK * 2)), 16, 0, 0);
        }
    };
    auto tile = [&](int e, const uint8_t *kt, uint8_t *vt, const uint16_t *ok) {
        // this lane's pieces of a tile (formed anew for each: kept, they would cost registers
        // that the products need)
        int ln = lane;
        asm volatile("" : "+v"(ln));
        const int kbase = (ln & 31) * (DK * 2), kx = (ln >> 5) ^ swz(ln & 31);
        const int vkey = 4 * (ln >> 5) + (ln & 15) / 4, vp = 2 * ((ln >> 4) & 1) + ((ln & 3) >> 1);
        const int j0 = tl.sp.block(e) * KB;
        const uint64_t okw = *(const uint64_t *)ok;
        const bool all = __builtin_amdgcn_readfirstlane(okw == ~0ull && j0 + KB - 1 <= tl.hi0 &&
                                                        (j0 >= tl.lo1 || j0 + KB <= a.sinks));
        // A value that only some rows see meets the others' probability 0, which
        // hides it unless it is not finite: such an element counts as 0 in the
        // product and is added afterwards to the rows that see it.
        int odd = 0;
        if (!all) {
            for (int i = tid; i < TB / 4; i += NTH) {
                uint32_t x = ((uint32_t *)vt)[i];
                const bool bl = kv_odd_lo<T>(x), bh = kv_odd_hi<T>(x);
                if (bl || bh) {
                    odd = 1;
                    x = (bl ? 0 : x & 0xffff) | (bh ? 0 : x & 0xffff0000u);
                    ((uint32_t *)vt)[i] = x;
                }
            }
            odd = __syncthreads_or(odd);
        }
#pragma unroll
        for (int n = 0; n < 2; n++) {
            f16v s = zero16();
#pragma unroll
            for (int u = 0; u < KS; u++) {
                const v8 k = *(const v8 *)(kt + 32 * n * (DK * 2) + kbase + ((2 * u) ^ kx) * 16);
#pragma unroll
                for (int x = 0; x < NT; x++) s = X::mfma32(k, q[u][x], s);
            }
            if (!all) {
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
            mx = fmaxf(mx, __shfl_xor(mx, 32, 64)) * sc;
            const bool up = mx > m + 6.0f;   // (m = -inf: any finite maximum)
            if (__any(up)) {
                const float al = up ? __builtin_amdgcn_exp2f(m - mx) : 1.0f;
                m = up ? mx : m;
                l *= al;
#pragma unroll
                for (int d = 0; d < DT; d++) o[d] *= al;
            }
            const float sub = 8.0f - (m == -INFINITY ? 0.0f : m);
#pragma unroll
            for (int g = 0; g < 2; g++) {
                float p[8];
#pragma unroll
                for (int x = 0; x < 8; x++) {
                    p[x] = __builtin_amdgcn_exp2f(fmaf(s[8 * g + x], sc, sub));
                    l += p[x];
                }
                v8 pt[NT];
                X::split(p, pt);
                // slots 8 hf + x: keys 32 n + 16 g + 4 hf + x (x < 4) and 8 further on
#pragma unroll
                for (int d = 0; d < DT; d++) {
                    s4 v[2];
#pragma unroll
                    for (int y = 0; y < 2; y++) {
                        const int key = 32 * n + 16 * g + 8 * y + vkey;
                        v[y] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                            (lds_s4 *)(vt + key * (DK * 2) + ((4 * d + vp) ^ swz(key)) * 16 + 8 * (ln & 1)));
                    }
                    const v8 vv = __builtin_bit_cast(v8, __builtin_shufflevector(v[0], v[1], 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
                    for (int x = 0; x < NT; x++) o[d] = X::mfma32(vv, pt[x], o[d]);
                }
            }
        }
        if (odd) {
            for (int jj = 0; jj < KB; jj++) {
                const int j = j0 + jj;
                if (!(okw >> jj & 1) || j > hi || (j < lo && j >= a.sinks)) continue;
                const T *vr = (const T *)t.v + (size_t)kv_slot(t, b, j, h) * DK;
#pragma unroll
                for (int d = 0; d < DT; d++)
#pragma unroll
                    for (int x = 0; x < 16; x++) {
                        const float v = (float)vr[32 * d + 8 * (x / 4) + 4 * hf + x % 4];
                        if (!(fabsf(v) < INFINITY)) o[d][x] += v;
                    }
            }
        }
    };

    if (e0 < e1) {
        copy(e0, page_of(e0), k0, v0, valid[0]);
        int pg = page_of(e0 + 1);
        for (int e = e0;; e += 2) {
            __builtin_amdgcn_s_waitcnt(0x0f70);   // vmcnt(0): this wave's copies
            __syncthreads();
            if (e + 1 < e1) copy(e + 1, pg, k1, v1, valid[1]);
            pg = page_of(e + 2);
            tile(e, k0, v0, valid[0]);
            if (e + 1 >= e1) break;
            __builtin_amdgcn_s_waitcnt(0x0f70);
            __syncthreads();
            if (e + 2 < e1) copy(e + 2, pg, k0, v0, valid[0]);
            pg = page_of(e + 3);
            tile(e + 1, k1, v1, valid[1]);
            if (e + 2 >= e1) break;
        }
    }
    l += __shfl_xor(l, 32, 64);
    if (r >= tl.live) return;
    if (nch == 1) {
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        float *op = a.out + (int64_t)(tl.s.r0 + tok) * a.ldo + head * DK + 4 * hf;
#pragma unroll
        for (int d = 0; d < DT; d++)
#pragma unroll
            for (int x = 0; x < 16; x += 4)
                *(f4 *)(op + 32 * d + 2 * x) = f4{o[d][x], o[d][x + 1], o[d][x + 2], o[d][x + 3]} * inv;
        return;
    }
    const size_t slot = (size_t)blockIdx.x * RT + r;
    float *op = A.part + slot * DK + 4 * hf;
#pragma unroll
    for (int d = 0; d < DT; d++)
#pragma unroll
        for (int x = 0; x < 16; x += 4) *(f4 *)(op + 32 * d + 2 * x) = f4{o[d][x], o[d][x + 1], o[d][x + 2], o[d][x + 3]};
    if (hf == 0) {
        float *ml = A.part + (size_t)gridDim.x * RT * DK + 2 * slot;
        ml[0] = m;
        ml[1] = l;
    }
}

// The chunks of a tile's rows, joined in their order, as k_kv_join.
template <int DK>
__global__ __launch_bounds__(NTH) void k_kv_prompt_join(const PromptArgs A) {
    constexpr int LN = DK / 4, RB = NTH / LN;   // lanes of a row, rows of a workgroup
    int at = blockIdx.x;
    const int h = at % A.t.Hk;
    at /= A.t.Hk;
    int b, rt;
    if (!find_tile(A.t, A.a, at, b, rt)) return;
    const KvTile tl = kv_tile<RT, KB>(A.t, A.a, b, rt);
    const int nch = (tl.sp.cnt + A.ct - 1) / A.ct, row = blockIdx.y * RB + threadIdx.x / LN;
    if (nch <= 1 || row >= tl.live) return;
    const int d = 4 * (threadIdx.x % LN);
    const size_t wgs = (size_t)A.t.Hk * A.ntile * A.nch;
    const float *ml = A.part + wgs * RT * DK;
    auto slot = [&](int i) { return (((size_t)i * A.ntile + at) * A.t.Hk + h) * RT + row; };
    float m = -INFINITY;
    for (int i = 0; i < nch; i++) m = fmaxf(m, ml[2 * slot(i)]);
    const float mz = m == -INFINITY ? 0.0f : m;
    f4 o = {0.0f, 0.0f, 0.0f, 0.0f};
    float l = 0.0f;
    for (int i = 0; i < nch; i++) {
        const size_t s = slot(i);
        const float f = exp2f(ml[2 * s] - mz);
        l += f * ml[2 * s + 1];
        o += f * *(const f4 *)(A.part + s * DK + d);
    }
    const int rr = rt * RT + row;
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    *(f4 *)(A.a.out + (int64_t)(tl.s.r0 + rr / A.a.G) * A.a.ldo + (h * A.a.G + rr % A.a.G) * DK + d) = o * inv;
}

// The launch's sizes, from the call's. A tile's keys are split into chunks (of 8
// tiles at least) where its row tiles alone would leave the chip's 512 places
// (two workgroups a CU) empty.
struct Plan {
    int ntile, nch, ct;
    int64_t wgs;
};
Plan plan_of(int nseq, int rows, int Hk, int page, int max_pages, const KvAttend &a) {
    Plan p;
    const int64_t per = ((int64_t)a.max_new * a.G + RT - 1) / RT;
    const int64_t most = ((int64_t)rows * a.G + RT - 1) / RT + nseq;
    const int64_t ntile = nseq * per < most ? nseq * per : most;
    const int64_t cap = (int64_t)max_pages * page;
    const int64_t keys = a.max_len < cap ? a.max_len : cap;
    int64_t blocks = (keys + KB - 1) / KB;
    if (a.window) {
        // a tile's rows are up to ceil(RT / G) tokens apart; each end of each part may cut a block
        const int64_t toks = (RT + a.G - 1) / a.G + 1;
        const int64_t win = ((int64_t)a.window + toks + KB - 1) / KB + 1, sink = ((int64_t)a.sinks + KB - 1) / KB + 1;
        if (win + sink < blocks) blocks = win + sink;
    }
    if (blocks < 1) blocks = 1;
    int64_t split = 512 / (ntile * Hk);
    if (split < 1) split = 1;
    int64_t ct = (blocks + split - 1) / split;
    if (ct < 8) ct = 8;
    p.ntile = ntile < 1 << 30 ? (int)ntile : 1 << 30;
    p.ct = (int)ct;
    p.nch = (int)((blocks + ct - 1) / ct);
    p.wgs = ntile * p.nch * Hk;
    return p;
}

}  // namespace

// Measured crossing of the two forms: see mh_launch_kv_attention.
bool mh_kv_prompt(int type, const KvAttend &a) { return type != KV_F32 && (int64_t)a.max_new * a.G > 64; }

int64_t mh_kv_prompt_ws(int nseq, int rows, int Hk, int page, int max_pages, int dk, const KvAttend &a) {
    const Plan p = plan_of(nseq, rows, Hk, page, max_pages, a);
    if (p.wgs >= 1 << 30) return -1;
    return p.nch > 1 ? p.wgs * RT * (dk + 2) : 0;
}

hipError_t mh_launch_kv_prompt(const KvTables &t, int type, int dk, const KvAttend &a, float *ws, hipStream_t st) {
    const Plan p = plan_of(t.nseq, t.rows, t.Hk, t.page, t.max_pages, a);
    const PromptArgs A{t, a, ws, p.ntile, p.nch, p.ct};
    auto go = [&](auto step, auto join) {
        hipLaunchKernelGGL(step, dim3((unsigned)p.wgs), dim3(NTH), 0, st, A);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess || p.nch <= 1) return e;
        hipLaunchKernelGGL(join, dim3((unsigned)((int64_t)p.ntile * t.Hk), RT / (NTH / (dk / 4))), dim3(NTH), 0, st, A);
        return hipGetLastError();
    };
    if (dk == 128)
        return type == KV_F16 ? go(k_kv_prompt<_Float16, 128>, k_kv_prompt_join<128>)
                              : go(k_kv_prompt<__bf16, 128>, k_kv_prompt_join<128>);
    return type == KV_F16 ? go(k_kv_prompt<_Float16, 64>, k_kv_prompt_join<64>)
                          : go(k_kv_prompt<__bf16, 64>, k_kv_prompt_join<64>);
}
