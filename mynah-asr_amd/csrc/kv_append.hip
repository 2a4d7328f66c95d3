// kv_append.hip — the rows of q, k and v on their way to attention over a paged
// cache: per-head RMS norm and position rotation of q and k, q into its buffer,
// k and v into the cache slots of the rows' positions.
//
//   x' = x / sqrt(mean(x^2) + eps) * w                     (squares summed in 64 bits)
//   pair i at position p: (a cos t - b sin t, a sin t + b cos t), t = p * freq[i]
//
// One row's heads (q heads, then k heads, then v heads) are units of DK / 8
// lanes, eight elements a lane: four pairs, so norm and rotation need nothing
// from another lane but the sum of squares. Pairs (i, i + rot/2): lane t holds
// elements 4t .. 4t+3 and rot/2 + 4t .. ; pairs (2i, 2i + 1), and what is not
// rotated: 8t .. 8t+7. Every access is 16 bytes of f32 or 8 of the cache.
// A workgroup serves one row (or, for few rows, a share of its heads): it finds the
// row's sequence by one search, forms the row's cosines and sines once, in LDS, and
// walks the heads.
// The angle is formed in 64 bits, in turns, and its whole turns dropped there:
// at position 2^17 an f32 product would be off by 2^-7 rad.
//
// What bounds it: memory (12 prompts, 8300 rows of 32 heads on 8 of 128, f16: 83 us, 418 MB
// at 5.0 TB/s; a large copy takes 4.8), for few rows a chain of four round trips, the
// first of which the row's own loads share (256 rows 4.9 us, 4 rows 3.4).
#include <hip/hip_runtime.h>
#include <math.h>

#include "kv.h"
#include "launch.h"
#include "product.h"

namespace {

constexpr int NTH = 256;

// The sequence of a row: how many of row_start[1 .. nseq] are at most `row`.
// A 256-ary search; every thread of the workgroup takes part.
__device__ __forceinline__ int find_seq(const int *row_start, int nseq, int row) {
    int lo = 0, n = nseq;
    while (n > 0) {
        const int step = (n + NTH - 1) / NTH, off = ((int)threadIdx.x + 1) * step;
        const int c = __syncthreads_count(off <= n && row_start[lo + min(off, n)] <= row);
        lo += c * step;
        n = min(step - 1, n - c * step);
    }
    return lo;
}

__device__ __forceinline__ void store4(float *p, f4 x) { *(f4 *)p = x; }
__device__ __forceinline__ void store4(_Float16 *p, f4 x) {
    typedef _Float16 h4 __attribute__((ext_vector_type(4)));
    *(h4 *)p = h4{(_Float16)x[0], (_Float16)x[1], (_Float16)x[2], (_Float16)x[3]};
}
__device__ __forceinline__ void store4(__bf16 *p, f4 x) {
    typedef __bf16 b4 __attribute__((ext_vector_type(4)));
    *(b4 *)p = b4{(__bf16)x[0], (__bf16)x[1], (__bf16)x[2], (__bf16)x[3]};
}

template <typename T, int DK>
__global__ __launch_bounds__(NTH) void k_kv_append(const KvTables t, const KvAppend a) {
    constexpr int TP = DK / 8;          // lanes of a head
    constexpr int UN = NTH / TP;        // heads at a time
    __shared__ float2 cs[DK / 2];
    const int row = blockIdx.x, tid = threadIdx.x, l = tid % TP;
    const bool split = !a.inter && l < a.rot / 8;
    const int e0 = split ? 4 * l : 8 * l, e1 = split ? a.rot / 2 + 4 * l : 8 * l + 4;
    const int units = a.Hq + 2 * t.Hk;
    // what the row's sequence has no part in is on its way before that is known
    f4 x0, x1;
    auto load = [&](int u) {
        const float *x = u < a.Hq ? a.q + row * a.ldq + u * DK
                         : u < a.Hq + t.Hk ? a.k + row * a.ldk + (u - a.Hq) * DK
                                           : a.v + row * a.ldv + (u - a.Hq - t.Hk) * DK;
        x0 = *(const f4 *)(x + e0);
        x1 = *(const f4 *)(x + e1);
    };
    int u = blockIdx.y * UN + tid / TP;
    if (u < units) load(u);
    const double freq = tid < a.rot / 2 ? a.freq[tid] * 0.15915494309189533577 : 0.0;   // turns: 1 / (2 pi)
    const int b = find_seq(t.row_start, t.nseq, row);
    if (b >= t.nseq) return;            // behind the last sequence
    const KvSeq s = kv_seq(t, b);
    if (row < s.r0 || row - s.r0 >= s.n) return;   // (before the first)
    const int p = s.L - s.n + (row - s.r0);
    const bool in_pool = p >= 0 && p / t.page < t.max_pages;
    const uint32_t at0 = in_pool ? kv_slot(t, b, p, 0) : KV_NONE;   // of head 0; a head's slots follow the one before's
    if (tid < a.rot / 2) {
        const double turns = (double)p * freq;
        float sn, c;
        sincospif(2.0f * (float)(turns - rint(turns)), &sn, &c);
        cs[tid] = make_float2(c, sn);
    }
    __syncthreads();
    for (; u < units; u += gridDim.y * UN) {
        const bool isq = u < a.Hq, isv = u >= a.Hq + t.Hk;
        const int h = isq ? u : isv ? u - a.Hq - t.Hk : u - a.Hq;
        const float *w = isv ? nullptr : isq ? a.qn : a.kn;
        if (w) {
            double ss = 0.0;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                ss = fma((double)x0[i], (double)x0[i], ss);
                ss = fma((double)x1[i], (double)x1[i], ss);
            }
#pragma unroll
            for (int m = 1; m < TP; m *= 2) ss += __shfl_xor(ss, m, 64);
            const double rd = rsqrt_d(ss / DK + (double)a.eps);
            // (without eps, the factor of subnormal elements passes f32's range: part of it goes first)
            const float up = rd > 0x1p120 ? 0x1p64f : 1.0f, r = (float)(rd / up);
            const f4 w0 = *(const f4 *)(w + e0), w1 = *(const f4 *)(w + e1);
#pragma unroll
            for (int i = 0; i < 4; i++) x0[i] = x0[i] * up * r * w0[i], x1[i] = x1[i] * up * r * w1[i];
        }
        if (!isv && l < a.rot / 8) {
            // pair i of this lane: (x0[i], x1[i]), or neighbours of x0 and x1
            float pa[4], pb[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float n0 = i < 2 ? x0[2 * i & 3] : x1[2 * i & 3], n1 = i < 2 ? x0[2 * i + 1 & 3] : x1[2 * i + 1 & 3];
                const float va = split ? x0[i] : n0, vb = split ? x1[i] : n1;
                const float2 c = cs[4 * l + i];
                pa[i] = va * c.x - vb * c.y;
                pb[i] = va * c.y + vb * c.x;
            }
            x0 = split ? f4{pa[0], pa[1], pa[2], pa[3]} : f4{pa[0], pb[0], pa[1], pb[1]};
            x1 = split ? f4{pb[0], pb[1], pb[2], pb[3]} : f4{pa[2], pb[2], pa[3], pb[3]};
        }
        if (isq) {
            float *o = a.qo + row * a.ldqo + h * DK;
            *(f4 *)(o + e0) = x0;
            *(f4 *)(o + e1) = x1;
        } else if (at0 != KV_NONE) {
            T *o = (T *)(isv ? t.v : t.k) + ((size_t)at0 + (size_t)h * t.page) * DK;
            store4(o + e0, x0);
            store4(o + e1, x1);
        }
        if (u + (int)gridDim.y * UN < units) load(u + gridDim.y * UN);
    }
}

}  // namespace

hipError_t mh_launch_kv_append(const KvTables &t, int type, int dk, const KvAppend &p, hipStream_t st) {
    const int un = NTH / (dk / 8), passes = (p.Hq + 2 * t.Hk + un - 1) / un;
    // few rows: a workgroup for each pass over the heads, until the chip is full
    int ny = 1;
    while (ny < passes && (int64_t)t.rows * ny < 1024) ny++;
    const dim3 grid(t.rows, ny);
    auto go = [&](auto kern) {
        hipLaunchKernelGGL(kern, grid, dim3(NTH), 0, st, t, p);
        return hipGetLastError();
    };
    if (dk == 128)
        return type == KV_F32 ? go(k_kv_append<float, 128>)
               : type == KV_F16 ? go(k_kv_append<_Float16, 128>) : go(k_kv_append<__bf16, 128>);
    return type == KV_F32 ? go(k_kv_append<float, 64>)
           : type == KV_F16 ? go(k_kv_append<_Float16, 64>) : go(k_kv_append<__bf16, 64>);
}
