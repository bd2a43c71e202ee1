// resnorm.hip — the norms around a block, with its gate and residual scale, in one pass over the rows (gfx950):
//
//     r = x + alpha * g o P(f),      u = Q(r) o (1 + s) + t
//     P(v) = ((v - m1) i1) o w1 + b1  or  v;     Q(v) = ((v - m2) i2) o w2 + b2
//     m = mean over the row's C values (rms norms: 0),   i = 1 / sqrt(mean((v - m)^2) + eps)
//
// g, s, t are vectors for each sample of T rows, or one for all rows; each may be missing, and so may f (then r = x and is not written), P and Q.
// Backward, with n1, n2 the normalised rows, q = n2 o w2 + b2, and the gradients R of r and U of u (either may be missing):
//     dq = U o (1 + s),      D = R + i2 (dq o w2 - mean(dq o w2) - n2 mean(dq o w2 o n2))      [rms: without the plain mean]
//     dx = D,                dp = alpha g o D,      df = i1 (dp o w1 - mean(..) - n1 mean(.. n1))
// All vector gradients follow from FOUR column sums over the rows of a sample,
//     A1 = sum D o n1,  A2 = sum D,  A3 = sum U o n2,  A4 = sum U:
//     dg = alpha (w1 A1 + b1 A2),  ds = w2 A3 + b2 A4,  dt = A4,   and over the samples   dw1 = sum alpha g A1,  db1 = sum alpha g A2,
//     dw2 = sum (1 + s) A3,  db2 = sum (1 + s) A4
// (without P, n1 = f and w1 = 1, b1 = 0).  The backward recomputes the row statistics from x and f, which it has to read anyway: nothing but the
// call's own inputs is kept for it, and r enters it unrounded as in the forward.
//
// Bound: HBM (four tensors of rows forward, six backward; ~20 / 60 operations a value).  A row lives in the registers of TPR threads, 8 values
// each, so it is read once whatever the number of reductions.  What makes it run at the memory's rate:
//   * loads without branches around them: a branch makes the compiler wait for each load at its end (the first form, with a branch for a row's
//     ragged end in every load, took 18.9 us for 8192 x 384 bf16 rows forward).  The last thread's 8 values are the row's LAST 8: they overlap its
//     neighbour's, count once in sums and are written twice with the same value.  Rows past a block's end repeat its last row the same way;
//   * the next row is requested before this one is worked on, and the vectors are folded to four (forward) or three (backward) per chunk of rows:
//     r = x + n1 (g w1) + g b1,   u = n2 (w2 (1 + s)) + (b2 (1 + s) + t);
//   * sums inside a wave on the lane-permute instructions (no LDS), across waves through LDS with ONE barrier: a wave hands over (mean, sum of
//     squares about it), of which every lane then takes one wave's and the same permutes add them up; they combine exactly, so a layer norm needs no second round and no difference of large sums.
// All arithmetic and all sums are fp32; a result is rounded once, when it is written.
#include <hip/hip_runtime.h>
#include <math.h>

#include "cdae.h"
#include "block_common.h"
#include "cdae_internal.h"

namespace {

constexpr int RN_V = 8;                          // values of a row in one thread's registers
constexpr int RN_MAX_C = 8192;                   // 1024 threads x 8
constexpr long RN_MAX_GRID = 1 << 20;            // (a launch holds fewer than 2^32 threads: more rows than this are walked by the same blocks)
constexpr long RN_MAX_BLOCKS = 1 << 22;          // chunks of a backward call: 2^22 x 1024 threads would be the bound itself

constexpr int RN_SUMS = 7;                       // of a sample: g A1, g A2, (1 + s) A3, (1 + s) A4, and the gradients of g, s, t
constexpr int RN_GROUPS = 1024;                  // groups of samples, of 32 at least, that are folded before their sums are written
constexpr long RN_SLAB = 1 << 22;                // column sums (of four) that a backward call keeps at a time: 64 MB, or what half a tensor of its 16-bit rows takes

struct RnArgs {
    cdae_resnorm p;
    int nch, rows_per_chunk;                     // chunks of a sample, rows of a chunk
};

template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
// sum over aligned groups of N lanes, in every lane of the group
template <int N>
__device__ __forceinline__ float lane_sum(float v) {
    v += dpp<0xb1>(v);                                                    // quad_perm 1 0 3 2
    if constexpr (N >= 4) v += dpp<0x4e>(v);                              // quad_perm 2 3 0 1
    if constexpr (N >= 8) v += dpp<0x141>(v);                             // the other quad of 8 lanes (half mirror)
    if constexpr (N >= 16) v += dpp<0x140>(v);                            // the other half of 16 lanes (mirror)
    if constexpr (N >= 32) {
        const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, v), __builtin_bit_cast(unsigned, v), false, false);
        v = __builtin_bit_cast(float, (unsigned)r[0]) + __builtin_bit_cast(float, (unsigned)r[1]);
    }
    if constexpr (N >= 64) {
        const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, v), __builtin_bit_cast(unsigned, v), false, false);
        v = __builtin_bit_cast(float, (unsigned)r[0]) + __builtin_bit_cast(float, (unsigned)r[1]);
    }
    return v;
}

// The sums of a row over its TPR threads.  Across waves: two LDS buffers in turn, so that one barrier separates a sum's writes from its reads and
// the buffer of the sum before last is free again (whoever has passed this barrier has read it).
template <int TPR>
struct RowSum {
    static constexpr int L = TPR < 64 ? TPR : 64, W = TPR / 64;           // (W: waves of a row; a row of up to 64 threads needs no LDS)
    float* sh;
    int turn = 0;
    __device__ explicit RowSum(float* buf) : sh(buf) {}
    template <int NV>
    __device__ __forceinline__ void add(float (&a)[NV]) {
#pragma unroll
        for (int i = 0; i < NV; ++i) a[i] = lane_sum<L>(a[i]);
        if constexpr (W > 1) {
            float* b = sh + (turn ^= 1) * (2 * W);
            if ((threadIdx.x & 63) == 0)
#pragma unroll
                for (int i = 0; i < NV; ++i) b[(threadIdx.x >> 6) * 2 + i] = a[i];
            __syncthreads();
#pragma unroll
            for (int i = 0; i < NV; ++i) a[i] = lane_sum<W>(b[(threadIdx.x & (W - 1)) * 2 + i]);
        }
    }
    // n = the normalised row, -> 1 / sqrt(mean square + eps)
    __device__ __forceinline__ float normalise(const float (&v)[RN_V], float (&n)[RN_V], int skip, int end, int C, int layer, float inv_c, float eps) {
        float m = 0.f, q[1] = {0.f};
        if (!layer) {
#pragma unroll
            for (int e = 0; e < RN_V; ++e) q[0] += e >= skip && e < end ? v[e] * v[e] : 0.f;
            add<1>(q);
        } else {
            float s = 0.f;
#pragma unroll
            for (int e = 0; e < RN_V; ++e) s += e >= skip && e < end ? v[e] : 0.f;
            if constexpr (W <= 1) {
                m = lane_sum<L>(s) * inv_c;
#pragma unroll
                for (int e = 0; e < RN_V; ++e) { const float d = v[e] - m; q[0] += e >= skip && e < end ? d * d : 0.f; }
                q[0] = lane_sum<L>(q[0]);
            } else {
                const int wave = threadIdx.x >> 6;
                auto count = [&](int w) { const int k = C - w * 64 * RN_V; return (float)(k < 0 ? 0 : k < 64 * RN_V ? k : 64 * RN_V); };
                const float mine = count(wave);
                const float mw = mine > 0.f ? lane_sum<64>(s) / mine : 0.f;
#pragma unroll
                for (int e = 0; e < RN_V; ++e) { const float d = v[e] - mw; q[0] += e >= skip && e < end ? d * d : 0.f; }
                q[0] = lane_sum<64>(q[0]);
                float* b = sh + (turn ^= 1) * (2 * W);
                if ((threadIdx.x & 63) == 0) { b[wave * 2] = mw; b[wave * 2 + 1] = q[0]; }
                __syncthreads();
                const int w = threadIdx.x & (W - 1);
                const float its = count(w), itsm = b[2 * w];
                m = lane_sum<W>(its * itsm) * inv_c;
                const float d = itsm - m;
                q[0] = lane_sum<W>(fmaf(its * d, d, b[2 * w + 1]));
            }
        }
        const float i = 1.f / sqrtf(q[0] * inv_c + eps);
#pragma unroll
        for (int e = 0; e < RN_V; ++e) n[e] = (v[e] - m) * i;
        return i;
    }
};

// A thread's 8 columns.  Rows of 8 values and more: columns c0 .. c0 + 7 with c0 at most C - 8, of which the first `skip` belong to the thread
// before (skip >= 8: all; such a thread repeats the last 8).  Shorter rows (SMALL): one thread's, with C values; the other threads repeat them.
template <bool SMALL>
struct Cols {
    int c0, skip, end, C;                        // (the thread's own values: [skip, end) of its 8)
    __device__ Cols(int lane, int C_) : C(C_) {
        const int want = lane * RN_V;
        c0 = SMALL ? 0 : want < C - RN_V ? want : C - RN_V;
        skip = SMALL ? (lane ? RN_V : 0) : want - c0;
        end = SMALL ? C : RN_V;
    }
    template <class T>
    __device__ __forceinline__ Pack<T, RN_V> raw(const T* __restrict__ p) const {
        if constexpr (SMALL) {
            Pack<T, RN_V> v;
#pragma unroll
            for (int e = 0; e < RN_V; ++e) v.v[e] = p[e < C ? e : C - 1];
            return v;
        } else {
            return *reinterpret_cast<const Pack<T, RN_V>*>(p + c0);
        }
    }
    template <class T>
    __device__ __forceinline__ void put(T* __restrict__ p, const float (&v)[RN_V]) const {
        if constexpr (SMALL) {
#pragma unroll
            for (int e = 0; e < RN_V; ++e) if (e < C) st1(p[e], v[e]);
        } else {
            stv<T, RN_V>(p + c0, v);
        }
    }
    template <class T>
    __device__ __forceinline__ void vec(const void* p, long off, int is32, float (&o)[RN_V]) const {
        if (is32) open(raw(reinterpret_cast<const float*>(p) + off), o);
        else open(raw(reinterpret_cast<const T*>(p) + off), o);
    }
    // values that are absent read as zero (SMALL) or count elsewhere (skip)
    template <class T>
    __device__ __forceinline__ void open(const Pack<T, RN_V>& r, float (&o)[RN_V]) const {
#pragma unroll
        for (int e = 0; e < RN_V; ++e) o[e] = SMALL && e >= C ? 0.f : ld1(r.v[e]);
    }
};

// the vectors folded: r = x + n1 gw + gb,  u = n2 sw + sb
template <class T, bool SMALL>
__device__ __forceinline__ void fold_cols(const cdae_resnorm& p, long b, const Cols<SMALL>& k, float (&gw)[RN_V], float (&gb)[RN_V], float (&sw)[RN_V], float (&sb)[RN_V]) {
    float t[RN_V];
#pragma unroll
    for (int e = 0; e < RN_V; ++e) { gw[e] = p.alpha; gb[e] = 0.f; sw[e] = 1.f; sb[e] = 0.f; }
    if (p.gate) {
        k.template vec<T>(p.gate, p.shared_gate ? 0 : b * p.ld_gate, p.vec32, t);
#pragma unroll
        for (int e = 0; e < RN_V; ++e) gw[e] *= t[e];
    }
    if (p.b1) {
        k.template vec<T>(p.b1, 0, p.w32, t);
#pragma unroll
        for (int e = 0; e < RN_V; ++e) gb[e] = gw[e] * t[e];
    }
    if (p.w1) {
        k.template vec<T>(p.w1, 0, p.w32, t);
#pragma unroll
        for (int e = 0; e < RN_V; ++e) gw[e] *= t[e];
    }
    if (p.scale) {
        k.template vec<T>(p.scale, p.shared_scale ? 0 : b * p.ld_scale, p.vec32, t);
#pragma unroll
        for (int e = 0; e < RN_V; ++e) sw[e] += t[e];
    }
    if (p.b2) {
        k.template vec<T>(p.b2, 0, p.w32, t);
#pragma unroll
        for (int e = 0; e < RN_V; ++e) sb[e] = sw[e] * t[e];
    }
    if (p.w2) {
        k.template vec<T>(p.w2, 0, p.w32, t);
#pragma unroll
        for (int e = 0; e < RN_V; ++e) sw[e] *= t[e];
    }
    if (p.shift) {
        k.template vec<T>(p.shift, p.shared_shift ? 0 : b * p.ld_shift, p.vec32, t);
#pragma unroll
        for (int e = 0; e < RN_V; ++e) sb[e] += t[e];
    }
}

// threads of a block: four waves of rows that need no LDS, or one row
constexpr int block_of(int tpr) { return tpr <= 64 ? 256 : tpr; }

// A group of TPR threads walks one chunk of a sample's rows.
template <class T, int TPR, bool SMALL>
__global__ __launch_bounds__(block_of(TPR)) void rn_fwd_kernel(const RnArgs a) {
    constexpr int GROUPS = block_of(TPR) / TPR;
    __shared__ float sh[TPR > 64 ? 4 * (TPR / 64) : 1];
    const cdae_resnorm& p = a.p;
    const Cols<SMALL> k(threadIdx.x & (TPR - 1), p.C);
    const float inv_c = 1.f / (float)p.C;
    const long chunks = (long)p.B * a.nch;
    RowSum<TPR> rows(sh);                        // (one for all chunks: the buffers have to go on taking turns where a chunk holds an odd number of sums)
    for (long c = (long)blockIdx.x * GROUPS + threadIdx.x / TPR; c < chunks; c += (long)gridDim.x * GROUPS) {      // (one group a block where there are barriers)
        const long b = c / a.nch;
        const int t0 = (int)(c - b * a.nch) * a.rows_per_chunk, t1 = t0 + a.rows_per_chunk < p.T ? t0 + a.rows_per_chunk : p.T;
        float gw[RN_V], gb[RN_V], sw[RN_V], sb[RN_V];
        const T* X = reinterpret_cast<const T*>(p.x) + (b * p.T) * p.ld_x;
        const T* F = reinterpret_cast<const T*>(p.f);
        if (F) F += b * p.T * p.ld_f;
        const long out = b * p.T * p.C;
        Pack<T, RN_V> xr = k.raw(X + t0 * p.ld_x), fr = k.raw(F ? F + t0 * p.ld_f : X + t0 * p.ld_x);
        fold_cols<T, SMALL>(p, b, k, gw, gb, sw, sb);
        for (int t = t0; t < t1; ++t) {
            const int next = t + 1 < t1 ? t + 1 : t;
            float r[RN_V], n[RN_V];
            k.open(xr, r);
            k.open(fr, n);
            xr = k.raw(X + next * p.ld_x);
            if (F) {
                fr = k.raw(F + next * p.ld_f);
                if (p.post) {
                    float f[RN_V];
#pragma unroll
                    for (int e = 0; e < RN_V; ++e) f[e] = n[e];
                    rows.normalise(f, n, k.skip, k.end, p.C, p.layer, inv_c, p.eps);
                }
#pragma unroll
                for (int e = 0; e < RN_V; ++e) r[e] = fmaf(n[e], gw[e], r[e]) + gb[e];
                k.put(reinterpret_cast<T*>(p.r) + out + (long)t * p.C, r);
            }
            if (p.pre) {
                rows.normalise(r, n, k.skip, k.end, p.C, p.layer, inv_c, p.eps);
#pragma unroll
                for (int e = 0; e < RN_V; ++e) n[e] = fmaf(n[e], sw[e], sb[e]);
                k.put(reinterpret_cast<T*>(p.u) + out + (long)t * p.C, n);
            }
        }
    }
}

// One block: rows [t0, t1) of one sample, its groups of TPR threads in turn.  Leaves dx, df, and the four column sums of its rows in part[chunk][4][C].
template <class T, int TPR, bool SMALL>
__global__ __launch_bounds__(block_of(TPR)) void rn_bwd_kernel(const RnArgs a) {
    constexpr int BLOCK = block_of(TPR), GROUPS = BLOCK / TPR;
    __shared__ float sh[TPR > 64 ? 4 * (TPR / 64) : 1];
    __shared__ float cols[GROUPS > 1 ? GROUPS * TPR * RN_V : 1];
    // rows of 1024 threads: a thread has 128 registers, and its three vectors (24) lie in LDS, each thread its own (2 x 1024 rows of 8192 bf16: 62 us;
    // with the vectors in registers and scratch 74)
    constexpr bool IN_LDS = TPR == 1024;
    __shared__ float4 vecs[IN_LDS ? 6 * TPR : 1];
    const cdae_resnorm& p = a.p;
    const int lane = threadIdx.x & (TPR - 1), grp = threadIdx.x / TPR;
    const Cols<SMALL> k(lane, p.C);
    RowSum<TPR> rows(sh);
    const float inv_c = 1.f / (float)p.C;
    const long b = blockIdx.x / a.nch;
    const int ch = blockIdx.x - (int)b * a.nch;
    const int t0 = ch * a.rows_per_chunk, t1 = t0 + a.rows_per_chunk < p.T ? t0 + a.rows_per_chunk : p.T;
    const T* X = reinterpret_cast<const T*>(p.x) + b * p.T * p.ld_x;
    const T* F = reinterpret_cast<const T*>(p.f);
    const T* R = reinterpret_cast<const T*>(p.dr);
    const T* U = reinterpret_cast<const T*>(p.du);
    if (F) F += b * p.T * p.ld_f;
    if (R) R += b * p.T * p.ld_dr;
    if (U) U += b * p.T * p.ld_du;
    const long out = b * p.T * p.C;
    // (a tensor that is absent is read as x and not used)
    const T* const Fs = F ? F : X; const T* const Rs = R ? R : X; const T* const Us = U ? U : X;
    const long lf = F ? p.ld_f : p.ld_x, lr = R ? p.ld_dr : p.ld_x, lu = U ? p.ld_du : p.ld_x;
    auto row_of = [&](int t) { return t + grp < t1 ? t + grp : t1 - 1; };
    int t = row_of(t0);
    constexpr bool AHEAD = TPR < 1024 || sizeof(T) == 2;          // (1024 threads of fp32 rows have no registers left for the next row: 115 us, with it 128)
    Pack<T, RN_V> xr = k.raw(X + t * p.ld_x), fr = k.raw(Fs + t * lf), rr = k.raw(Rs + t * lr), ur = k.raw(Us + t * lu);
    float gw[RN_V], gb[RN_V], sw[RN_V], sb[RN_V];
    fold_cols<T, SMALL>(p, b, k, gw, gb, sw, sb);
    if constexpr (IN_LDS)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            vecs[h * TPR + lane] = {gw[4 * h], gw[4 * h + 1], gw[4 * h + 2], gw[4 * h + 3]};
            vecs[(2 + h) * TPR + lane] = {gb[4 * h], gb[4 * h + 1], gb[4 * h + 2], gb[4 * h + 3]};
            vecs[(4 + h) * TPR + lane] = {sw[4 * h], sw[4 * h + 1], sw[4 * h + 2], sw[4 * h + 3]};
        }
    auto again = [&](int j, float (&v)[RN_V]) {
        if constexpr (IN_LDS)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const float4 q = vecs[(2 * j + h) * TPR + lane];
                v[4 * h] = q.x; v[4 * h + 1] = q.y; v[4 * h + 2] = q.z; v[4 * h + 3] = q.w;
            }
    };
    float A[4][RN_V];
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int e = 0; e < RN_V; ++e) A[j][e] = 0.f;
    for (int tb = t0; tb < t1; tb += GROUPS) {                    // (the trip count is the block's: its barriers are met by every thread)
        const float live = tb + grp < t1 ? 1.f : 0.f;
        t = row_of(tb);
        const int next = row_of(tb + GROUPS < t1 ? tb + GROUPS : tb);
        float r[RN_V], n1[RN_V], n2[RN_V], D[RN_V], h[RN_V];
        if (!AHEAD) { xr = k.raw(X + t * p.ld_x); fr = k.raw(Fs + t * lf); rr = k.raw(Rs + t * lr); ur = k.raw(Us + t * lu); }
        k.open(xr, r);
        k.open(fr, n1);
        k.open(rr, D);
        k.open(ur, h);
        if (AHEAD) { xr = k.raw(X + next * p.ld_x); fr = k.raw(Fs + next * lf); rr = k.raw(Rs + next * lr); ur = k.raw(Us + next * lu); }
        float i1 = 1.f;
        if (!R)
#pragma unroll
            for (int e = 0; e < RN_V; ++e) D[e] = 0.f;
        if (F) {
            if (p.post) {
                float f[RN_V];
#pragma unroll
                for (int e = 0; e < RN_V; ++e) f[e] = n1[e];
                i1 = rows.normalise(f, n1, k.skip, k.end, p.C, p.layer, inv_c, p.eps);
            }
            again(0, gw);
            again(1, gb);
#pragma unroll
            for (int e = 0; e < RN_V; ++e) r[e] = fmaf(n1[e], gw[e], r[e]) + gb[e];
        }
        if (U) {
            const float i2 = rows.normalise(r, n2, k.skip, k.end, p.C, p.layer, inv_c, p.eps);
            float s[2] = {0.f, 0.f};
            again(2, sw);
#pragma unroll
            for (int e = 0; e < RN_V; ++e) {
                A[2][e] = fmaf(live * h[e], n2[e], A[2][e]);
                A[3][e] = fmaf(live, h[e], A[3][e]);
                h[e] *= sw[e];
                if (e >= k.skip && e < k.end) { s[0] = fmaf(h[e], n2[e], s[0]); s[1] += h[e]; }
            }
            rows.add(s);
            const float m1 = s[0] * inv_c, m0 = p.layer ? s[1] * inv_c : 0.f;
#pragma unroll
            for (int e = 0; e < RN_V; ++e) D[e] = fmaf(i2, h[e] - m0 - n2[e] * m1, D[e]);
        }
        if (p.dx) k.put(reinterpret_cast<T*>(p.dx) + out + (long)t * p.C, D);
        if (F) {
            float s[2] = {0.f, 0.f};
            again(0, gw);
#pragma unroll
            for (int e = 0; e < RN_V; ++e) {
                A[0][e] = fmaf(live * D[e], n1[e], A[0][e]);
                A[1][e] = fmaf(live, D[e], A[1][e]);
                D[e] *= gw[e];
                if (e >= k.skip && e < k.end) { s[0] = fmaf(D[e], n1[e], s[0]); s[1] += D[e]; }
            }
            if (p.df) {
                if (p.post) {
                    rows.add(s);
                    const float m1 = s[0] * inv_c, m0 = p.layer ? s[1] * inv_c : 0.f;
#pragma unroll
                    for (int e = 0; e < RN_V; ++e) D[e] = i1 * (D[e] - m0 - n1[e] * m1);
                }
                k.put(reinterpret_cast<T*>(p.df) + out + (long)t * p.C, D);
            }
        }
    }
    if (!p.ws) return;                                            // (no vector has a gradient)
    float* part = p.ws + (long)blockIdx.x * 4 * p.C;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if constexpr (GROUPS > 1) {                               // the block's groups, added in a fixed order
            __syncthreads();
#pragma unroll
            for (int e = 0; e < RN_V; ++e) if (SMALL ? e < p.C && !lane : true) cols[grp * TPR * RN_V + k.c0 + e] = A[j][e];
            __syncthreads();
            for (int c = threadIdx.x; c < p.C; c += BLOCK) {
                float s = 0.f;
#pragma unroll 4
                for (int g = 0; g < GROUPS; ++g) s += cols[g * TPR * RN_V + c];
                part[j * p.C + c] = s;
            }
        } else {
            k.put(part + j * p.C, A[j]);
        }
    }
}

// Gradients of a sample's own gate, scale and shift in column c from its column sums, written; o: what it gives to the sums that samples share
template <class T>
__device__ __forceinline__ void fold_sample(const cdae_resnorm& p, long b, int c, float w1, float b1, float w2, float b2, const float (&A)[4], float (&o)[RN_SUMS]) {
    auto vec = [&](const void* v, long off, float none) { return !v ? none : p.vec32 ? ((const float*)v)[off] : ld1(((const T*)v)[off]); };
    const float g = vec(p.gate, (p.shared_gate ? 0 : b * p.ld_gate) + c, 1.f) * p.alpha, s1 = 1.f + vec(p.scale, (p.shared_scale ? 0 : b * p.ld_scale) + c, 0.f);
    const float dg = p.alpha * (w1 * A[0] + b1 * A[1]), ds = w2 * A[2] + b2 * A[3];
    if (p.dgate && !p.shared_gate) st2<T>(p.dgate, b * p.C + c, p.vec32, dg);
    if (p.dscale && !p.shared_scale) st2<T>(p.dscale, b * p.C + c, p.vec32, ds);
    if (p.dshift && !p.shared_shift) st2<T>(p.dshift, b * p.C + c, p.vec32, A[3]);
    o[0] = g * A[0]; o[1] = g * A[1]; o[2] = s1 * A[2]; o[3] = s1 * A[3]; o[4] = dg; o[5] = ds; o[6] = A[3];
}
template <class T>
__device__ __forceinline__ float weight_of(const cdae_resnorm& p, const void* v, int c, float none) { return !v ? none : p.w32 ? ((const float*)v)[c] : ld1(((const T*)v)[c]); }
// where sum j of all samples belongs, or NULL
__device__ __forceinline__ void* shared_of(const cdae_resnorm& p, int j) {
    void* const dst[RN_SUMS] = {p.dw1, p.db1, p.dw2, p.db2, p.shared_gate ? p.dgate : nullptr, p.shared_scale ? p.dscale : nullptr, p.shared_shift ? p.dshift : nullptr};
    void* out = nullptr;
#pragma unroll
    for (int i = 0; i < RN_SUMS; ++i) if (i == j) out = dst[i];
    return out;
}

// The column sums of each sample from its chunks, and from them the gradients of gate, scale and shift; what the samples
// share goes to sums[b][7][C], or for a single sample to the results themselves (a launch less: 30000 rows of 600 fp16, all of the backward, 93 and 91 us).
// A block: 32 columns (one line of a chunk's row) x 32 lanes of chunks (16 x 64 leave fewer CUs idle in front of narrow rows and cost wider ones as much).
template <class T>
__global__ __launch_bounds__(1024) void rn_fold_kernel(const RnArgs a, float* __restrict__ sums) {
    const cdae_resnorm& p = a.p;
    const int ncb = (p.C + 31) / 32, cl = threadIdx.x & 31, q = threadIdx.x >> 5;
    __shared__ float sh[4][32][33];
    for (long job = blockIdx.x; job < (long)p.B * ncb; job += gridDim.x) {        // (the block's: its barriers are met by every thread)
        const long b = job / ncb;
        const int c = (int)(job - b * ncb) * 32 + cl;
        float A[4] = {0.f, 0.f, 0.f, 0.f};
        const float* part = p.ws + b * a.nch * 4 * p.C + (c < p.C ? c : p.C - 1);
#pragma unroll 4
        for (int ch = q; ch < a.nch; ch += 32) {
#pragma unroll
            for (int j = 0; j < 4; ++j) A[j] += part[((long)ch * 4 + j) * p.C];
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 4; ++j) sh[j][q][cl] = A[j];
        __syncthreads();
        if (q < 4) {                                                      // the threads of q add sum q, in order
            float s = 0.f;
#pragma unroll
            for (int i = 0; i < 32; ++i) s += sh[q][i][cl];
            sh[q][0][cl] = s;
        }
        __syncthreads();
        if (q || c >= p.C) continue;
#pragma unroll
        for (int j = 0; j < 4; ++j) A[j] = sh[j][0][cl];
        float o[RN_SUMS];
        fold_sample<T>(p, b, c, weight_of<T>(p, p.w1, c, 1.f), weight_of<T>(p, p.b1, c, 0.f), weight_of<T>(p, p.w2, c, 1.f), weight_of<T>(p, p.b2, c, 0.f), A, o);
#pragma unroll
        for (int j = 0; j < RN_SUMS; ++j) {
            if (p.B > 1) sums[(b * RN_SUMS + j) * p.C + c] = o[j];
            else if (void* const out = shared_of(p, j)) st2<T>(out, c, j < 4 ? p.w32 : p.vec32, o[j]);
        }
    }
}

// The same for samples of one chunk each, `per_group` to a block of 32 columns x 32 lanes of samples: what they share is added up before it is written, to
// sums[group][7][C] or, for a single group, to the results themselves.  (A whole backward of 2000 x 64 rows of 512 bf16: 181 us; with a block for each sample, 31 of
// its 32 lanes without a chunk, 377.  5000 single rows of 24: 48, bound by the host, and 126.)
template <class T>
__global__ __launch_bounds__(1024) void rn_fold_samples_kernel(const RnArgs a, float* __restrict__ sums, int per_group, int single) {
    const cdae_resnorm& p = a.p;
    const int ncb = (p.C + 31) / 32, cl = threadIdx.x & 31, q = threadIdx.x >> 5, group = blockIdx.x / ncb, c = (blockIdx.x - group * ncb) * 32 + cl;
    __shared__ float sh[RN_SUMS][32][33];
    float total[RN_SUMS] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (c < p.C) {
        const float w1 = weight_of<T>(p, p.w1, c, 1.f), b1 = weight_of<T>(p, p.b1, c, 0.f), w2 = weight_of<T>(p, p.w2, c, 1.f), b2 = weight_of<T>(p, p.b2, c, 0.f);
        const int first = group * per_group, end = first + per_group < p.B ? first + per_group : p.B;
        for (int b = first + q; b < end; b += 32) {
            float A[4], o[RN_SUMS];
#pragma unroll
            for (int j = 0; j < 4; ++j) A[j] = p.ws[((long)b * 4 + j) * p.C + c];
            fold_sample<T>(p, b, c, w1, b1, w2, b2, A, o);
#pragma unroll
            for (int j = 0; j < RN_SUMS; ++j) total[j] += o[j];
        }
    }
#pragma unroll
    for (int j = 0; j < RN_SUMS; ++j) sh[j][q][cl] = total[j];
    __syncthreads();
    if (q >= RN_SUMS || c >= p.C) return;                                 // the threads of q add sum q, in order
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 32; ++i) s += sh[q][i][cl];
    if (!single) sums[((long)group * RN_SUMS + q) * p.C + c] = s;
    else if (void* const out = shared_of(p, q)) st2<T>(out, c, q < 4 ? p.w32 : p.vec32, s);
}

// what all samples share: grid y picks one of the seven sums; 32 columns x 8 lanes of samples or groups of them
template <class T>
__global__ __launch_bounds__(256) void rn_shared_kernel(const cdae_resnorm p, const float* __restrict__ sums, int count) {
    const int cl = threadIdx.x & 31, q = threadIdx.x >> 5, c = blockIdx.x * 32 + cl, j = blockIdx.y;
    __shared__ float sh[8][32];
    void* const out = shared_of(p, j);
    if (!out) return;                                                     // (block-uniform)
    float s = 0.f;
    const float* at = sums + (long)j * p.C + (c < p.C ? c : p.C - 1);
#pragma unroll 4
    for (int b = q; b < count; b += 8) s += at[(long)b * RN_SUMS * p.C];
    sh[q][cl] = s;
    __syncthreads();
    if (q || c >= p.C) return;
#pragma unroll
    for (int i = 1; i < 8; ++i) s += sh[i][cl];
    st2<T>(out, c, j < 4 ? p.w32 : p.vec32, s);
}

int threads_per_row(int C) {
    int t = 1;
    while (t * RN_V < C) t *= 2;
    return t < 8 ? 8 : t;
}

// Backward: chunks of a sample, a multiple of the block's groups of rows each, for as many blocks in all as run at once at 140 to 160 registers a thread,
// and not one more (30 x 1000 rows of 512 fp16: 53 us for 510 blocks, 61 for 540): more blocks leave more partial sums.  Two blocks of 256 threads a CU (8 x 4096
// rows of 2048 bf16: 179 us; 256 blocks 234, 768 blocks 187), one of 512 and more (4 x 2048 rows of 4096: 100 us; two 108), and of blocks of 128 threads
// six, or four on fp32 rows (30000 rows of 600 fp16: 93 us; 1024 blocks 100, 512 blocks 156; 11 x 1700 of 700 fp32: 81; 1536 blocks 85, 512 blocks 96).
void chunks_of(int B, int T, int C, bool wide, int& nch, int& rows) {
    const int tpr = threads_per_row(C), groups = block_of(tpr) / tpr, at_once = tpr >= 512 ? 256 : tpr == 128 ? (wide ? 1024 : 1536) : 512;
    const int want = B < at_once ? at_once / B : 1;
    rows = (T + want - 1) / want;
    rows = (rows + groups - 1) / groups * groups;
    nch = (T + rows - 1) / rows;
}
// Forward: a group's rows, so that the 16 waves a CU that run at once take them all (4 x 2000 rows of 4000 fp16: 58 us, and 75 where a few blocks are left
// for a second round), up to 16 rows; where that takes more rounds, 8 rows each for an even end (8 x 4096 rows of 2048 bf16: 103 us; 16 rows 110), and 16 of
// the widest rows (8000 rows of 8000 fp16: 116 us; 8 rows 121).
void fwd_chunks(int B, int T, int C, int& nch, int& rows) {
    const long tpr = threads_per_row(C), r = ((long)B * T * tpr / 64 + 4095) / 4096;
    rows = r < 1 ? 1 : r <= 16 ? (int)r : tpr == 1024 ? 16 : 8;
    nch = (T + rows - 1) / rows;
}

int check(const cdae_resnorm* p) {
    if (!p || p->B <= 0 || p->T <= 0 || p->C <= 0 || p->C > RN_MAX_C) return cdae_fail("resnorm: B, T >= 1 and 1 <= C <= 8192 required");
    if ((long)p->B * p->T > 1L << 30) return cdae_fail("resnorm: at most 2^30 rows");
    if (p->dt < 0 || p->dt > 2) return cdae_fail("resnorm: row type 0 (bf16), 1 (fp16) or 2 (fp32)");
    if (!p->x || (!p->f && !p->pre)) return cdae_fail("resnorm: x and a block output or a pre norm required");
    if (!p->f && (p->post || p->gate)) return cdae_fail("resnorm: a post norm or a gate needs a block output");
    if (!p->pre && (p->w2 || p->b2 || p->scale || p->shift)) return cdae_fail("resnorm: w2, b2, scale and shift belong to a pre norm");
    if (!p->post && (p->w1 || p->b1)) return cdae_fail("resnorm: w1 and b1 belong to a post norm");
    if (!(p->eps >= 0.f)) return cdae_fail("resnorm: eps must be >= 0");
    return 0;
}

#define RN_TPR(CALL)                                    \
    if (p->C < RN_V) { CALL(8, true); }                 \
    else switch (threads_per_row(p->C)) {               \
        case 8: { CALL(8, false); break; }              \
        case 16: { CALL(16, false); break; }            \
        case 32: { CALL(32, false); break; }            \
        case 64: { CALL(64, false); break; }            \
        case 128: { CALL(128, false); break; }          \
        case 256: { CALL(256, false); break; }          \
        case 512: { CALL(512, false); break; }          \
        default: { CALL(1024, false); break; }          \
    }

template <class T>
void fwd(const cdae_resnorm* p, hipStream_t st) {
    RnArgs a;
    a.p = *p;
    fwd_chunks(p->B, p->T, p->C, a.nch, a.rows_per_chunk);
    const long chunks = (long)p->B * a.nch;
#define RN_CALL(N, S) { constexpr int G = block_of(N) / N; const long g = (chunks + G - 1) / G; \
                        hipLaunchKernelGGL((rn_fwd_kernel<T, N, S>), dim3((unsigned)(g < RN_MAX_GRID ? g : RN_MAX_GRID)), dim3(block_of(N)), 0, st, a); }
    RN_TPR(RN_CALL)
#undef RN_CALL
}
bool any_vector(const cdae_resnorm* p) { return p->dgate || p->dscale || p->dshift || p->dw1 || p->db1 || p->dw2 || p->db2; }
bool any_shared(const cdae_resnorm* p) {
    return p->dw1 || p->db1 || p->dw2 || p->db2 || (p->dgate && p->shared_gate) || (p->dscale && p->shared_scale) || (p->dshift && p->shared_shift);
}
// Samples of a group, and samples of a slab: with few rows a sample the four column sums of every sample would be a multiple of the rows themselves (16 bytes
// a value beside 2), so that such calls go over the samples in slabs, which share one place for them.  More than one slab means one chunk a sample.
// 65536 single rows of 1024 bf16: 1.0 ms in 16 slabs; with all sums kept, 3.0 GB, and a block for each sample's fold 17.6 ms.
int group_of(int B) { return 32 * (int)((B + 32L * RN_GROUPS - 1) / (32L * RN_GROUPS)); }
int slab_of(int B, int T, int C) {
    const long rows = (long)B * T * C / 16, most = (rows > RN_SLAB ? rows : RN_SLAB) / C, per = group_of(B);
    return most >= B ? B : (int)(most < per ? per : most / per * per);
}
size_t sums_at(int B, int T, int C, int nch) { return 4 * (size_t)C * (nch > 1 ? (size_t)B * nch : (size_t)slab_of(B, T, C)); }      // (floats in front of the shared sums)
size_t scratch_floats(int B, int T, int C, int nch) {
    return sums_at(B, T, C, nch) + RN_SUMS * (size_t)C * (nch > 1 ? B : (B + group_of(B) - 1) / group_of(B));
}

// samples from `first` on, `count` of them
template <class T>
cdae_resnorm part_of(const cdae_resnorm& whole, long first, int count) {
    cdae_resnorm p = whole;
    const long t = first * p.T, vec = p.vec32 ? 4 : sizeof(T);
    auto in = [](const void*& v, long by) { if (v) v = (const char*)v + by; };
    auto out = [](void*& v, long by) { if (v) v = (char*)v + by; };
    p.B = count;
    in(p.x, t * p.ld_x * sizeof(T)); in(p.f, t * p.ld_f * sizeof(T)); in(p.dr, t * p.ld_dr * sizeof(T)); in(p.du, t * p.ld_du * sizeof(T));
    out(p.dx, t * p.C * sizeof(T)); out(p.df, t * p.C * sizeof(T));
    if (!p.shared_gate) { in(p.gate, first * p.ld_gate * vec); out(p.dgate, first * p.C * vec); }
    if (!p.shared_scale) { in(p.scale, first * p.ld_scale * vec); out(p.dscale, first * p.C * vec); }
    if (!p.shared_shift) { in(p.shift, first * p.ld_shift * vec); out(p.dshift, first * p.C * vec); }
    return p;
}
template <class T>
void bwd_rows(const RnArgs& a, hipStream_t st) {
    const cdae_resnorm* p = &a.p;
#define RN_CALL(N, S) hipLaunchKernelGGL((rn_bwd_kernel<T, N, S>), dim3((unsigned)((long)p->B * a.nch)), dim3(block_of(N)), 0, st, a)
    RN_TPR(RN_CALL)
#undef RN_CALL
}
template <class T>
void bwd(const cdae_resnorm* p, hipStream_t st) {
    RnArgs a;
    a.p = *p;
    chunks_of(p->B, p->T, p->C, sizeof(T) == 4, a.nch, a.rows_per_chunk);
    if (!any_vector(p)) {
        a.p.ws = nullptr;
        return bwd_rows<T>(a, st);
    }
    float* const sums = p->ws + sums_at(p->B, p->T, p->C, a.nch);
    const int ncb = (p->C + 31) / 32;
    int count = p->B;                                                     // of the shared sums' parts
    if (a.nch > 1) {
        bwd_rows<T>(a, st);
        const long jobs = (long)ncb * p->B;
        hipLaunchKernelGGL((rn_fold_kernel<T>), dim3((unsigned)(jobs < RN_MAX_GRID ? jobs : RN_MAX_GRID)), dim3(1024), 0, st, a, sums);
    } else {
        const int per = group_of(p->B), slab = slab_of(p->B, p->T, p->C);
        count = (p->B + per - 1) / per;
        for (long first = 0; first < p->B; first += slab) {
            a.p = part_of<T>(*p, first, (int)(p->B - first < slab ? p->B - first : slab));
            bwd_rows<T>(a, st);
            hipLaunchKernelGGL((rn_fold_samples_kernel<T>), dim3((unsigned)(ncb * ((a.p.B + per - 1) / per))), dim3(1024), 0, st, a,
                               sums + first / per * RN_SUMS * p->C, per, count == 1);
        }
    }
    if (count > 1 && any_shared(p)) hipLaunchKernelGGL((rn_shared_kernel<T>), dim3(ncb, RN_SUMS), dim3(256), 0, st, *p, sums, count);
}

}  // namespace

extern "C" {

size_t cdae_resnorm_workspace_bytes(int B, int T, int C) {
    if (B <= 0 || T <= 0 || C <= 0 || C > RN_MAX_C) return 0;
    int nch, nch32, rows;
    chunks_of(B, T, C, false, nch, rows);
    chunks_of(B, T, C, true, nch32, rows);
    const size_t n = scratch_floats(B, T, C, nch), n32 = scratch_floats(B, T, C, nch32);
    return sizeof(float) * (n > n32 ? n : n32);
}

int cdae_resnorm_fwd(const cdae_resnorm* p, void* stream) {
    if (check(p)) return -1;
    if ((p->f && !p->r) || (p->pre && !p->u)) return cdae_fail("resnorm_fwd: r with a block output, u with a pre norm");
    hipStream_t st = (hipStream_t)stream;
    const double rows = (double)p->B * p->T * p->C * (p->dt == DT_F32 ? 4 : 2);
    const Timed timed(PROF_GN, rows * (1 + 2 * (p->f != nullptr) + (p->pre != 0)), rows * (1 + 2 * (p->f != nullptr) + (p->pre != 0)), st);
    if (p->dt == DT_F32) fwd<float>(p, st);
    else if (p->dt == DT_F16) fwd<F16>(p, st);
    else fwd<Bf16>(p, st);
    return hipGetLastError() == hipSuccess ? 0 : cdae_fail("resnorm_fwd launch failed");
}

int cdae_resnorm_bwd(const cdae_resnorm* p, void* stream) {
    if (check(p)) return -1;
    if (p->B >= RN_MAX_BLOCKS) return cdae_fail("resnorm_bwd: fewer than 2^22 samples");
    if (!p->dr && !p->du) return cdae_fail("resnorm_bwd: the gradient of r or of u required");
    if (p->du && !p->pre) return cdae_fail("resnorm_bwd: the gradient of u without a pre norm");
    if (!p->f && (p->df || p->dgate || p->dw1 || p->db1)) return cdae_fail("resnorm_bwd: gradients of a block output that is not there");
    if ((p->dgate && !p->gate) || (p->dscale && !p->scale) || (p->dshift && !p->shift) || (p->dw1 && !p->w1) || (p->db1 && !p->b1) || (p->dw2 && !p->w2) ||
        (p->db2 && !p->b2))
        return cdae_fail("resnorm_bwd: a gradient of a vector that is not there");
    if (!p->ws || ((size_t)p->ws & 15) || p->ws_bytes < (any_vector(p) ? cdae_resnorm_workspace_bytes(p->B, p->T, p->C) : 256))
        return cdae_fail("resnorm_bwd: workspace of cdae_resnorm_workspace_bytes(), or of 256 bytes without gradients of vectors, required");
    hipStream_t st = (hipStream_t)stream;
    const double rows = (double)p->B * p->T * p->C * (p->dt == DT_F32 ? 4 : 2) * (1 + (p->f != nullptr) + (p->dr != nullptr) + (p->du != nullptr) + (p->dx != nullptr) + (p->df != nullptr));
    const Timed timed(PROF_GN, rows, rows, st);
    if (p->dt == DT_F32) bwd<float>(p, st);
    else if (p->dt == DT_F16) bwd<F16>(p, st);
    else bwd<Bf16>(p, st);
    return hipGetLastError() == hipSuccess ? 0 : cdae_fail("resnorm_bwd launch failed");
}

}  // extern "C"
