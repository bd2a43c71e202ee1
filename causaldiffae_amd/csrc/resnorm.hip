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
// each, so it is read once whatever the number of reductions; a row's sums are a butterfly inside a wave and a pass through LDS across waves.
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
constexpr long RN_MAX_FOLD = 1 << 23;            // samples x 64-column blocks of a backward call (the same bound)

constexpr int RN_SUMS = 7;                       // of a sample: g A1, g A2, (1 + s) A3, (1 + s) A4, and the gradients of g, s, t

struct RnArgs {
    cdae_resnorm p;
    int nch, rows_per_chunk;                     // backward: chunks of a sample, rows of a chunk
};

// sums of a (and b) over the TPR threads of a row
template <int TPR, int NV>
__device__ __forceinline__ void row_sum(float (&a)[NV], float* sh) {
#pragma unroll
    for (int o = (TPR < 64 ? TPR : 64) / 2; o > 0; o >>= 1)
#pragma unroll
        for (int i = 0; i < NV; ++i) a[i] += __shfl_xor(a[i], o);
    if constexpr (TPR > 64) {
        constexpr int W = TPR / 64;
        const int wave = threadIdx.x >> 6;
        __syncthreads();
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int i = 0; i < NV; ++i) sh[wave * NV + i] = a[i];
        __syncthreads();
        const int w0 = wave / W * W;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            float s = 0.f;
#pragma unroll
            for (int w = 0; w < W; ++w) s += sh[(w0 + w) * NV + i];
            a[i] = s;
        }
    }
}

// n = normalised v (n values present), i = 1 / sqrt(mean square + eps); two passes over registers: the squares are of centred values
template <int TPR>
__device__ __forceinline__ float normalise(const float (&v)[RN_V], float (&n)[RN_V], int have, int layer, float inv_c, float eps, float* sh) {
    float m = 0.f;
    if (layer) {
        float s[1] = {0.f};
#pragma unroll
        for (int e = 0; e < RN_V; ++e) s[0] += v[e];              // (absent values are zero)
        row_sum<TPR, 1>(s, sh);
        m = s[0] * inv_c;
    }
    float q[1] = {0.f};
#pragma unroll
    for (int e = 0; e < RN_V; ++e) { n[e] = e < have ? v[e] - m : 0.f; q[0] = fmaf(n[e], n[e], q[0]); }
    row_sum<TPR, 1>(q, sh);
    const float i = 1.f / sqrtf(q[0] * inv_c + eps);
#pragma unroll
    for (int e = 0; e < RN_V; ++e) n[e] *= i;
    return i;
}

struct RnCol { float g[RN_V], w1[RN_V], b1[RN_V], w2[RN_V], b2[RN_V], s[RN_V], t[RN_V]; };

template <class T>
__device__ __forceinline__ void load_cols(const cdae_resnorm& p, long b, int c0, int have, RnCol& k, bool shift) {
#pragma unroll
    for (int e = 0; e < RN_V; ++e) { k.g[e] = p.alpha; k.w1[e] = 1.f; k.b1[e] = 0.f; k.w2[e] = 1.f; k.b2[e] = 0.f; k.s[e] = 1.f; k.t[e] = 0.f; }
    if (p.gate) {
        ldv_n2<T, RN_V>(p.gate, (p.shared_gate ? 0 : b * p.ld_gate) + c0, p.vec32, have, k.g);
#pragma unroll
        for (int e = 0; e < RN_V; ++e) k.g[e] *= p.alpha;
    }
    if (p.w1) ldv_n2<T, RN_V>(p.w1, c0, p.w32, have, k.w1);
    if (p.b1) ldv_n2<T, RN_V>(p.b1, c0, p.w32, have, k.b1);
    if (p.w2) ldv_n2<T, RN_V>(p.w2, c0, p.w32, have, k.w2);
    if (p.b2) ldv_n2<T, RN_V>(p.b2, c0, p.w32, have, k.b2);
    if (p.scale) {
        ldv_n2<T, RN_V>(p.scale, (p.shared_scale ? 0 : b * p.ld_scale) + c0, p.vec32, have, k.s);
#pragma unroll
        for (int e = 0; e < RN_V; ++e) k.s[e] += 1.f;
    }
    if (shift && p.shift) ldv_n2<T, RN_V>(p.shift, (p.shared_shift ? 0 : b * p.ld_shift) + c0, p.vec32, have, k.t);
}

template <class T, int TPR>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void rn_fwd_kernel(const RnArgs a) {
    constexpr int BLOCK = TPR < 256 ? 256 : TPR, RPB = BLOCK / TPR;
    __shared__ float sh[16];
    const cdae_resnorm& p = a.p;
    const int c0 = (threadIdx.x & (TPR - 1)) * RN_V;
    const int have = p.C - c0 < 0 ? 0 : p.C - c0 < RN_V ? p.C - c0 : RN_V;
    const float inv_c = 1.f / (float)p.C;
    const long M = (long)p.B * p.T;
    for (long row0 = (long)blockIdx.x * RPB; row0 < M; row0 += (long)gridDim.x * RPB) {
    const long row = row0 + threadIdx.x / TPR;
    const bool live = row < M;
    const int mine = live ? have : 0;
    const long rr = live ? row : M - 1;                          // (a row past the end computes the last one's and writes nothing)
    RnCol k;
    load_cols<T>(p, rr / p.T, c0, have, k, true);
    float r[RN_V];
    ldv_n<T, RN_V>(reinterpret_cast<const T*>(p.x) + rr * p.ld_x + c0, have, r);
    if (p.f) {
        float f[RN_V], n[RN_V];
        ldv_n<T, RN_V>(reinterpret_cast<const T*>(p.f) + rr * p.ld_f + c0, have, f);
        if (p.post) {
            normalise<TPR>(f, n, have, p.layer, inv_c, p.eps, sh);
#pragma unroll
            for (int e = 0; e < RN_V; ++e) f[e] = fmaf(n[e], k.w1[e], k.b1[e]);
        }
#pragma unroll
        for (int e = 0; e < RN_V; ++e) r[e] = e < have ? fmaf(k.g[e], f[e], r[e]) : 0.f;
        stv_n<T, RN_V>(reinterpret_cast<T*>(p.r) + rr * p.C + c0, mine, r);
    }
    if (p.pre) {
        float n[RN_V];
        normalise<TPR>(r, n, have, p.layer, inv_c, p.eps, sh);
#pragma unroll
        for (int e = 0; e < RN_V; ++e) n[e] = fmaf(fmaf(n[e], k.w2[e], k.b2[e]), k.s[e], k.t[e]);
        stv_n<T, RN_V>(reinterpret_cast<T*>(p.u) + rr * p.C + c0, mine, n);
    }
    }
}

// One block: rows [r0, r1) of one sample.  Leaves dx, df, and the four column sums of its rows in part[chunk][4][C].
template <class T, int TPR>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void rn_bwd_kernel(const RnArgs a) {
    constexpr int BLOCK = TPR < 256 ? 256 : TPR, RPB = BLOCK / TPR;
    __shared__ float sh[32];
    __shared__ float cols[RPB > 1 ? RPB * TPR * RN_V : 1];
    const cdae_resnorm& p = a.p;
    const int lane = threadIdx.x & (TPR - 1), grp = threadIdx.x / TPR;
    const int c0 = lane * RN_V;
    const int have = p.C - c0 < 0 ? 0 : p.C - c0 < RN_V ? p.C - c0 : RN_V;
    const float inv_c = 1.f / (float)p.C;
    const int b = blockIdx.x / a.nch, ch = blockIdx.x - b * a.nch;
    const long first = (long)b * p.T;
    const int t0 = ch * a.rows_per_chunk, t1 = t0 + a.rows_per_chunk < p.T ? t0 + a.rows_per_chunk : p.T;
    RnCol k;
    load_cols<T>(p, b, c0, have, k, false);
    float A[4][RN_V];
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int e = 0; e < RN_V; ++e) A[j][e] = 0.f;
    for (int tb = t0; tb < t1; tb += RPB) {                       // (the trip count is the block's: its barriers are met by every thread)
        const bool live = tb + grp < t1;
        const long row = first + (live ? tb + grp : t1 - 1);
        const int mine = live ? have : 0;
        float r[RN_V], n1[RN_V], D[RN_V], f[RN_V];
        float i1 = 0.f;
        ldv_n<T, RN_V>(reinterpret_cast<const T*>(p.x) + row * p.ld_x + c0, have, r);
#pragma unroll
        for (int e = 0; e < RN_V; ++e) { D[e] = 0.f; n1[e] = 0.f; }
        if (p.dr) ldv_n<T, RN_V>(reinterpret_cast<const T*>(p.dr) + row * p.ld_dr + c0, mine, D);
        if (p.f) {
            ldv_n<T, RN_V>(reinterpret_cast<const T*>(p.f) + row * p.ld_f + c0, have, f);
            if (p.post) i1 = normalise<TPR>(f, n1, have, p.layer, inv_c, p.eps, sh);
            else
#pragma unroll
                for (int e = 0; e < RN_V; ++e) n1[e] = f[e];
#pragma unroll
            for (int e = 0; e < RN_V; ++e) r[e] = e < have ? fmaf(k.g[e], fmaf(n1[e], k.w1[e], k.b1[e]), r[e]) : 0.f;
        }
        if (p.pre && p.du) {
            float U[RN_V], n2[RN_V];
            ldv_n<T, RN_V>(reinterpret_cast<const T*>(p.du) + row * p.ld_du + c0, mine, U);
            const float i2 = normalise<TPR>(r, n2, have, p.layer, inv_c, p.eps, sh);
            float s[2] = {0.f, 0.f};
#pragma unroll
            for (int e = 0; e < RN_V; ++e) {
                A[2][e] = fmaf(U[e], n2[e], A[2][e]);
                A[3][e] += U[e];
                U[e] = U[e] * k.s[e] * k.w2[e];
                s[0] = fmaf(U[e], n2[e], s[0]);
                s[1] += U[e];
            }
            row_sum<TPR, 2>(s, sh);
            const float m1 = s[0] * inv_c, m0 = p.layer ? s[1] * inv_c : 0.f;
#pragma unroll
            for (int e = 0; e < RN_V; ++e) D[e] += e < mine ? i2 * (U[e] - m0 - n2[e] * m1) : 0.f;
        }
        if (p.dx) stv_n<T, RN_V>(reinterpret_cast<T*>(p.dx) + row * p.C + c0, mine, D);
        if (p.f) {
            float s[2] = {0.f, 0.f};
#pragma unroll
            for (int e = 0; e < RN_V; ++e) {
                A[0][e] = fmaf(D[e], n1[e], A[0][e]);
                A[1][e] += D[e];
                D[e] = D[e] * k.g[e] * k.w1[e];
                s[0] = fmaf(D[e], n1[e], s[0]);
                s[1] += D[e];
            }
            if (p.post && p.df) {
                row_sum<TPR, 2>(s, sh);
                const float m1 = s[0] * inv_c, m0 = p.layer ? s[1] * inv_c : 0.f;
#pragma unroll
                for (int e = 0; e < RN_V; ++e) D[e] = i1 * (D[e] - m0 - n1[e] * m1);
            }
            if (p.df) stv_n<T, RN_V>(reinterpret_cast<T*>(p.df) + row * p.C + c0, mine, D);
        }
    }
    float* part = p.ws + (long)blockIdx.x * 4 * p.C;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if constexpr (RPB > 1) {                                  // the block's row groups, added in a fixed order
            __syncthreads();
#pragma unroll
            for (int e = 0; e < RN_V; ++e) cols[(grp * TPR + lane) * RN_V + e] = A[j][e];
            __syncthreads();
            for (int c = threadIdx.x; c < p.C; c += BLOCK) {
                float s = 0.f;
                for (int g = 0; g < RPB; ++g) s += cols[g * TPR * RN_V + c];
                part[j * p.C + c] = s;
            }
        } else {
            stv_n<float, RN_V>(part + j * p.C + c0, have, A[j]);
        }
    }
}

// The column sums of each sample from its chunks, and from them the gradients of gate, scale and shift; what the samples
// share goes to sums[b][7][C].  A block: 64 columns x 4 lanes of chunks.
template <class T>
__global__ __launch_bounds__(256) void rn_fold_kernel(const RnArgs a, float* __restrict__ sums) {
    const cdae_resnorm& p = a.p;
    const int ncb = (p.C + 63) / 64, b = blockIdx.x / ncb;
    const int c = (blockIdx.x - b * ncb) * 64 + (threadIdx.x & 63), q = threadIdx.x >> 6;
    __shared__ float sh[4][4][64];
    float A[4] = {0.f, 0.f, 0.f, 0.f};
    if (c < p.C)
        for (int ch = q; ch < a.nch; ch += 4) {
            const float* part = p.ws + ((long)b * a.nch + ch) * 4 * p.C + c;
#pragma unroll
            for (int j = 0; j < 4; ++j) A[j] += part[(long)j * p.C];
        }
#pragma unroll
    for (int j = 0; j < 4; ++j) sh[q][j][threadIdx.x & 63] = A[j];
    __syncthreads();
    if (q || c >= p.C) return;
#pragma unroll
    for (int j = 0; j < 4; ++j) A[j] = (sh[0][j][threadIdx.x] + sh[1][j][threadIdx.x]) + (sh[2][j][threadIdx.x] + sh[3][j][threadIdx.x]);
    auto vec = [&](const void* v, long off, int is32, float none) { return !v ? none : is32 ? ((const float*)v)[off] : ld1(((const T*)v)[off]); };
    const float g = vec(p.gate, (p.shared_gate ? 0 : b * p.ld_gate) + c, p.vec32, 1.f) * p.alpha, s1 = 1.f + vec(p.scale, (p.shared_scale ? 0 : b * p.ld_scale) + c, p.vec32, 0.f);
    const float w1 = vec(p.w1, c, p.w32, 1.f), b1 = vec(p.b1, c, p.w32, 0.f), w2 = vec(p.w2, c, p.w32, 1.f), b2 = vec(p.b2, c, p.w32, 0.f);
    const float dg = p.alpha * (w1 * A[0] + b1 * A[1]), ds = w2 * A[2] + b2 * A[3];
    if (p.dgate && !p.shared_gate) st2<T>(p.dgate, (long)b * p.C + c, p.vec32, dg);
    if (p.dscale && !p.shared_scale) st2<T>(p.dscale, (long)b * p.C + c, p.vec32, ds);
    if (p.dshift && !p.shared_shift) st2<T>(p.dshift, (long)b * p.C + c, p.vec32, A[3]);
    const float o[RN_SUMS] = {g * A[0], g * A[1], s1 * A[2], s1 * A[3], dg, ds, A[3]};
#pragma unroll
    for (int j = 0; j < RN_SUMS; ++j) sums[((long)b * RN_SUMS + j) * p.C + c] = o[j];
}

// what all samples share: grid y picks one of the seven sums
template <class T>
__global__ __launch_bounds__(256) void rn_shared_kernel(const RnArgs a, const float* __restrict__ sums) {
    const cdae_resnorm& p = a.p;
    const int c = blockIdx.x * 256 + threadIdx.x, j = blockIdx.y;
    void* const dst[RN_SUMS] = {p.dw1, p.db1, p.dw2, p.db2, p.shared_gate ? p.dgate : nullptr, p.shared_scale ? p.dscale : nullptr, p.shared_shift ? p.dshift : nullptr};
    void* out = nullptr;
#pragma unroll
    for (int i = 0; i < RN_SUMS; ++i) if (i == j) out = dst[i];
    if (!out || c >= p.C) return;
    float s = 0.f;
    for (int b = 0; b < p.B; ++b) s += sums[((long)b * RN_SUMS + j) * p.C + c];
    st2<T>(out, c, j < 4 ? p.w32 : p.vec32, s);
}

int threads_per_row(int C) {
    int t = 1;
    while (t * RN_V < C) t *= 2;
    return t < 8 ? 8 : t;
}

// chunks of a sample: about 1024 blocks in all, at least one pass of a block's row groups each
void chunks_of(int B, int T, int C, int& nch, int& rows) {
    const int tpr = threads_per_row(C), rpb = tpr < 256 ? 256 / tpr : 1;
    long want = (1024 + B - 1) / B;
    rows = (int)((T + want - 1) / want);
    if (rows < rpb) rows = rpb;
    rows = (rows + rpb - 1) / rpb * rpb;
    nch = (T + rows - 1) / rows;
}

int check(const cdae_resnorm* p) {
    if (!p || p->B <= 0 || p->T <= 0 || p->C <= 0 || p->C > RN_MAX_C) return cdae_fail("resnorm: B, T >= 1 and 1 <= C <= 8192 required");
    if ((long)p->B * p->T > 0x7fffffffL) return cdae_fail("resnorm: at most 2^31 - 1 rows");
    if (p->dt < 0 || p->dt > 2) return cdae_fail("resnorm: row type 0 (bf16), 1 (fp16) or 2 (fp32)");
    if (!p->x || (!p->f && !p->pre)) return cdae_fail("resnorm: x and a block output or a pre norm required");
    if (!p->f && (p->post || p->gate)) return cdae_fail("resnorm: a post norm or a gate needs a block output");
    if (!p->pre && (p->w2 || p->b2 || p->scale || p->shift)) return cdae_fail("resnorm: w2, b2, scale and shift belong to a pre norm");
    if (!p->post && (p->w1 || p->b1)) return cdae_fail("resnorm: w1 and b1 belong to a post norm");
    if (!(p->eps >= 0.f)) return cdae_fail("resnorm: eps must be >= 0");
    return 0;
}

#define RN_TPR(CALL)                          \
    switch (threads_per_row(p->C)) {          \
        case 8: { CALL(8); break; }           \
        case 16: { CALL(16); break; }         \
        case 32: { CALL(32); break; }         \
        case 64: { CALL(64); break; }         \
        case 128: { CALL(128); break; }       \
        case 256: { CALL(256); break; }       \
        case 512: { CALL(512); break; }       \
        default: { CALL(1024); break; }       \
    }

template <class T>
void fwd(const cdae_resnorm* p, hipStream_t st) {
    RnArgs a;
    a.p = *p; a.nch = a.rows_per_chunk = 0;
    const long M = (long)p->B * p->T;
#define RN_CALL(N) { constexpr int BL = N < 256 ? 256 : N; const long g = (M + BL / N - 1) / (BL / N); \
                     hipLaunchKernelGGL((rn_fwd_kernel<T, N>), dim3((unsigned)(g < RN_MAX_GRID ? g : RN_MAX_GRID)), dim3(BL), 0, st, a); }
    RN_TPR(RN_CALL)
#undef RN_CALL
}
template <class T>
void bwd(const cdae_resnorm* p, hipStream_t st) {
    RnArgs a;
    a.p = *p;
    chunks_of(p->B, p->T, p->C, a.nch, a.rows_per_chunk);
    float* sums = p->ws + (long)p->B * a.nch * 4 * p->C;
#define RN_CALL(N) { constexpr int BL = N < 256 ? 256 : N; hipLaunchKernelGGL((rn_bwd_kernel<T, N>), dim3((unsigned)((long)p->B * a.nch)), dim3(BL), 0, st, a); }
    RN_TPR(RN_CALL)
#undef RN_CALL
    if (!(p->dgate || p->dscale || p->dshift || p->dw1 || p->db1 || p->dw2 || p->db2)) return;
    hipLaunchKernelGGL((rn_fold_kernel<T>), dim3((unsigned)((p->C + 63) / 64 * (long)p->B)), dim3(256), 0, st, a, sums);
    if (p->dw1 || p->db1 || p->dw2 || p->db2 || (p->dgate && p->shared_gate) || (p->dscale && p->shared_scale) || (p->dshift && p->shared_shift))
        hipLaunchKernelGGL((rn_shared_kernel<T>), dim3((p->C + 255) / 256, RN_SUMS), dim3(256), 0, st, a, sums);
}

}  // namespace

extern "C" {

size_t cdae_resnorm_workspace_bytes(int B, int T, int C) {
    if (B <= 0 || T <= 0 || C <= 0 || C > RN_MAX_C) return 0;
    int nch, rows;
    chunks_of(B, T, C, nch, rows);
    return sizeof(float) * 4 * (size_t)C * B * nch + sizeof(float) * RN_SUMS * (size_t)C * B;
}

int cdae_resnorm_fwd(const cdae_resnorm* p, void* stream) {
    if (check(p)) return -1;
    if ((p->f && !p->r) || (p->pre && !p->u)) return cdae_fail("resnorm_fwd: r with a block output, u with a pre norm");
    hipStream_t st = (hipStream_t)stream;
    if (p->dt == DT_F32) fwd<float>(p, st);
    else if (p->dt == DT_F16) fwd<F16>(p, st);
    else fwd<Bf16>(p, st);
    return hipGetLastError() == hipSuccess ? 0 : cdae_fail("resnorm_fwd launch failed");
}

int cdae_resnorm_bwd(const cdae_resnorm* p, void* stream) {
    if (check(p)) return -1;
    if ((long)p->B * ((p->C + 63) / 64) > RN_MAX_FOLD) return cdae_fail("resnorm_bwd: at most 2^23 / ceil(C / 64) samples");
    if (!p->dr && !p->du) return cdae_fail("resnorm_bwd: the gradient of r or of u required");
    if (p->du && !p->pre) return cdae_fail("resnorm_bwd: the gradient of u without a pre norm");
    if (!p->f && (p->df || p->dgate || p->dw1 || p->db1)) return cdae_fail("resnorm_bwd: gradients of a block output that is not there");
    if ((p->dgate && !p->gate) || (p->dscale && !p->scale) || (p->dshift && !p->shift) || (p->dw1 && !p->w1) || (p->db1 && !p->b1) || (p->dw2 && !p->w2) ||
        (p->db2 && !p->b2))
        return cdae_fail("resnorm_bwd: a gradient of a vector that is not there");
    if (!p->ws || p->ws_bytes < cdae_resnorm_workspace_bytes(p->B, p->T, p->C)) return cdae_fail("resnorm_bwd: workspace of cdae_resnorm_workspace_bytes() required");
    hipStream_t st = (hipStream_t)stream;
    if (p->dt == DT_F32) bwd<float>(p, st);
    else if (p->dt == DT_F16) bwd<F16>(p, st);
    else bwd<Bf16>(p, st);
    return hipGetLastError() == hipSuccess ? 0 : cdae_fail("resnorm_bwd launch failed");
}

}  // extern "C"
