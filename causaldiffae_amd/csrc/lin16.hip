// lin16.hip — linear layers on bf16 / f16 rows with activation and residual in the product's epilogue, and their gradients (gfx950):
//
//     z = x W^T + b,     y = act(z) + res                                     x [M][K], W [N][K]
//     dz = dy o act'(z),   dx = dz W,   dW = dz^T x,   db = sum over rows of dz
//
// All three products are C[m][n] = sum over k of A(m, k) B(n, k) with an operand's k running along its rows (KC) or across them (MC):
// forward KC x KC, data gradient KC x MC (k = N), weight gradient MC x MC (k = M).  MC fragments come out of LDS through the hardware transpose read.
#include <hip/hip_runtime.h>
#include <math.h>

#include "cdae.h"
#include "block_common.h"
#include "cdae_internal.h"

namespace {

typedef unsigned short u16;
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __fp16 fp16x4 __attribute__((__vector_size__(4 * sizeof(__fp16))));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

enum { L_NONE = 0, L_SILU = 1, L_RELU = 3, L_GELU = 5, L_GELU_TANH = 6 };      // (the numbers of ops.ACT_*)

__device__ __attribute__((aligned(16))) unsigned g_zero_lin16[4] = {0u, 0u, 0u, 0u};

__device__ __forceinline__ float act_fwd(float z, int act) {
    switch (act) {
        case L_SILU: return z * cdae_sigmoid(z);
        case L_RELU: return z > 0.f ? z : (z != z ? z : 0.f);
        case L_GELU: return 0.5f * z * (1.f + erff(z * 0.70710678118654752f));
        case L_GELU_TANH: return z * cdae_sigmoid(1.5957691216057308f * fmaf(0.044715f * z * z, z, z));      // 0.5 (1 + tanh a) = sigmoid(2 a)
        default: return z;
    }
}
__device__ __forceinline__ float act_slope(float z, int act) {
    switch (act) {
        case L_SILU: { const float s = cdae_sigmoid(z); return s * fmaf(z, 1.f - s, 1.f); }
        case L_RELU: return z > 0.f ? 1.f : 0.f;
        case L_GELU: return fmaf(0.3989422804014327f * z, expf(-0.5f * z * z), 0.5f * (1.f + erff(z * 0.70710678118654752f)));
        case L_GELU_TANH: {
            const float s = cdae_sigmoid(1.5957691216057308f * fmaf(0.044715f * z * z, z, z));
            return s * fmaf(z * (1.f - s), 1.5957691216057308f * fmaf(0.134145f * z, z, 1.f), 1.f);
        }
        default: return 1.f;
    }
}
// The pre-activation is kept for the backward in f16 whatever the rows' type: its 11 bits cost the slope a quarter of what the rounding of dz to
// bf16 costs, and where f16 ends (65504) every slope has long reached its limit, so larger values are clamped there.
__device__ __forceinline__ _Float16 keep_z(float z) { return (_Float16)(fabsf(z) > 65504.f ? copysignf(65504.f, z) : z); }

struct LinArgs {
    const u16* A; long lda;                 // KC: [M][K], MC: [K][M]
    const u16* B; long ldb;                 // KC: [N][K], MC: [K][N]
    int M, N, K;
    const u16* bias; const u16* res; long ldres; u16* y; long ldy; _Float16* z; long ldz; int act;
    float* slab; int splits, k_per_split;   // splits > 1: partial sums [split][M][N] instead of the epilogue
    int tiles_m, tiles_n;
};

template <class T> struct Mfma;
template <> struct Mfma<Bf16> {
    static __device__ __forceinline__ f32x4 go(u32x4 a, u32x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
};
template <> struct Mfma<F16> {
    static __device__ __forceinline__ f32x4 go(u32x4 a, u32x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
};

// v[0..n) of row m from column n0: bias, activation, residual, rounding
template <class T, int V>
__device__ __forceinline__ void finish_row(const LinArgs& p, long m, int n0, int n, float (&v)[V]) {
    if (n <= 0) return;
    float t[V];
    if (p.bias) {
        ldv_n<T, V>(reinterpret_cast<const T*>(p.bias) + n0, n, t);
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] += t[i];
    }
    if (p.z) {
        _Float16* zp = p.z + m * p.ldz + n0;
        Pack<F16, V> k;
#pragma unroll
        for (int i = 0; i < V; ++i) k.v[i].h = keep_z(v[i]);
        if (n >= V) *reinterpret_cast<Pack<F16, V>*>(zp) = k;
        else
#pragma unroll
            for (int i = 0; i < V; ++i) if (i < n) zp[i] = k.v[i].h;
    }
    if (p.act != L_NONE)
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = act_fwd(v[i], p.act);
    if (p.res) {
        ldv_n<T, V>(reinterpret_cast<const T*>(p.res) + m * p.ldres + n0, n, t);
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] += t[i];
    }
    stv_n<T, V>(reinterpret_cast<T*>(p.y) + m * p.ldy + n0, n, v);
}

// 128 x 128 tile, four waves of 64 x 64, 32 k a step
template <class T, bool AMC, bool BMC>
__global__ __launch_bounds__(256, 2) void lin_tile_kernel(const LinArgs p) {
    constexpr int OPB = 128 * 64, STAGE = 2 * OPB;                       // bytes of one operand's step
    __shared__ __attribute__((aligned(1024))) unsigned char lds[2 * STAGE];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int i16 = lane & 15, q = lane >> 4;
    const int tiles = p.tiles_m * p.tiles_n;
    const int split = blockIdx.x / tiles, tile = blockIdx.x - split * tiles;
    const int tm = tile / p.tiles_n, tn = tile - tm * p.tiles_n;
    const int m0 = tm * 128, n0 = tn * 128;
    const int kb = split * p.k_per_split, ke = kb + p.k_per_split < p.K ? kb + p.k_per_split : p.K;
    const int steps = (ke - kb + 31) / 32;
    const unsigned base = (unsigned)(size_t)lds;
    const void* zero = (const void*)g_zero_lin16;
    asm volatile("" : "+s"(zero));

    // One operand's step: 8 DMAs of 1 KB, two a wave.  KC: 16 rows x four 16-byte pieces, piece j of row r <- piece j ^ (r >> 2 & 3) (16 rows at one
    // piece then cover all banks once); MC: four k rows x 16 pieces, piece j of row r <- j ^ 2 (r & 3 | (r >> 3 & 1) << 2).
    // A piece outside the operand is read from a line of zeros: the sizes along k and along the rows are multiples of 8.
    auto fetch = [&](bool mc, const u16* X, long ldx, int rows, int r0, int k0, unsigned dst) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int d = 2 * wave + e;
            const void* src;
            if (!mc) {
                const int r = 16 * d + (lane >> 2), pc = (lane & 3) ^ ((r >> 2) & 3), k = k0 + 8 * pc;
                const int row = r0 + r < rows ? r0 + r : rows - 1;
                src = k < ke ? (const void*)(X + (long)row * ldx + k) : zero;
            } else {
                const int r = 4 * d + (lane >> 4), pc = (lane & 15) ^ (2 * ((r & 3) | (((r >> 3) & 1) << 2)));
                const int k = k0 + r, c = r0 + 8 * pc;
                src = k < ke && c < rows ? (const void*)(X + (long)k * ldx + c) : zero;
            }
            cdae_lds_dma16(src, dst + d * 1024);
        }
    };
    auto frag = [&](bool mc, const unsigned char* img, int r0) -> u32x4 {            // 8 k (8 q .. + 7) of row r0 + i16
        if (!mc) {
            const int r = r0 + i16;
            return *reinterpret_cast<const u32x4*>(img + r * 64 + ((q ^ ((r >> 2) & 3)) * 16));
        }
        const int k = 8 * q + (i16 >> 2), pp = i16 & 3;
        const unsigned char* src = img + k * 256 + ((((r0 >> 3) + (pp >> 1)) ^ (2 * ((k & 3) | (((k >> 3) & 1) << 2)))) * 16) + (pp & 1) * 8;
        const fp16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4f16((__attribute__((address_space(3))) fp16x4*)(src));
        const fp16x4 c = __builtin_amdgcn_ds_read_tr16_b64_v4f16((__attribute__((address_space(3))) fp16x4*)(src + 4 * 256));
        const u32x2 a2 = __builtin_bit_cast(u32x2, a), c2 = __builtin_bit_cast(u32x2, c);
        u32x4 v;
        v[0] = a2[0]; v[1] = a2[1]; v[2] = c2[0]; v[3] = c2[1];
        return v;
    };

    const int wm = wave >> 1, wn = wave & 1;
    f32x4 acc[4][4];
#pragma unroll
    for (int a = 0; a < 4; ++a)
#pragma unroll
        for (int b = 0; b < 4; ++b) acc[a][b] = (f32x4){0.f, 0.f, 0.f, 0.f};

    fetch(AMC, p.A, p.lda, p.M, m0, kb, base);
    fetch(BMC, p.B, p.ldb, p.N, n0, kb, base + OPB);
    for (int s = 0; s < steps; ++s) {
        const int slot = s & 1;
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (s + 1 < steps) {
            fetch(AMC, p.A, p.lda, p.M, m0, kb + 32 * (s + 1), base + (slot ^ 1) * STAGE);
            fetch(BMC, p.B, p.ldb, p.N, n0, kb + 32 * (s + 1), base + (slot ^ 1) * STAGE + OPB);
        }
        const unsigned char* as = lds + slot * STAGE;
        const unsigned char* bs = as + OPB;
        u32x4 fa[4], fb[4];
#pragma unroll
        for (int a = 0; a < 4; ++a) { fa[a] = frag(AMC, as, wm * 64 + a * 16); fb[a] = frag(BMC, bs, wn * 64 + a * 16); }
#pragma unroll
        for (int a = 0; a < 4; ++a)
#pragma unroll
            for (int b = 0; b < 4; ++b) acc[a][b] = Mfma<T>::go(fb[b], fa[a], acc[a][b]);       // rows of the result: n (4 q + r), columns: m (i16)
    }
#pragma unroll
    for (int a = 0; a < 4; ++a) {
        const int m = m0 + wm * 64 + a * 16 + i16;
        if (m >= p.M) continue;
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            const int n = n0 + wn * 64 + b * 16 + 4 * q;
            float v[4] = {acc[a][b][0], acc[a][b][1], acc[a][b][2], acc[a][b][3]};
            if (p.splits > 1) { if (n < p.N) stv_n<float, 4>(p.slab + ((long)split * p.M + m) * p.N + n, p.N - n, v); }
            else finish_row<T, 4>(p, m, n, p.N - n, v);
        }
    }
}

// partial sums of the splits, added in order, then the epilogue: 8 columns a thread
template <class T>
__global__ __launch_bounds__(256) void lin_finish_kernel(const LinArgs p) {
    const long per = (p.N + 7) / 8, total = per * p.M;
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long)gridDim.x * 256) {
        const long m = i / per;
        const int n = (int)(i - m * per) * 8, have = p.N - n;
        float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        for (int s = 0; s < p.splits; ++s) {
            float t[8];
            ldv_n<float, 8>(p.slab + ((long)s * p.M + m) * p.N + n, have, t);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] += t[e];
        }
        finish_row<T, 8>(p, m, n, have, v);
    }
}

// [rows][cols] at any pitch and alignment -> a dense image whose rows are padded with zeros to `pitch` (a multiple of 8)
__global__ __launch_bounds__(256) void lin_pad_kernel(const u16* __restrict__ src, long lds_, u16* __restrict__ dst, long rows, int cols, int pitch) {
    const long per = pitch / 8, total = per * rows;
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long)gridDim.x * 256) {
        const long r = i / per;
        const int c = (int)(i - r * per) * 8, have = cols - c;
        const u16* s = src + r * lds_ + c;
        Pack<u16, 8> t;
        if (have >= 8) t = *reinterpret_cast<const Pack<u16, 8>*>(s);
        else
#pragma unroll
            for (int e = 0; e < 8; ++e) t.v[e] = e < have ? s[e] : (u16)0;
        u32x4 w;
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = (unsigned)t.v[2 * e] | (unsigned)t.v[2 * e + 1] << 16;
        *reinterpret_cast<u32x4*>(dst + r * pitch + c) = w;
    }
}

// dz = dy o act'(z) (written where wanted) and its column sums over a block's rows.  A block: 256 columns x 8 row lanes, 8 columns a thread.
template <class T>
__global__ __launch_bounds__(256) void lin_slope_kernel(const T* __restrict__ dy, long lddy, const _Float16* __restrict__ z, long ldz, T* __restrict__ dz, long lddz,
                                                        float* __restrict__ part, int M, int N, int rows_per_block, int ncb, int act) {
    __shared__ float sh[8][256];
    const int cb = blockIdx.x % ncb, rb = blockIdx.x / ncb;
    const int cl = threadIdx.x & 31, rl = threadIdx.x >> 5;
    const int c = cb * 256 + cl * 8, have = N - c;
    const long r0 = (long)rb * rows_per_block, r1 = r0 + rows_per_block < M ? r0 + rows_per_block : M;
    float s[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (have > 0)
        for (long r = r0 + rl; r < r1; r += 8) {
            float g[8];
            ldv_n<T, 8>(dy + r * lddy + c, have, g);
            if (act != L_NONE) {
                float zz[8];
                ldv_n<F16, 8>(reinterpret_cast<const F16*>(z) + r * ldz + c, have, zz);
#pragma unroll
                for (int e = 0; e < 8; ++e) g[e] *= act_slope(zz[e], act);
            }
            if (dz) {
                if (have >= 8 || c + 8 <= lddz) {                         // (a padded row takes its zeros along)
                    stv<T, 8>(dz + r * lddz + c, g);
                } else stv_n<T, 8>(dz + r * lddz + c, have, g);
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) s[e] += g[e];
        }
    if (!part) return;
#pragma unroll
    for (int e = 0; e < 8; ++e) sh[rl][cl * 8 + e] = s[e];
    __syncthreads();
    const int cc = cb * 256 + threadIdx.x;
    if (cc < N) {
        float t = 0.f;
#pragma unroll
        for (int r = 0; r < 8; ++r) t += sh[r][threadIdx.x];
        part[(long)rb * N + cc] = t;
    }
}
template <class T>
__global__ __launch_bounds__(256) void lin_bias_kernel(const float* __restrict__ part, int blocks, int N, T* __restrict__ db) {
    __shared__ float sh[4][64];
    const int cl = threadIdx.x & 63, q = threadIdx.x >> 6, c = blockIdx.x * 64 + cl;
    float s = 0.f;
    if (c < N)
        for (int b = q; b < blocks; b += 4) s += part[(long)b * N + c];
    sh[q][cl] = s;
    __syncthreads();
    if (q == 0 && c < N) st1(db[c], (sh[0][cl] + sh[1][cl]) + (sh[2][cl] + sh[3][cl]));
}

long up8(long v) { return (v + 7) / 8 * 8; }
bool al16(const void* p) { return ((size_t)p & 15) == 0; }
size_t up256(size_t b) { return (b + 255) / 256 * 256; }

// splits of the sum over k: where the tiles alone leave most of the 512 block slots (two a CU) empty, and a split keeps at least 256 of k
int splits_of(int M, int N, int K) {
    const long tiles = (long)((M + 127) / 128) * ((N + 127) / 128);
    long s = 512 / (tiles > 0 ? tiles : 1);
    if (s > K / 256) s = K / 256;
    if (s > 64) s = 64;
    return s < 1 ? 1 : (int)s;
}
size_t gemm_ws(int M, int N, int K) {
    const int s = splits_of(M, N, K);
    return s > 1 ? up256((size_t)s * M * N * 4) : 0;
}

// One operand in the form the tile kernel reads: 16-byte pieces, rows of a multiple of 8 values.  Copies it into `ws` where it is not.
int prepare(const u16*& X, long& ldx, long rows, int cols, char*& ws, hipStream_t st) {
    if (cols % 8 == 0 && ldx % 8 == 0 && al16(X)) return 0;
    const long pitch = up8(cols);
    u16* dst = (u16*)ws;
    ws += up256((size_t)rows * pitch * 2);
    const long total = rows * (pitch / 8);
    const long g = (total + 255) / 256;
    hipLaunchKernelGGL(lin_pad_kernel, dim3((unsigned)(g < 8192 ? g : 8192)), dim3(256), 0, st, X, ldx, dst, rows, cols, (int)pitch);
    X = dst; ldx = pitch;
    return hipGetLastError() == hipSuccess ? 0 : cdae_fail("lin16: launch failed");
}

template <class T, bool AMC, bool BMC>
int product(LinArgs p, char* ws, hipStream_t st) {
    p.tiles_m = (p.M + 127) / 128; p.tiles_n = (p.N + 127) / 128;
    // (rows of an MC operand are padded to 8 values, so the kernel may see up to 7 columns more than there are: it reads them, and writes none)
    p.splits = splits_of(p.M, p.N, p.K);
    p.k_per_split = ((p.K + p.splits - 1) / p.splits + 31) / 32 * 32;
    p.splits = (p.K + p.k_per_split - 1) / p.k_per_split;
    p.slab = (float*)ws;
    const long blocks = (long)p.tiles_m * p.tiles_n * p.splits;
    if (blocks > (1L << 23)) return cdae_fail("lin16: product too large");
    hipLaunchKernelGGL((lin_tile_kernel<T, AMC, BMC>), dim3((unsigned)blocks), dim3(256), 0, st, p);
    if (hipGetLastError() != hipSuccess) return cdae_fail("lin16: launch failed");
    if (p.splits > 1) {
        const long g = ((long)p.M * ((p.N + 7) / 8) + 255) / 256;
        hipLaunchKernelGGL((lin_finish_kernel<T>), dim3((unsigned)(g < 8192 ? g : 8192)), dim3(256), 0, st, p);
        if (hipGetLastError() != hipSuccess) return cdae_fail("lin16: launch failed");
    }
    return 0;
}

int bad_dims(int M, int N, int K, int dt) {
    if (M < 0 || N <= 0 || K <= 0) return cdae_fail("lin16: M >= 0, N >= 1 and K >= 1 required");
    if (dt != DT_BF16 && dt != DT_F16) return cdae_fail("lin16: type 0 (bf16) or 1 (fp16)");
    return 0;
}
bool known_act(int a) { return a == L_NONE || a == L_SILU || a == L_RELU || a == L_GELU || a == L_GELU_TANH; }

int slope_rows(int M, int N) {           // rows of a block of the slope pass: about 2048 blocks, at most 64 row blocks for the fold of the sums
    const int ncb = (N + 255) / 256;
    int rb = (2048 + ncb - 1) / ncb;
    if (rb > 64) rb = 64;
    int rows = (M + rb - 1) / rb;
    return rows < 8 ? 8 : rows;
}

}  // namespace

extern "C" {

size_t cdae_lin16_workspace_bytes(int op, int M, int N, int K) {
    if (M <= 0 || N <= 0 || K <= 0) return 0;
    const size_t x = up256((size_t)M * up8(K) * 2), w = up256((size_t)N * up8(K) * 2), d = up256((size_t)M * up8(N) * 2);
    if (op == CDAE_LIN16_FWD) return x + w + gemm_ws(M, N, K) + 256;
    if (op == CDAE_LIN16_BWD) {
        const int rows = slope_rows(M, N);
        const size_t sums = up256(sizeof(float) * (size_t)N * ((M + rows - 1) / rows)), one = w + gemm_ws(M, K, N), two = x + gemm_ws(N, K, M);
        const size_t most = one > two ? one : two;
        return d + (sums > most ? sums : most) + 256;
    }
    return 0;
}

int cdae_lin16_fwd(const void* x, long ldx, const void* w, long ldw, const void* bias, const void* res, long ldres, void* y, long ldy, void* z, long ldz, int M,
                   int N, int K, int act, int dt, void* ws, size_t ws_bytes, void* stream) {
    if (bad_dims(M, N, K, dt)) return -1;
    if (!known_act(act)) return cdae_fail("lin16_fwd: activation 0 (none), 1 (SiLU), 3 (ReLU), 5 (GELU) or 6 (GELU, tanh form)");
    if (M == 0) return 0;
    if (!x || !w || !y || ldx < K || ldw < K || ldy < N || (res && ldres < N) || (z && ldz < N)) return cdae_fail("lin16_fwd: x, w, y and row pitches of at least a row required");
    if (ws_bytes < cdae_lin16_workspace_bytes(CDAE_LIN16_FWD, M, N, K) || !ws) return cdae_fail("lin16_fwd: workspace of cdae_lin16_workspace_bytes() required");
    hipStream_t st = (hipStream_t)stream;
    LinArgs p{};
    char* at = (char*)ws;
    p.A = (const u16*)x; p.lda = ldx; p.B = (const u16*)w; p.ldb = ldw;
    if (prepare(p.A, p.lda, M, K, at, st) || prepare(p.B, p.ldb, N, K, at, st)) return -1;
    p.M = M; p.N = N; p.K = K;
    p.bias = (const u16*)bias; p.res = (const u16*)res; p.ldres = ldres; p.y = (u16*)y; p.ldy = ldy; p.z = (_Float16*)z; p.ldz = ldz; p.act = act;
    return dt == DT_BF16 ? product<Bf16, false, false>(p, at, st) : product<F16, false, false>(p, at, st);
}

int cdae_lin16_bwd(const void* dy, long lddy, const void* x, long ldx, const void* w, long ldw, const void* z, long ldz, void* dx, long lddx, void* dw, long lddw,
                   void* dbias, int M, int N, int K, int act, int dt, void* ws, size_t ws_bytes, void* stream) {
    if (bad_dims(M, N, K, dt)) return -1;
    if (!known_act(act)) return cdae_fail("lin16_bwd: activation 0 (none), 1 (SiLU), 3 (ReLU), 5 (GELU) or 6 (GELU, tanh form)");
    if (M == 0) return cdae_fail("lin16_bwd: no rows");
    if (!dy || lddy < N || (act != L_NONE && (!z || ldz < N))) return cdae_fail("lin16_bwd: dy, and z with an activation, required");
    if ((dx && (!w || ldw < K || lddx < K)) || (dw && (!x || ldx < K || lddw < K))) return cdae_fail("lin16_bwd: w for dx, x for dw, row pitches of at least a row");
    if (!ws || ws_bytes < cdae_lin16_workspace_bytes(CDAE_LIN16_BWD, M, N, K)) return cdae_fail("lin16_bwd: workspace of cdae_lin16_workspace_bytes() required");
    hipStream_t st = (hipStream_t)stream;
    char* at = (char*)ws;
    const bool copy = act != L_NONE || N % 8 || lddy % 8 || !al16(dy);
    u16* dz = nullptr;
    if (copy && (dx || dw)) { dz = (u16*)at; at += up256((size_t)M * up8(N) * 2); }
    if (dz || dbias) {
        const int ncb = (N + 255) / 256, rows = slope_rows(M, N), rb = (M + rows - 1) / rows;
        float* part = dbias ? (float*)at : nullptr;
        const dim3 grid((unsigned)(ncb * rb));
        if (dt == DT_BF16)
            hipLaunchKernelGGL((lin_slope_kernel<Bf16>), grid, dim3(256), 0, st, (const Bf16*)dy, lddy, (const _Float16*)z, ldz, (Bf16*)dz, up8(N), part, M, N, rows, ncb, act);
        else
            hipLaunchKernelGGL((lin_slope_kernel<F16>), grid, dim3(256), 0, st, (const F16*)dy, lddy, (const _Float16*)z, ldz, (F16*)dz, up8(N), part, M, N, rows, ncb, act);
        if (dbias) {
            if (dt == DT_BF16) hipLaunchKernelGGL((lin_bias_kernel<Bf16>), dim3((N + 63) / 64), dim3(256), 0, st, part, rb, N, (Bf16*)dbias);
            else hipLaunchKernelGGL((lin_bias_kernel<F16>), dim3((N + 63) / 64), dim3(256), 0, st, part, rb, N, (F16*)dbias);
        }
        if (hipGetLastError() != hipSuccess) return cdae_fail("lin16_bwd: launch failed");
    }
    const u16* d = dz ? dz : (const u16*)dy;
    const long ldd = dz ? up8(N) : lddy;
    if (dx) {
        LinArgs p{};
        p.A = d; p.lda = ldd; p.B = (const u16*)w; p.ldb = ldw;
        char* tmp = at;                                     // (a stream's launches run in order: the products use the same scratch one after the other)
        if (prepare(p.B, p.ldb, N, K, tmp, st)) return -1;
        p.M = M; p.N = K; p.K = N;
        p.y = (u16*)dx; p.ldy = lddx;
        if (dt == DT_BF16 ? product<Bf16, false, true>(p, tmp, st) : product<F16, false, true>(p, tmp, st)) return -1;
    }
    if (dw) {
        LinArgs p{};
        p.A = d; p.lda = ldd; p.B = (const u16*)x; p.ldb = ldx;
        char* tmp = at;
        if (prepare(p.B, p.ldb, M, K, tmp, st)) return -1;
        p.M = N; p.N = K; p.K = M;
        p.y = (u16*)dw; p.ldy = lddw;
        if (dt == DT_BF16 ? product<Bf16, true, true>(p, tmp, st) : product<F16, true, true>(p, tmp, st)) return -1;
    }
    return 0;
}

}  // extern "C"
