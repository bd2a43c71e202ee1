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

// Activations and slopes for results of 16 bits: a few steps of fp32 from the exact value, on the exp2 and reciprocal instructions.
//   logistic(a) = 1 / (1 + 2^(-a log2 e)): where 2^t overflows the reciprocal is 0, the limit.
//   The normal distribution function after Abramowitz & Stegun, Handbook of Mathematical Functions, 7.1.26 (absolute error 1.5e-7, and its
//   exp(-z^2 / 2) is the density the slope needs): 15 instructions where the library's erf takes about 40, and the epilogue is bound by them
//   (12.6 million values of a 8192 x 1536 result: 40 instructions a value are 13 us of all vector units).
__device__ __forceinline__ float logistic(float a) { return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.4426950408889634f * a)); }
__device__ __forceinline__ float normal_cdf(float z, float& e) {
    const float x = fabsf(z) * 0.70710678118654752f, t = __builtin_amdgcn_rcpf(fmaf(0.3275911f, x, 1.f));
    e = __builtin_amdgcn_exp2f(-0.72134752044448170f * z * z);                                       // exp(-z^2 / 2)
    const float p = t * fmaf(t, fmaf(t, fmaf(t, fmaf(t, 1.061405429f, -1.453152027f), 1.421413741f), -0.284496736f), 0.254829592f);
    const float tail = 0.5f * p * e;                                                                 // of the side that z points to
    return z < 0.f ? tail : 1.f - tail;
}
__device__ __forceinline__ float gelu_tanh_arg(float z) { return 1.5957691216057308f * z * fmaf(0.044715f * z, z, 1.f); }      // 0.5 (1 + tanh a) = logistic(2 a)

__device__ __forceinline__ float act_fwd(float z, int act) {
    switch (act) {
        case L_SILU: return z * logistic(z);
        case L_RELU: return z > 0.f ? z : (z != z ? z : 0.f);
        case L_GELU: { float e; return z * normal_cdf(z, e); }
        case L_GELU_TANH: return z * logistic(gelu_tanh_arg(z));
        default: return z;
    }
}
__device__ __forceinline__ float act_slope(float z, int act) {
    switch (act) {
        case L_SILU: { const float s = logistic(z); return s * fmaf(z, 1.f - s, 1.f); }
        case L_RELU: return z > 0.f ? 1.f : (z != z ? z : 0.f);
        case L_GELU: { float e; const float c = normal_cdf(z, e); return fmaf(0.3989422804014327f * z, e, c); }
        case L_GELU_TANH: {
            const float s = logistic(gelu_tanh_arg(z));
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
__device__ __forceinline__ void finish_row(const LinArgs& p, long m, int n0, int n, float (&v)[V], const float (&bias)[V]) {
    if (n <= 0) return;
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] += bias[i];
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
        float t[V];
        ldv_n<T, V>(reinterpret_cast<const T*>(p.res) + m * p.ldres + n0, n, t);
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] += t[i];
    }
    stv_n<T, V>(reinterpret_cast<T*>(p.y) + m * p.ldy + n0, n, v);
}
template <class T, int V>
__device__ __forceinline__ void load_bias(const LinArgs& p, int n0, int n, float (&b)[V]) {
#pragma unroll
    for (int i = 0; i < V; ++i) b[i] = 0.f;
    if (p.bias && n > 0) ldv_n<T, V>(reinterpret_cast<const T*>(p.bias) + n0, n, b);
}

// LDS-DMA with a scalar base and a 32-bit offset a lane: advancing along k costs no vector instruction
__device__ __forceinline__ void lds_dma16_s(const void* base, unsigned off, unsigned lds_dst) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds_dst), "v"(off), "s"(base) : "memory", "m0");
}

// One BM x BN tile of the result (and one range of k): WM x WN waves, 64 k a stage.
//   * stages arrive by LDS-DMA in two slots; the request for stage S + 2 goes out when the second half of stage S begins, one barrier a stage;
//   * the fragments of the next 32 k are read from LDS while these 32 k run on the matrix cores (two register sets), so no product waits for LDS;
//   * operand images: KC, rows of 128 bytes (whole cache lines: with 64-byte rows each line was fetched twice, 581 us for 16384 x 8192 x 2048 where
//     the MC x MC product of the same size took 458) whose 16-byte piece j lies at j ^ f(row); MC, 128-column planes of 256-byte k rows whose piece j lies
//     at j ^ 2 g(k row), read through the transpose read.  f, g spread the rows that one read touches over all banks; the permutation is applied to
//     the global address of the DMA lane;
//   * the operands are swapped in the instruction (B in the A slot): a lane's four accumulators are four consecutive columns of one row;
//   * blocks that run on one XCD (block number mod 8) take neighbouring tiles, 8 rows of tiles at a time: an operand's panel is read from HBM once an XCD.
template <class T, bool AMC, bool BMC, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN, 2) void lin_tile_kernel(const LinArgs p) {
    constexpr int TM = BM / WM, TN = BN / WN, FA = TM / 16, FB = TN / 16;                 // a wave's part and its fragments
    constexpr int AB = BM * 128, STAGE = (BM + BN) * 128, DMAS = STAGE / (1024 * WM * WN);  // bytes of a stage's images; DMAs of 1 KB a wave
    static_assert(TN == 64 && TM % 64 == 0 && STAGE * 2 == 16384 * WM * WN && AB / 1024 % DMAS == 0, "16 KB a wave; a wave's DMAs belong to one operand");
    extern __shared__ __attribute__((aligned(1024))) unsigned char lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int i16 = lane & 15, q = lane >> 4;
    const int tiles = p.tiles_m * p.tiles_n;
    const int split = blockIdx.x / tiles, id = blockIdx.x - split * tiles;
    int tm, tn;
    {
        const int x = id & 7, per = tiles >> 3, more = tiles & 7;
        const int t = x * per + (x < more ? x : more) + (id >> 3);
        const int band = 8 * p.tiles_n, g = t / band, in = t - g * band;               // bands of 8 tile rows, walked column by column
        const int high = p.tiles_m - 8 * g < 8 ? p.tiles_m - 8 * g : 8;
        tn = in / high;
        tm = 8 * g + in - tn * high;
    }
    const int m0 = tm * BM, n0 = tn * BN;
    const int kb = split * p.k_per_split, ke = kb + p.k_per_split < p.K ? kb + p.k_per_split : p.K;
    const int stages = (ke - kb + 63) / 64, full = (ke - kb) / 64;
    const unsigned base = (unsigned)(size_t)lds;

    // This wave's DMAs: DMAS of 1 KB, of operand A (waves of the first AB bytes) or B.  Lane l reads 16 bytes of
    //   KC: row 8 d + l / 8, piece (l % 8) ^ f(row);     MC: k row 4 d + l / 16 of a plane, piece (l % 16) ^ 2 g(k row).
    // Rows past the operand repeat its last row or piece: they reach results that are not written.
    const bool isa = wave * DMAS < AB / 1024;
    const int d0 = isa ? wave * DMAS : wave * DMAS - AB / 1024;
    auto place = [&](bool mc, int rows, int r0, int d, int& row, int& k) {
        if (!mc) {
            const int r = 8 * d + (lane >> 3);
            k = 8 * ((lane & 7) ^ (r >> 1 & 7));
            row = r0 + r < rows ? r0 + r : rows - 1;
        } else {
            k = 4 * (d & 15) + (lane >> 4);
            const int c = r0 + 128 * (d >> 4) + 8 * ((lane & 15) ^ (2 * ((k & 3) | (((k >> 3) & 1) << 2))));
            row = c < rows ? c : (rows - 1) & ~7;
        }
    };
    auto where = [&](int d, int& k) -> unsigned {                         // byte offset from the operand's stage base
        int row;
        if (isa) {
            place(AMC, p.M, m0, d, row, k);
            return (unsigned)(2 * (AMC ? k * p.lda + row : (row - m0) * p.lda + k));
        }
        place(BMC, p.N, n0, d, row, k);
        return (unsigned)(2 * (BMC ? k * p.ldb + row : (row - n0) * p.ldb + k));
    };
    const u16* const mine = isa ? (AMC ? p.A + (long)kb * p.lda : p.A + (long)m0 * p.lda + kb) : (BMC ? p.B + (long)kb * p.ldb : p.B + (long)n0 * p.ldb + kb);
    const long step = isa ? (AMC ? 64 * p.lda : 64) : (BMC ? 64 * p.ldb : 64);
    unsigned off[DMAS];
#pragma unroll
    for (int e = 0; e < DMAS; ++e) { int k; off[e] = where(d0 + e, k); }
    auto fetch = [&](int s) {
        const unsigned dst = base + (s & 1) * STAGE + wave * (DMAS * 1024);
        const u16* src = mine + s * step;
        if (s < full) {
#pragma unroll
            for (int e = 0; e < DMAS; ++e) lds_dma16_s(src, off[e], dst + e * 1024);
        } else {                                                          // the last, partial stage: what lies past ke reads a line of zeros
#pragma unroll 1
            for (int e = 0; e < DMAS; ++e) {
                int k;
                const unsigned o = where(d0 + e, k);
                cdae_lds_dma16(kb + 64 * s + k < ke ? (const void*)((const char*)src + o) : (const void*)g_zero_lin16, dst + e * 1024);
            }
        }
    };

    const int wm = wave / WN, wn = wave - wm * WN;
    // lane offsets of the fragment reads: KC at the row's piece q (first half of a stage; the second half's is 64 bytes away, ^ 64), MC at k row 8 q + ..
    const int kq = 8 * q + (i16 >> 2), mcs = 2 * ((kq & 3) | (((kq >> 3) & 1) << 2));
    const int ra = (wm * TM + i16) * 128 + ((q ^ (i16 >> 1 & 7)) * 16);
    const int rb = (wn * TN + i16) * 128 + ((q ^ (i16 >> 1 & 7)) * 16);
    auto frag_mc = [&](const unsigned char* img, int r0, int h) -> u32x4 {      // 8 k (32 h + 8 q .. + 7) of column r0 + i16
        const unsigned char* src = img + (r0 >> 7) * 16384 + h * 8192 + kq * 256 + (((((r0 & 127) >> 3) + ((i16 & 3) >> 1)) ^ mcs) * 16) + (i16 & 1) * 8;
        const fp16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4f16((__attribute__((address_space(3))) fp16x4*)(src));
        const fp16x4 c = __builtin_amdgcn_ds_read_tr16_b64_v4f16((__attribute__((address_space(3))) fp16x4*)(src + 4 * 256));
        const u32x2 a2 = __builtin_bit_cast(u32x2, a), c2 = __builtin_bit_cast(u32x2, c);
        u32x4 v;
        v[0] = a2[0]; v[1] = a2[1]; v[2] = c2[0]; v[3] = c2[1];
        return v;
    };
    auto read = [&](int slot, int h, u32x4 (&fa)[FA], u32x4 (&fb)[FB]) {
        const unsigned char* as = lds + slot * STAGE;
        const unsigned char* bs = as + AB;
#pragma unroll
        for (int b = 0; b < FB; ++b) {
            if constexpr (BMC) fb[b] = frag_mc(bs, wn * TN + b * 16, h);
            else fb[b] = *reinterpret_cast<const u32x4*>(bs + (rb ^ (64 * h)) + b * 2048);
        }
#pragma unroll
        for (int a = 0; a < FA; ++a) {
            if constexpr (AMC) fa[a] = frag_mc(as, wm * TM + a * 16, h);
            else fa[a] = *reinterpret_cast<const u32x4*>(as + (ra ^ (64 * h)) + a * 2048);
        }
    };
    f32x4 acc[FA][FB];
#pragma unroll
    for (int a = 0; a < FA; ++a)
#pragma unroll
        for (int b = 0; b < FB; ++b) acc[a][b] = (f32x4){0.f, 0.f, 0.f, 0.f};
    auto multiply = [&](u32x4 (&fa)[FA], u32x4 (&fb)[FB]) {
#pragma unroll
        for (int a = 0; a < FA; ++a)
#pragma unroll
            for (int b = 0; b < FB; ++b) acc[a][b] = Mfma<T>::go(fb[b], fa[a], acc[a][b]);       // rows of the result: n (4 q + r), columns: m (i16)
    };

    u32x4 fa[2][FA], fb[2][FB];
    fetch(0);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (stages > 1) fetch(1);
    read(0, 0, fa[0], fb[0]);
    for (int s = 0; s < stages; ++s) {
        read(s & 1, 1, fa[1], fb[1]);
        multiply(fa[0], fb[0]);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");                  // stage s + 1 has landed (here; behind the barrier for every wave) ...
        __syncthreads();                                                  // ... and every wave has read the whole of stage s
        if (s + 2 < stages) fetch(s + 2);
        if (s + 1 < stages) read((s + 1) & 1, 0, fa[0], fb[0]);
        multiply(fa[1], fb[1]);
    }

    // Epilogue through the wave's own 16 KB of the stages, 64 rows at a time, so that one short loop serves every variant (unrolled over the accumulators
    // it was 60 000 instructions) and rows leave as whole lines.  Row r's 16-byte piece j (4 columns) lies at j ^ (r & 15).
    unsigned char* const own = lds + wave * 16384;
    const int cl = 8 * (lane & 7), n = n0 + wn * TN + cl, have = p.N - n;
    float bias[8];
    load_bias<T, 8>(p, n, have, bias);
#pragma unroll
    for (int h = 0; h < FA / 4; ++h) {
#pragma unroll
        for (int a = 0; a < 4; ++a)
#pragma unroll
            for (int b = 0; b < FB; ++b) *reinterpret_cast<f32x4*>(own + (16 * a + i16) * 256 + (((4 * b + q) ^ i16) * 16)) = acc[4 * h + a][b];
#pragma unroll 1
        for (int i = 0; i < 8; ++i) {
            const int r = 8 * i + (lane >> 3), m = m0 + wm * TM + 64 * h + r;
            const f32x4 lo = *reinterpret_cast<const f32x4*>(own + r * 256 + ((((cl >> 2)) ^ (r & 15)) * 16));
            const f32x4 hi = *reinterpret_cast<const f32x4*>(own + r * 256 + ((((cl >> 2) + 1) ^ (r & 15)) * 16));
            float v[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
            if (m < p.M && have > 0) {
                if (p.splits > 1) stv_n<float, 8>(p.slab + ((long)split * p.M + m) * p.N + n, have, v);
                else finish_row<T, 8>(p, m, n, have, v, bias);
            }
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
        float bias[8];
        load_bias<T, 8>(p, n, have, bias);
        finish_row<T, 8>(p, m, n, have, v, bias);
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

// Tile and splits of the sum over k.  256 x 256 tiles (one block a CU) where they alone fill the CUs; else 128 x 128 tiles (two a CU), and where those
// leave most of the 512 slots empty the sum is split, a split keeping at least 256 of k.
struct Plan { int bm, splits; };
Plan plan(int M, int N, int K) {
    const long big = ((M + 255L) / 256) * ((N + 255L) / 256), tiles = ((M + 127L) / 128) * ((N + 127L) / 128);
    if (big >= 256) return {256, 1};
    long s = 512 / (tiles > 0 ? tiles : 1);
    if (s > K / 256) s = K / 256;
    if (s > 64) s = 64;
    return {128, s < 1 ? 1 : (int)s};
}
size_t gemm_ws(int M, int N, int K) {
    const int s = plan(M, N, K).splits;
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

template <class T, bool AMC, bool BMC, int BM, int WN>
int launch_tiles(const LinArgs& p, unsigned blocks, hipStream_t st) {
    constexpr int smem = 2 * 2 * BM * 128;
    auto* kernel = &lin_tile_kernel<T, AMC, BMC, BM, BM, 2, WN>;
    if (smem > 65536 && hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, smem) != hipSuccess)
        return cdae_fail("lin16: hipFuncSetAttribute(max dynamic LDS) failed");
    hipLaunchKernelGGL(kernel, dim3(blocks), dim3(128 * WN), smem, st, p);
    return hipGetLastError() == hipSuccess ? 0 : cdae_fail("lin16: launch failed");
}
template <class T, bool AMC, bool BMC>
int product(LinArgs p, char* ws, hipStream_t st) {
    const Plan pl = plan(p.M, p.N, p.K);
    p.tiles_m = (p.M + pl.bm - 1) / pl.bm; p.tiles_n = (p.N + pl.bm - 1) / pl.bm;
    p.splits = pl.splits;
    p.k_per_split = ((p.K + p.splits - 1) / p.splits + 63) / 64 * 64;
    p.splits = (p.K + p.k_per_split - 1) / p.k_per_split;
    p.slab = (float*)ws;
    const long blocks = (long)p.tiles_m * p.tiles_n * p.splits;
    // (a lane's offset inside a stage is 32 bits: 256 rows, or 64 k rows and the columns)
    if (blocks > (1L << 22) || 512 * (AMC ? p.lda / 4 + p.M / 256 : p.lda) >= (1L << 32) || 512 * (BMC ? p.ldb / 4 + p.N / 256 : p.ldb) >= (1L << 32)) return cdae_fail("lin16: product too large");
    if (pl.bm == 256 ? launch_tiles<T, AMC, BMC, 256, 4>(p, (unsigned)blocks, st) : launch_tiles<T, AMC, BMC, 128, 2>(p, (unsigned)blocks, st)) return -1;
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
