// lin16.hip — linear layers on bf16 / f16 rows with activation and residual in the product's epilogue, and their gradients (gfx950):
//
//     z = x W^T + b,     y = act(z) + res                                     x [M][K], W [N][K]
//     dz = dy o act'(z),   dx = dz W,   dW = dz^T x,   db = sum over rows of dz
//
// All three products are C[m][n] = sum over k of A(m, k) B(n, k) with an operand's k running along its rows (KC) or across them (MC):
// forward KC x KC, data gradient KC x MC (k = N), weight gradient MC x MC (k = M).  MC fragments come out of LDS through the hardware transpose read.
#include <hip/hip_runtime.h>
#include <math.h>

#include <atomic>
#include <initializer_list>
#include <type_traits>

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

// Activations and slopes for results of 16 bits, on the exp2 and reciprocal instructions.  An exponential 2^t is off by t steps of fp32, relative to itself
// (t is rounded), everything else by a few: what is left of the normal distribution at z = -12 is good to 1e-5.
//   logistic(a) = 1 / (1 + 2^(-a log2 e)): where 2^t overflows the reciprocal is 0, the limit.
//   The tail of the normal distribution beyond |z| is exp(-z^2 / 2) times a function that falls like 1 / |z|: t Q(t) with t = 1 / (1 + 0.373 |z| / sqrt 2) and Q
//   of degree 6, fitted so that its largest RELATIVE error is least, 6e-7 (9e-7 in fp32) up to |z| = 13.5, where the exponential is below fp32's numbers.  (A fit
//   of least absolute error, 1.5e-7, was 6e-4 off at z = -4.2 and 3 % at -8.)  The exponential is the density that the slope needs.  16 instructions where
//   the library's erf takes about 40, and the epilogue is bound by them (12.6 million values of a 8192 x 1536 result: 40 instructions a value are 13 us of
//   all vector units).
__device__ __forceinline__ float logistic(float a) { return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.4426950408889634f * a)); }
__device__ __forceinline__ float normal_cdf(float z, float& e) {
    const float t = __builtin_amdgcn_rcpf(fmaf(0.26375083f, fabsf(z), 1.f));
    e = __builtin_amdgcn_exp2f(-0.72134752044448170f * z * z);                                       // exp(-z^2 / 2)
    const float q = fmaf(t, fmaf(t, fmaf(t, fmaf(t, fmaf(t, fmaf(t, -0.069476977f, 0.20486708f), -0.0779428855f), 0.149652228f), 0.0800528601f), 0.107777007f), 0.105070531f);
    const float tail = t * q * e;                                                                    // of the side that z points to
    return z < 0.f ? tail : 1.f - tail;
}
__device__ __forceinline__ float gelu_tanh_arg(float z) { return 1.5957691216057308f * z * fmaf(0.044715f * z, z, 1.f); }      // 0.5 (1 + tanh a) = logistic(2 a)

template <int ACT>
__device__ __forceinline__ float act_of(float z) {
    if constexpr (ACT == L_SILU) return z * logistic(z);
    else if constexpr (ACT == L_RELU) return z < 0.f ? 0.f : z;
    else if constexpr (ACT == L_GELU) { float e; return z * normal_cdf(z, e); }
    else if constexpr (ACT == L_GELU_TANH) return z * logistic(gelu_tanh_arg(z));
    else return z;
}
template <int ACT>
__device__ __forceinline__ float slope_of(float z) {
    if constexpr (ACT == L_SILU) { const float s = logistic(z); return s * fmaf(z, 1.f - s, 1.f); }
    else if constexpr (ACT == L_RELU) return z > 0.f ? 1.f : z * 0.f;                 // (not a number stays one)
    else if constexpr (ACT == L_GELU) { float e; const float c = normal_cdf(z, e); return fmaf(0.3989422804014327f * z, e, c); }
    else if constexpr (ACT == L_GELU_TANH) {
        const float s = logistic(gelu_tanh_arg(z));
        return s * fmaf(z * (1.f - s), 1.5957691216057308f * fmaf(0.134145f * z, z, 1.f), 1.f);
    } else return 1.f;
}
// CALL(activation) with the number as a constant: one branch for all values of a thread
#define LIN_ACT(act, CALL)                                            \
    switch (act) {                                                    \
        case L_SILU: CALL(L_SILU); break;                             \
        case L_RELU: CALL(L_RELU); break;                             \
        case L_GELU: CALL(L_GELU); break;                             \
        case L_GELU_TANH: CALL(L_GELU_TANH); break;                   \
        default: break;                                               \
    }
// The pre-activation is kept for the backward in f16 whatever the rows' type: its 11 bits cost the slope a quarter of what the rounding of dz to
// bf16 costs.  Beyond f16's range it becomes infinite, and the slope there is taken at the range's end, where every slope has long reached its limit.
// Below that range it becomes zero, where every slope but ReLU's is continuous: finish_row keeps ReLU's positive values positive.
__device__ __forceinline__ float kept_z(F16 v) { const float z = ld1(v); return fabsf(z) > 65504.f ? copysignf(65504.f, z) : z; }

struct LinArgs {
    const u16* A; long lda;                 // KC: [M][K], MC: [K][M]
    const u16* B; long ldb;                 // KC: [N][K], MC: [K][N]
    int M, N, K;
    const u16* bias; const u16* res; long ldres; u16* y; long ldy; _Float16* z; long ldz; int act;
    float* slab; int splits, k_per_split;   // splits > 1: partial sums [split][M][N] instead of the epilogue
    int tiles_m, tiles_n;
    int past;                               // the result is larger than the caches: written past them
    const float* sums; void* db; int sum_rows;      // weight gradient beside the data gradient: the bias gradient's partial sums [sum_rows][M] and db, or NULL
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

// v[0..n) of row m from column n0: bias, activation, residual (in r), rounding
template <class T, int V>
__device__ __forceinline__ void finish_row(const LinArgs& p, long m, int n0, int n, float (&v)[V], const float (&bias)[V], const Pack<T, V>& r) {
    if (n <= 0) return;
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] += bias[i];
    if (p.z) {
        _Float16* zp = p.z + m * p.ldz + n0;
        Pack<F16, V> k;
#pragma unroll
        for (int i = 0; i < V; ++i) k.v[i].h = (_Float16)v[i];
        if (p.act == L_RELU)                                               // (its slope jumps at zero: what is above stays above, as f16's smallest number)
#pragma unroll
            for (int i = 0; i < V; ++i) if (v[i] > 0.f) k.v[i].h = (_Float16)fmaxf(v[i], 0x1p-24f);
        if (n >= V) store_past(reinterpret_cast<Pack<F16, V>*>(zp), k);    // (the backward reads it, long after)
        else
#pragma unroll
            for (int i = 0; i < V; ++i) if (i < n) zp[i] = k.v[i].h;
    }
#define LIN_CALL(A) _Pragma("unroll") for (int i = 0; i < V; ++i) v[i] = act_of<A>(v[i])
    LIN_ACT(p.act, LIN_CALL)
#undef LIN_CALL
    if (p.res)
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] += ld1(r.v[i]);
    T* const yp = reinterpret_cast<T*>(p.y) + m * p.ldy + n0;
    if (n >= V && p.past) {
        Pack<T, V> w;
#pragma unroll
        for (int i = 0; i < V; ++i) st1(w.v[i], v[i]);
        store_past(reinterpret_cast<Pack<T, V>*>(yp), w);
    } else stv_n<T, V>(yp, n, v);
}
// the residual of a row's n values (present ones only)
template <class T, int V>
__device__ __forceinline__ void load_res(const LinArgs& p, long m, int n0, int n, Pack<T, V>& r) {
    const T* at = reinterpret_cast<const T*>(p.res) + m * p.ldres + n0;
    if (n >= V) r = *reinterpret_cast<const Pack<T, V>*>(at);
    else
#pragma unroll
        for (int i = 0; i < V; ++i) if (i < n) r.v[i] = at[i];
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
//   * stages arrive by LDS-DMA in SLOTS slots; the request for stage S + SLOTS goes out when the second half of stage S begins; counted vmcnt, one
//     barrier a stage;
//   * the fragments of the next 32 k are read from LDS while these 32 k run on the matrix cores (two register sets); reads, requests and products
//     are interleaved by hand;
//   * operand images: KC, rows of 128 bytes (whole cache lines: with 64-byte rows each line was fetched twice, 581 us for 16384 x 8192 x 2048 where the
//     MC x MC product of the same size took 458) whose
//     16-byte piece j lies at j ^ f(row); MC, planes of up to 128 columns whose k row's piece j lies at j ^ 2 g(k row), read through the transpose
//     read.  f, g spread the rows that one read touches over all banks; the permutation is applied to the global address of the DMA lane;
//   * the operands are swapped in the instruction (B in the A slot): a lane's four accumulators are four consecutive columns of one row;
//   * blocks that run on one XCD (block number mod 8) take neighbouring tiles, 8 rows of tiles at a time: an operand's panel is read from HBM once an XCD.
template <class T, bool AMC, bool BMC, int BM, int BN, int WM, int WN, int SLOTS>
__device__ __forceinline__ void lin_tile(const LinArgs& p, const int block, unsigned char* const lds) {
    constexpr int TM = BM / WM, TN = BN / WN, FA = TM / 16, FB = TN / 16;                 // a wave's part and its fragments
    constexpr int AB = BM * 128, STAGE = (BM + BN) * 128, DMAS = STAGE / (1024 * WM * WN);  // bytes of a stage's images; DMAs of 1 KB a wave
    constexpr int PA = BM < 128 ? BM : 128, PB = BN < 128 ? BN : 128;                     // columns of an MC plane
    static_assert(TN == 64 && AB / 1024 % DMAS == 0 && PA == PB, "64 columns a wave; a wave's DMAs belong to one operand");
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int i16 = lane & 15, q = lane >> 4;
    const int tiles = p.tiles_m * p.tiles_n;
    const int split = block / tiles, id = block - split * tiles;
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
    //   KC: row 8 d + l / 8, piece (l % 8) ^ f(row);     MC (128 columns): k row 4 d + l / 16 of a plane, piece (l % 16) ^ 2 g(k row);
    //   MC (64 columns): k row 8 d + l / 8, piece (l % 8) ^ 2 g(k row).
    // Rows past the operand repeat its last row or piece: they reach results that are not written.
    const bool isa = wave * DMAS < AB / 1024;
    const int d0 = isa ? wave * DMAS : wave * DMAS - AB / 1024;
    auto place = [&](bool mc, int rows, int r0, int d, int& row, int& k) {
        if (!mc) {
            const int r = 8 * d + (lane >> 3);
            k = 8 * ((lane & 7) ^ (r >> 1 & 7));
            row = r0 + r < rows ? r0 + r : rows - 1;
        } else {
            k = PA == 128 ? 4 * (d & 15) + (lane >> 4) : 8 * d + (lane >> 3);
            const int c = PA == 128 ? r0 + 128 * (d >> 4) + 8 * ((lane & 15) ^ (2 * ((k & 3) | (((k >> 3) & 1) << 2)))) : r0 + 8 * ((lane & 7) ^ (2 * ((k >> 1 & 1) | (k >> 3 & 1) << 1)));
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
        const unsigned dst = base + s % SLOTS * STAGE + wave * (DMAS * 1024);
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
    const int kq = 8 * q + (i16 >> 2), mcs = PA == 128 ? 2 * ((kq & 3) | (((kq >> 3) & 1) << 2)) : 2 * ((kq >> 1 & 1) | (kq >> 3 & 1) << 1);
    const int ra = (wm * TM + i16) * 128 + ((q ^ (i16 >> 1 & 7)) * 16);
    const int rb = (wn * TN + i16) * 128 + ((q ^ (i16 >> 1 & 7)) * 16);
    auto frag_mc = [&](const unsigned char* img, int r0, int h) -> u32x4 {      // 8 k (32 h + 8 q .. + 7) of column r0 + i16
        const unsigned char* src = img + r0 / PA * (PA * 128) + h * (PA * 64) + kq * (PA * 2) + ((((r0 % PA >> 3) + ((i16 & 3) >> 1)) ^ mcs) * 16) + (i16 & 1) * 8;
        const fp16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4f16((__attribute__((address_space(3))) fp16x4*)(src));
        const fp16x4 c = __builtin_amdgcn_ds_read_tr16_b64_v4f16((__attribute__((address_space(3))) fp16x4*)(src + 8 * PA));
        const u32x2 a2 = __builtin_bit_cast(u32x2, a), c2 = __builtin_bit_cast(u32x2, c);
        u32x4 v;
        v[0] = a2[0]; v[1] = a2[1]; v[2] = c2[0]; v[3] = c2[1];
        return v;
    };
    auto read_a = [&](int slot, int h, int a) -> u32x4 {
        const unsigned char* as = lds + slot * STAGE;
        if constexpr (AMC) return frag_mc(as, wm * TM + a * 16, h);
        else return *reinterpret_cast<const u32x4*>(as + (ra ^ (64 * h)) + a * 2048);
    };
    auto read_b = [&](int slot, int h, int b) -> u32x4 {
        const unsigned char* bs = lds + slot * STAGE + AB;
        if constexpr (BMC) return frag_mc(bs, wn * TN + b * 16, h);
        else return *reinterpret_cast<const u32x4*>(bs + (rb ^ (64 * h)) + b * 2048);
    };
    f32x4 acc[FA][FB];
#pragma unroll
    for (int a = 0; a < FA; ++a)
#pragma unroll
        for (int b = 0; b < FB; ++b) acc[a][b] = (f32x4){0.f, 0.f, 0.f, 0.f};
    // 32 k on the matrix cores from set `cur`, a row of fragments at a time; between the rows the next half's fragments are read into the other set
    // and (FETCH) the DMAs of a later stage issued.  All of a stage's DMAs in one go behind the barrier held every wave up for the 16 cycles a
    // KB that the four or eight waves' requests take: 1665 cycles a stage of a lone 128 x 128 block against 512 of products.
    u32x4 fa[2][FA], fb[2][FB];
    auto half = [&](auto fetching, int cur, bool more, int slot, int h, const u16* src, unsigned dst) {
        constexpr bool FETCH = decltype(fetching)::value;
#pragma unroll
        for (int a = 0; a < FA; ++a) {
            if constexpr (FETCH)
#pragma unroll
                for (int e = a * DMAS / FA; e < (a + 1) * DMAS / FA; ++e) lds_dma16_s(src, off[e], dst + e * 1024);
            if (more) {
#pragma unroll
                for (int b = a * FB / FA; b < (a + 1) * FB / FA; ++b) fb[cur ^ 1][b] = read_b(slot, h, b);
                fa[cur ^ 1][a] = read_a(slot, h, a);
            }
#pragma unroll
            for (int b = 0; b < FB; ++b) acc[a][b] = Mfma<T>::go(fb[cur][b], fa[cur][a], acc[a][b]);       // rows of the result: n (4 q + r), columns: m (i16)
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    using Yes = std::true_type;
    using No = std::false_type;
#pragma unroll
    for (int s = 0; s < SLOTS; ++s) if (s < stages) fetch(s);
    if (stages >= SLOTS) asm volatile("s_waitcnt vmcnt(%0)" ::"n"((SLOTS - 1) * DMAS) : "memory");
    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
#pragma unroll
    for (int b = 0; b < FB; ++b) fb[0][b] = read_b(0, 0, b);
#pragma unroll
    for (int a = 0; a < FA; ++a) fa[0][a] = read_a(0, 0, a);
    int slot = 0, s = 0;
    // behind the barrier: stage s + 1 has landed for every wave, and every wave has read the whole of stage s, whose slot is then free
    for (; s + SLOTS < full; ++s) {
        const int after = slot == SLOTS - 1 ? 0 : slot + 1;
        half(No{}, 0, true, slot, 1, nullptr, 0u);
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"((SLOTS - 2) * DMAS) : "memory");
        __syncthreads();
        half(Yes{}, 1, true, after, 0, mine + (s + SLOTS) * step, base + slot * STAGE + wave * (DMAS * 1024));
        slot = after;
    }
    for (; s < stages; ++s) {                                             // the last stages: nothing or a partial stage left to request
        const int after = slot == SLOTS - 1 ? 0 : slot + 1;
        half(No{}, 0, true, slot, 1, nullptr, 0u);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (s + SLOTS < stages) fetch(s + SLOTS);
        half(No{}, 1, s + 1 < stages, after, 0, nullptr, 0u);
        slot = after;
    }

    // Epilogue through the wave's own part of the stages, up to 64 rows at a time, so that one short loop serves every variant (unrolled over the
    // accumulators it was 60 000 instructions) and rows leave as whole lines.  Row r's 16-byte piece j (4 columns) lies at j ^ (r & 15).
    constexpr int PR = FA < 4 ? FA : 4, RB = 2 * PR < 4 ? 2 * PR : 4;     // 16-row groups of a pass; 8-row groups whose residuals are on their way together
    static_assert(PR * 4096 * WM * WN <= SLOTS * STAGE, "the epilogue fits the stages");
    unsigned char* const own = lds + wave * (PR * 4096);
    const int cl = 8 * (lane & 7), n = n0 + wn * TN + cl, have = p.N - n;
    float bias[8];
    load_bias<T, 8>(p, n, have, bias);
#pragma unroll
    for (int h = 0; h < FA / PR; ++h) {
#pragma unroll
        for (int a = 0; a < PR; ++a)
#pragma unroll
            for (int b = 0; b < FB; ++b) *reinterpret_cast<f32x4*>(own + (16 * a + i16) * 256 + (((4 * b + q) ^ i16) * 16)) = acc[PR * h + a][b];
        asm volatile("" ::: "memory");                                    // (other lanes' values: the wave's LDS accesses run in the order written)
#pragma unroll 1
        for (int i = 0; i < 2 * PR; i += RB) {
            const int r0 = 8 * i + (lane >> 3);
            const long mr = m0 + wm * TM + 16 * PR * h + r0;
            Pack<T, 8> res[RB];
            if (p.res && p.splits == 1)
#pragma unroll
                for (int e = 0; e < RB; ++e) load_res<T, 8>(p, mr + 8 * e < p.M ? mr + 8 * e : p.M - 1, have > 0 ? n : 0, have > 0 ? have : 0, res[e]);
#pragma unroll
            for (int e = 0; e < RB; ++e) {
                const int r = r0 + 8 * e;
                const long m = mr + 8 * e;
                const f32x4 lo = *reinterpret_cast<const f32x4*>(own + r * 256 + (((cl >> 2) ^ (r & 15)) * 16));
                const f32x4 hi = *reinterpret_cast<const f32x4*>(own + r * 256 + ((((cl >> 2) + 1) ^ (r & 15)) * 16));
                float v[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
                if (m < p.M && have > 0) {
                    if (p.splits > 1) stv_n<float, 8>(p.slab + ((long)split * p.M + m) * p.N + n, have, v);
                    else finish_row<T, 8>(p, m, n, have, v, bias, res[e]);
                }
            }
        }
        asm volatile("" ::: "memory");
    }
}
// the column sums of the slope pass's blocks, in order: 32 columns x THREADS / 32 lanes of blocks
template <class T, int THREADS>
__device__ __forceinline__ void fold_bias(const float* __restrict__ part, int blocks, int N, T* __restrict__ db, int job, float* sh) {
    constexpr int Q = THREADS / 32;
    const int cl = threadIdx.x & 31, q = threadIdx.x >> 5, c = job * 32 + cl;
    const float* at = part + (c < N ? c : N - 1);
    float s = 0.f;
#pragma unroll 4
    for (int b = q; b < blocks; b += Q) s += at[(long)b * N];
    sh[q * 33 + cl] = s;
    __syncthreads();
    if (q || c >= N) return;
#pragma unroll
    for (int i = 1; i < Q; ++i) s += sh[i * 33 + cl];
    st1(db[c], s);
}
template <class T, bool AMC, bool BMC, int BM, int WM, int WN, int SLOTS>
__global__ __launch_bounds__(64 * WM * WN, 2) void lin_tile_kernel(const LinArgs p) {
    extern __shared__ __attribute__((aligned(1024))) unsigned char lds[];
    lin_tile<T, AMC, BMC, BM, BM, WM, WN, SLOTS>(p, blockIdx.x, lds);
}
// Both products of a backward pass in one launch: the weight gradient's blocks, then (from a multiple of 8, for the XCDs) the data gradient's.  Each alone
// leaves CUs without work at its end, or from the beginning.  So do both together, and the fold of the bias gradient's sums is done there, by the last blocks
// (8192 x 384 -> 1536, a whole training pass: 76.6 us with the fold in a launch of its own, 74.2 so; behind a lone product that fills all CUs, 8192 x 2048 ->
// 512, 86.0 and 87.7).
template <class T, int BM, int WM, int WN, int SLOTS>
__global__ __launch_bounds__(64 * WM * WN, 2) void lin_pair_kernel(const LinArgs pw, const LinArgs px, const int blocks_w, const int bias_from) {
    extern __shared__ __attribute__((aligned(1024))) unsigned char lds[];
    const int second = (blocks_w + 7) & ~7, block = blockIdx.x;
    if (block >= bias_from) fold_bias<T, 64 * WM * WN>(pw.sums, pw.sum_rows, pw.M, reinterpret_cast<T*>(pw.db), block - bias_from, reinterpret_cast<float*>(lds));
    else if (block < blocks_w) lin_tile<T, true, true, BM, BM, WM, WN, SLOTS>(pw, block, lds);
    else if (block >= second) lin_tile<T, false, true, BM, BM, WM, WN, SLOTS>(px, block - second, lds);
}

// partial sums of the splits, added in order, then the epilogue: 4 columns a thread, eight splits in flight
template <class T>
__global__ __launch_bounds__(256) void lin_finish_kernel(const LinArgs p) {
    const long per = (p.N + 3) / 4, total = per * p.M, plane = (long)p.M * p.N;
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long)gridDim.x * 256) {
        const long m = i / per;
        const int n = (int)(i - m * per) * 4, have = p.N - n;
        float v[4] = {0.f, 0.f, 0.f, 0.f};
        const float* at = p.slab + m * p.N + n;
        if (have >= 4) {
#pragma unroll 8
            for (int s = 0; s < p.splits; ++s) {
                const Pack<float, 4> t = *reinterpret_cast<const Pack<float, 4>*>(at + s * plane);
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] += t.v[e];
            }
        } else {
            for (int s = 0; s < p.splits; ++s)
                for (int e = 0; e < have; ++e) v[e] += at[s * plane + e];
        }
        float bias[4];
        load_bias<T, 4>(p, n, have, bias);
        Pack<T, 4> res;
        if (p.res) load_res<T, 4>(p, m, n, have, res);
        finish_row<T, 4>(p, m, n, have, v, bias, res);
    }
}

// [rows][cols] at any pitch and alignment -> dense rows padded with zeros to `pitch`, a multiple of 8; up to two operands in one launch
struct PadJob { const u16* src; u16* dst; long ld, rows; int cols, pitch; };
struct PadJobs { PadJob j[2]; };
__global__ __launch_bounds__(256) void lin_pad_kernel(const PadJobs jobs) {
    const PadJob p = jobs.j[blockIdx.y];
    const long per = p.pitch / 8, total = per * p.rows;
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long)gridDim.x * 256) {
        const long r = i / per;
        const int c = (int)(i - r * per) * 8, have = p.cols - c;
        const u16* s = p.src + r * p.ld + c;
        Pack<u16, 8> t;
        if (have >= 8) t = *reinterpret_cast<const Pack<u16, 8>*>(s);
        else
#pragma unroll
            for (int e = 0; e < 8; ++e) t.v[e] = e < have ? s[e] : (u16)0;
        u32x4 w;
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = (unsigned)t.v[2 * e] | (unsigned)t.v[2 * e + 1] << 16;
        *reinterpret_cast<u32x4*>(p.dst + r * p.pitch + c) = w;
    }
}

// dz = dy o act'(z) (written where wanted) and its column sums over a block's rows.  An HBM stream (three values of 2 bytes a result).  A block: 256
// columns x 8 lanes of rows, 8 columns a thread, one row at a time (8192 x 1536 with GELU, sums only: 14.2 us; two rows in flight 15.9, four 17.7, eight
// 29.3: the waves' number is worth more than their registers).  Loads and stores have no branches around them: the last thread of a row takes the row's
// LAST 8 values (its neighbour's are among them, written twice with the same value and summed once).  SMALL: rows of fewer than 8 values.
// dz is written in the rows' type because the matrix instructions take both operands in one 16-bit type.  That rounding is a second one, independent of the
// result's: relative to 64 bits dx and dw are 2.35e-3 off in bf16 and 3.0e-4 in fp16, where one rounding leaves 1.66e-3 and 2.1e-4 (measured at 8192 x 384 ->
// 1536 and 1021 x 393 -> 771).  A second operand with what the rounding drops would remove it and double both products.  The sums take dz unrounded.
template <class T, bool SMALL>
__global__ __launch_bounds__(256) void lin_slope_kernel(const T* __restrict__ dy, long lddy, const F16* __restrict__ z, long ldz, T* __restrict__ dz, long lddz,
                                                        float* __restrict__ part, T* __restrict__ db, int M, int N, int rows_per_block, int ncb, int act) {
    __shared__ float sh[8][256];
    const int cb = blockIdx.x % ncb, rb = blockIdx.x / ncb;
    const int cl = threadIdx.x & 31, rl = threadIdx.x >> 5;
    const int want = cb * 256 + cl * 8, c = SMALL ? 0 : want < N - 8 ? want : N - 8;
    const long r0 = (long)rb * rows_per_block, r1 = r0 + rows_per_block < M ? r0 + rows_per_block : M;
    float s[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    for (long r = r0 + rl; r < r1; r += 8) {
        Pack<T, 8> g;
        Pack<F16, 8> k;
        if constexpr (SMALL) {
#pragma unroll
            for (int e = 0; e < 8; ++e) { g.v[e] = dy[r * lddy + (e < N ? e : N - 1)]; if (act != L_NONE) k.v[e] = z[r * ldz + (e < N ? e : N - 1)]; }
        } else {
            g = *reinterpret_cast<const Pack<T, 8>*>(dy + r * lddy + c);
            if (act != L_NONE) k = *reinterpret_cast<const Pack<F16, 8>*>(z + r * ldz + c);
        }
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = ld1(g.v[e]);
#define LIN_CALL(A) _Pragma("unroll") for (int e = 0; e < 8; ++e) v[e] *= slope_of<A>(kept_z(k.v[e]))
        LIN_ACT(act, LIN_CALL)
#undef LIN_CALL
#pragma unroll
        for (int e = 0; e < 8; ++e) s[e] += v[e];
        if (!dz) continue;
        if constexpr (SMALL) {
            if (cl == 0)
#pragma unroll
                for (int e = 0; e < 8; ++e) st1(dz[r * lddz + e], e < N ? v[e] : 0.f);
        } else {
            stv<T, 8>(dz + r * lddz + c, v);
            if (N & 7 && want <= N && want + 8 > N)                        // the row's padding to a multiple of 8
                for (int e = N; e < lddz; ++e) st1(dz[r * lddz + e], 0.f);
        }
    }
    if (!part && !db) return;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const int at = c + e - cb * 256;                                   // (columns before this thread's own are its neighbour's sums too)
        if (SMALL ? cl == 0 : c + e >= want) sh[rl][at] = s[e];
    }
    __syncthreads();
    const int cc = cb * 256 + threadIdx.x;
    if (cc < N) {
        float t = 0.f;
#pragma unroll
        for (int r = 0; r < 8; ++r) t += sh[r][threadIdx.x];
        if (db) st1(db[cc], t);                                            // (one block of rows: its sums are the result)
        else part[(long)rb * N + cc] = t;
    }
}
template <class T>
__global__ __launch_bounds__(1024) void lin_bias_kernel(const float* __restrict__ part, int blocks, int N, T* __restrict__ db) {
    __shared__ float sh[32 * 33];
    fold_bias<T, 1024>(part, blocks, N, db, blockIdx.x, sh);
}

long up8(long v) { return (v + 7) / 8 * 8; }
bool al16(const void* p) { return ((size_t)p & 15) == 0; }
size_t up256(size_t b) { return (b + 255) / 256 * 256; }

// Tile, slots and splits of the sum over k: the cheapest by what a stage of 64 k and a tile's beginning and end cost (us), as measured on bf16 operands:
//     256 x 256, one block a CU                    1.5   9      16384 x 2048 x 8192 weight gradient, 256 tiles of 256 stages: 390 us (128 x 128 521)
//     128 x 128, four slots, one block a CU        0.5   3      8192 x 2048 -> 512 forward, 256 tiles of 32 stages: 21.3 us (two slots 25.1, 64 x 64 28.3, 256 x 256 42.4)
//     128 x 128, two slots, two blocks a CU        1.03  2.7    8192 x 384 -> 1536 forward, 768 tiles of 6 stages: 18.6 us (256 x 256 18.6, 64 x 64 25.8)
//     64 x 64, one block a CU                      0.26  2.5    1024 x 392 -> 768 data gradient, 112 tiles of 12 stages: 6.6 us (128 x 128 10.8)
//     64 x 64, two blocks a CU                     0.38  3.5    2048 x 1024 -> 1024 forward, 512 tiles of 16 stages: 9.4 us (128 x 128 12.1)
// (kernel times, launch after launch on the same operands; with other work between them the forward of 8192 x 2048 -> 512 with a residual takes 25.2.)
// A split costs a second launch (3.5) and its partial sums twice (6 TB/s): 1536 x 384 over 8192 rows 27.0 us in seven splits, 33.6 in one; 2048 x 1024 over
// 1024 rows 10.2 in one, 22.8 in two.
// (A call works its plan out anew, twice with the question for the workspace, so this is host time of every call: tables first, then the combinations.)
struct Kind { int bm, slots, at_once; double stage, ends; };
const Kind kinds[] = {{256, 2, 256, 1.5, 9.0}, {128, 4, 256, 0.5, 3.0}, {128, 2, 512, 1.03, 2.7}, {64, 4, 256, 0.26, 2.5}, {64, 4, 512, 0.38, 3.5}};
struct Forced {                              // (tests)
    int tile = cdae_tune(TUNE_LIN16_TILE), splits = cdae_tune(TUNE_LIN16_SPLITS);
    bool kind(const Kind& k) const { return !tile || (k.bm == kinds[tile - 1].bm && k.slots == kinds[tile - 1].slots); }
    bool split(int K, int s) const { return splits ? s == splits : s == 1 || K >= 256 * s; }
};
long tiles_of(const Kind& k, int M, int N) { return ((M + k.bm - 1L) / k.bm) * ((N + k.bm - 1L) / k.bm); }
int stages_of(int K, int s) { return ((K + s - 1) / s + 63) / 64; }
double split_cost(int M, int N, int s) { return s > 1 ? 3.5 + 8.0 * s * M * N / 6e6 : 0.0; }
size_t slab_of(int M, int N, int s) { return s > 1 ? up256((size_t)s * M * N * 4) : 0; }

struct Plan { int bm, slots, splits; double cost; };
Plan plan(int M, int N, int K) {
    static const int splits[] = {1, 2, 3, 4, 5, 6, 7, 8, 10, 12, 14, 16, 20, 24, 28, 32, 48, 64};
    const Forced forced;
    Plan best{256, 2, 1, 1e30};
    long tiles[5];
    for (int i = 0; i < 5; ++i) tiles[i] = forced.kind(kinds[i]) ? tiles_of(kinds[i], M, N) : 1L << 40;
    for (int s : splits) {
        if (!forced.split(K, s)) continue;
        const int stages = stages_of(K, s);
        const double extra = split_cost(M, N, s);
        for (int i = 0; i < 5; ++i) {
            const Kind& k = kinds[i];
            if (tiles[i] > (1L << 22) || (s > 1 && tiles[i] * s > k.at_once && !forced.splits)) continue;
            const double cost = (double)((tiles[i] * s + k.at_once - 1) / k.at_once) * (stages * k.stage + k.ends) + extra;
            if (cost < best.cost) best = {k.bm, k.slots, s, cost};
        }
    }
    return best;
}
// A backward's two products: dx [M][K] over N, dw [N][K] over M, each by its own plan, or together on one kind of tile where that is cheaper by the same
// model (a launch that keeps all slots busy takes its blocks' time over the slots, and half a block for its end).
// 8192 x 384 -> 1536: 34 us together, 44 one after the other (traced).
struct Pair { Plan x, w; bool together; int bm, slots, sx, sw; };
Pair pair_plan(int M, int N, int K) {
    constexpr int S = 8;
    static const int splits[S] = {1, 2, 3, 4, 6, 8, 12, 16};
    const Forced forced;
    Pair best{plan(M, K, N), plan(N, K, M), false, 0, 0, 1, 1};
    double least = best.x.cost + best.w.cost + 2.5, ex[S], ew[S];
    int px[S], pw[S];                                                     // stages; 0: not allowed
    for (int i = 0; i < S; ++i) {
        px[i] = forced.split(N, splits[i]) ? stages_of(N, splits[i]) : 0;
        pw[i] = forced.split(M, splits[i]) ? stages_of(M, splits[i]) : 0;
        ex[i] = split_cost(M, K, splits[i]);
        ew[i] = split_cost(N, K, splits[i]);
    }
    for (const Kind& k : kinds) {
        const long tx = tiles_of(k, M, K), tw = tiles_of(k, N, K);
        if (!forced.kind(k) || tx + tw > (1L << 21)) continue;
        for (int i = 0; i < S; ++i) {
            if (!px[i]) continue;
            const double cx = px[i] * k.stage + k.ends, nx = (double)tx * splits[i];
            if (cx + ex[i] >= least) continue;
            for (int j = 0; j < S; ++j) {
                if (!pw[j]) continue;
                const double cw = pw[j] * k.stage + k.ends, nw = (double)tw * splits[j], longest = cx > cw ? cx : cw;
                const double cost = (nx + nw <= k.at_once ? longest : (nx * cx + nw * cw) / k.at_once + 0.5 * longest) + ex[i] + ew[j];
                if (cost < least) { least = cost; best.together = true; best.bm = k.bm; best.slots = k.slots; best.sx = splits[i]; best.sw = splits[j]; }
            }
        }
    }
    return best;
}
size_t bwd_ws(const Pair& b, int M, int N, int K) {
    const size_t x = slab_of(M, K, b.x.splits), w = slab_of(N, K, b.w.splits), one = x > w ? x : w;
    const size_t both = b.together ? slab_of(M, K, b.sx) + slab_of(N, K, b.sw) : 0;
    return one > both ? one : both;                                       // (a call may want one product only)
}

// Operands in the form the tile kernel reads: 16-byte pieces, rows of a multiple of 8 values, at most 2^22 from row to row (a lane's offsets inside a
// stage are 32 bits).  Those that are not are copied into `ws` by one launch.
bool as_it_lies(const void* X, long ldx, int cols) { return cols % 8 == 0 && ldx % 8 == 0 && ldx <= 1L << 22 && al16(X); }
struct Operand { const u16** X; long* ldx; long rows; int cols; };
int prepare(std::initializer_list<Operand> ops, char*& ws, hipStream_t st) {
    PadJobs jobs{};
    int n = 0;
    long most = 0;
    for (const Operand& o : ops) {
        if (as_it_lies(*o.X, *o.ldx, o.cols)) continue;
        const long pitch = up8(o.cols), pieces = o.rows * (pitch / 8);
        u16* dst = (u16*)ws;
        ws += up256((size_t)o.rows * pitch * 2);
        jobs.j[n++] = {*o.X, dst, *o.ldx, o.rows, o.cols, (int)pitch};
        *o.X = dst; *o.ldx = pitch;
        if (pieces > most) most = pieces;
    }
    if (!n) return 0;
    const long g = (most + 255) / 256;
    hipLaunchKernelGGL(lin_pad_kernel, dim3((unsigned)(g < 8192 ? g : 8192), n), dim3(256), 0, st, jobs);
    return hipGetLastError() == hipSuccess ? 0 : cdae_fail("lin16: launch failed");
}

// dynamic LDS beyond 64 KB has to be asked for, once a device and kernel (`done`: its devices)
int allow_lds(const void* kernel, int bytes, std::atomic<unsigned long long>& done) {
    if (bytes <= 65536) return 0;
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess) return cdae_fail("lin16: no device");
    const unsigned long long bit = 1ull << (dev & 63);
    if (done.load(std::memory_order_relaxed) & bit) return 0;
    if (hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes) != hipSuccess) return cdae_fail("lin16: hipFuncSetAttribute(max dynamic LDS) failed");
    done.fetch_or(bit, std::memory_order_relaxed);
    return 0;
}
// a product's tiles and splits for tiles of bm; -> blocks, or -1
template <bool AMC, bool BMC>
long lay_out(LinArgs& p, int bm, int splits, char* slab) {
    p.tiles_m = (p.M + bm - 1) / bm; p.tiles_n = (p.N + bm - 1) / bm;
    p.k_per_split = ((p.K + splits - 1) / splits + 63) / 64 * 64;
    p.splits = (p.K + p.k_per_split - 1) / p.k_per_split;
    p.slab = (float*)slab;
    // (16384 x 2048 -> 8192 forward with GELU and its pre-activation kept: 534 us through the caches, 514 with the pre-activation past them, 490 with both)
    p.past = (double)p.M * p.N * 2 > 64e6;
    const long blocks = (long)p.tiles_m * p.tiles_n * p.splits;
    // (a lane's offset inside a stage is 32 bits: 256 rows, or 64 k rows and the columns)
    if (blocks > (1L << 22) || 512 * (AMC ? p.lda / 4 + p.M / 256 : p.lda) >= (1L << 32) || 512 * (BMC ? p.ldb / 4 + p.N / 256 : p.ldb) >= (1L << 32)) {
        cdae_fail("lin16: product too large");
        return -1;
    }
    return blocks;
}
template <class T>
int finish(const LinArgs& p, hipStream_t st) {
    if (p.splits <= 1) return 0;
    const long f = ((long)p.M * ((p.N + 3) / 4) + 255) / 256;
    hipLaunchKernelGGL((lin_finish_kernel<T>), dim3((unsigned)(f < 16384 ? f : 16384)), dim3(256), 0, st, p);
    return hipGetLastError() == hipSuccess ? 0 : cdae_fail("lin16: launch failed");
}
template <class T, bool AMC, bool BMC, int BM, int WM, int WN, int SLOTS>
int launch_tiles(const LinArgs& p, long blocks, hipStream_t st) {
    constexpr int smem = SLOTS * 2 * BM * 128;
    static std::atomic<unsigned long long> done{0};
    auto* kernel = &lin_tile_kernel<T, AMC, BMC, BM, WM, WN, SLOTS>;
    if (allow_lds(reinterpret_cast<const void*>(kernel), smem, done)) return -1;
    hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(64 * WM * WN), smem, st, p);
    return hipGetLastError() == hipSuccess ? 0 : cdae_fail("lin16: launch failed");
}
template <class T, int BM, int WM, int WN, int SLOTS>
int launch_pair(const LinArgs& pw, const LinArgs& px, long blocks_w, long blocks_x, hipStream_t st) {
    constexpr int smem = SLOTS * 2 * BM * 128;
    static std::atomic<unsigned long long> done{0};
    auto* kernel = &lin_pair_kernel<T, BM, WM, WN, SLOTS>;
    if (allow_lds(reinterpret_cast<const void*>(kernel), smem, done)) return -1;
    const long bias_from = (blocks_w + 7) / 8 * 8 + blocks_x;
    hipLaunchKernelGGL(kernel, dim3((unsigned)(bias_from + (pw.db ? (pw.M + 31) / 32 : 0))), dim3(64 * WM * WN), smem, st, pw, px, (int)blocks_w, (int)bias_from);
    return hipGetLastError() == hipSuccess ? 0 : cdae_fail("lin16: launch failed");
}
template <class T, bool AMC, bool BMC>
int product(LinArgs p, const Plan& pl, char* ws, hipStream_t st) {
    const long g = lay_out<AMC, BMC>(p, pl.bm, pl.splits, ws);
    if (g < 0) return -1;
    if (pl.bm == 256 ? launch_tiles<T, AMC, BMC, 256, 2, 4, 2>(p, g, st)
        : pl.bm == 64 ? launch_tiles<T, AMC, BMC, 64, 4, 1, 4>(p, g, st)
        : pl.slots == 4 ? launch_tiles<T, AMC, BMC, 128, 2, 2, 4>(p, g, st)
                        : launch_tiles<T, AMC, BMC, 128, 2, 2, 2>(p, g, st))
        return -1;
    return finish<T>(p, st);
}
// px: dx [M][K] over N;  pw: dw [N][K] over M
template <class T>
int products(LinArgs px, LinArgs pw, const Pair& pl, char* ws, hipStream_t st) {
    if (!pl.together) return product<T, false, true>(px, pl.x, ws, st) || product<T, true, true>(pw, pl.w, ws, st) ? -1 : 0;
    const long gx = lay_out<false, true>(px, pl.bm, pl.sx, ws), gw = lay_out<true, true>(pw, pl.bm, pl.sw, ws + slab_of(px.M, px.N, pl.sx));
    if (gx < 0 || gw < 0) return -1;
    if (pl.bm == 256 ? launch_pair<T, 256, 2, 4, 2>(pw, px, gw, gx, st)
        : pl.bm == 64 ? launch_pair<T, 64, 4, 1, 4>(pw, px, gw, gx, st)
        : pl.slots == 4 ? launch_pair<T, 128, 2, 2, 4>(pw, px, gw, gx, st)
                        : launch_pair<T, 128, 2, 2, 2>(pw, px, gw, gx, st))
        return -1;
    return finish<T>(px, st) || finish<T>(pw, st) ? -1 : 0;
}

int bad_dims(int M, int N, int K, int dt) {
    if (M < 0 || N <= 0 || K <= 0) return cdae_fail("lin16: M >= 0, N >= 1 and K >= 1 required");
    if (M > 1 << 30 || N > 1 << 22 || K > 1 << 22) return cdae_fail("lin16: at most 2^30 rows and 2^22 features");
    if (dt != DT_BF16 && dt != DT_F16) return cdae_fail("lin16: type 0 (bf16) or 1 (fp16)");
    return 0;
}
bool known_act(int a) { return a == L_NONE || a == L_SILU || a == L_RELU || a == L_GELU || a == L_GELU_TANH; }

int slope_rows(int M, int N) {           // rows of a block of the slope pass: about 2048 blocks (eight a CU), 32 rows (four a thread) at least, 512 row blocks at most
    const int ncb = (N + 255) / 256;
    int rb = (2048 + ncb - 1) / ncb;
    if (rb > 512) rb = 512;
    const int rows = (int)(((long)M + rb - 1) / rb);
    return rows < 32 ? 32 : (rows + 7) / 8 * 8;
}
int slope_blocks(int M, int N) { return (M + slope_rows(M, N) - 1) / slope_rows(M, N); }
template <class T>
void slope_launch(const void* dy, long lddy, const void* z, long ldz, u16* dz, float* part, void* dbias, bool fold, int M, int N, int act, hipStream_t st) {
    const int ncb = (N + 255) / 256, rows = slope_rows(M, N), rb = slope_blocks(M, N);
    auto* kernel = N < 8 ? &lin_slope_kernel<T, true> : &lin_slope_kernel<T, false>;
    hipLaunchKernelGGL(kernel, dim3((unsigned)(ncb * rb)), dim3(256), 0, st, (const T*)dy, lddy, (const F16*)z, ldz, (T*)dz, up8(N), part, rb == 1 ? (T*)dbias : nullptr, M, N, rows, ncb, act);
    if (dbias && rb > 1 && fold) hipLaunchKernelGGL((lin_bias_kernel<T>), dim3((N + 31) / 32), dim3(1024), 0, st, part, rb, N, (T*)dbias);
}

// scratch: copies of operands that cannot be read as they lie, partial sums of the splits; backward: dz and the bias gradient's partial sums too
size_t copies_of(int lies, int M, int N, int K) { return lies ? 0 : up256((size_t)M * up8(K) * 2) + up256((size_t)N * up8(K) * 2); }
size_t fwd_bytes(const Plan& pl, int lies, int M, int N, int K) { return copies_of(lies, M, N, K) + slab_of(M, N, pl.splits) + 256; }
size_t bwd_bytes(const Pair& pl, int lies, int M, int N, int K) {
    return up256((size_t)M * up8(N) * 2) + up256(sizeof(float) * (size_t)N * slope_blocks(M, N)) + copies_of(lies, M, N, K) + bwd_ws(pl, M, N, K) + 256;
}

}  // namespace

extern "C" {

size_t cdae_lin16_workspace_bytes(int op, int M, int N, int K) {
    if (M <= 0 || N <= 0 || K <= 0) return 0;
    switch (op & ~CDAE_LIN16_ALIGNED) {
        case CDAE_LIN16_FWD: return fwd_bytes(plan(M, N, K), op & CDAE_LIN16_ALIGNED, M, N, K);
        case CDAE_LIN16_BWD: return bwd_bytes(pair_plan(M, N, K), op & CDAE_LIN16_ALIGNED, M, N, K);
        default: return 0;
    }
}

int cdae_lin16_fwd(const void* x, long ldx, const void* w, long ldw, const void* bias, const void* res, long ldres, void* y, long ldy, void* z, long ldz, int M,
                   int N, int K, int act, int dt, void* ws, size_t ws_bytes, void* stream) {
    if (bad_dims(M, N, K, dt)) return -1;
    if (!known_act(act)) return cdae_fail("lin16_fwd: activation 0 (none), 1 (SiLU), 3 (ReLU), 5 (GELU) or 6 (GELU, tanh form)");
    if (M == 0) return 0;
    if (!x || !w || !y || ldx < K || ldw < K || ldy < N || (res && ldres < N) || (z && ldz < N)) return cdae_fail("lin16_fwd: x, w, y and row pitches of at least a row required");
    const int lies = as_it_lies(x, ldx, K) && as_it_lies(w, ldw, K) ? CDAE_LIN16_ALIGNED : 0;
    const Plan pl = plan(M, N, K);
    if (!ws || !al16(ws) || ws_bytes < fwd_bytes(pl, lies, M, N, K)) return cdae_fail("lin16_fwd: workspace of cdae_lin16_workspace_bytes() required");
    hipStream_t st = (hipStream_t)stream;
    const Timed timed(PROF_IGEMM, 2.0 * M * N * K, 2.0 * ((double)M * K + (double)N * K + (double)M * N * (1 + (res != nullptr) + (z != nullptr))), st);
    LinArgs p{};
    char* at = (char*)ws;
    p.A = (const u16*)x; p.lda = ldx; p.B = (const u16*)w; p.ldb = ldw;
    if (prepare({{&p.A, &p.lda, M, K}, {&p.B, &p.ldb, N, K}}, at, st)) return -1;
    p.M = M; p.N = N; p.K = K;
    p.bias = (const u16*)bias; p.res = (const u16*)res; p.ldres = ldres; p.y = (u16*)y; p.ldy = ldy; p.z = (_Float16*)z; p.ldz = ldz; p.act = act;
    return dt == DT_BF16 ? product<Bf16, false, false>(p, pl, at, st) : product<F16, false, false>(p, pl, at, st);
}

int cdae_lin16_bwd(const void* dy, long lddy, const void* x, long ldx, const void* w, long ldw, const void* z, long ldz, void* dx, long lddx, void* dw, long lddw,
                   void* dbias, int M, int N, int K, int act, int dt, void* ws, size_t ws_bytes, void* stream) {
    if (bad_dims(M, N, K, dt)) return -1;
    if (!known_act(act)) return cdae_fail("lin16_bwd: activation 0 (none), 1 (SiLU), 3 (ReLU), 5 (GELU) or 6 (GELU, tanh form)");
    if (M == 0) return cdae_fail("lin16_bwd: no rows");
    if (!dy || lddy < N || (act != L_NONE && (!z || ldz < N))) return cdae_fail("lin16_bwd: dy, and z with an activation, required");
    if ((dx && (!w || ldw < K || lddx < K)) || (dw && (!x || ldx < K || lddw < K))) return cdae_fail("lin16_bwd: w for dx, x for dw, row pitches of at least a row");
    const int lies = (!dx || as_it_lies(w, ldw, K)) && (!dw || as_it_lies(x, ldx, K)) ? CDAE_LIN16_ALIGNED : 0;
    const Pair pl = pair_plan(M, N, K);
    if (!ws || !al16(ws) || ws_bytes < bwd_bytes(pl, lies, M, N, K)) return cdae_fail("lin16_bwd: workspace of cdae_lin16_workspace_bytes() required");
    hipStream_t st = (hipStream_t)stream;
    const Timed timed(PROF_IGEMM, 2.0 * M * N * K * ((dx != nullptr) + (dw != nullptr)),
                      2.0 * ((double)M * N * (act ? 2 : 1) + (double)M * K * ((dx != nullptr) + (dw != nullptr)) + (double)N * K * ((dx != nullptr) + (dw != nullptr))), st);
    char* at = (char*)ws;
    const bool copy = act != L_NONE || !as_it_lies(dy, lddy, N);
    const bool together = dx && dw && pl.together;
    u16* dz = nullptr;
    float* part = nullptr;
    if (copy && (dx || dw)) { dz = (u16*)at; at += up256((size_t)M * up8(N) * 2); }
    if (dz || dbias) {
        part = dbias ? (float*)at : nullptr;
        if (dbias) at += up256(sizeof(float) * (size_t)N * slope_blocks(M, N));
        if (dt == DT_BF16) slope_launch<Bf16>(dy, lddy, z, ldz, dz, part, dbias, !together, M, N, act, st);
        else slope_launch<F16>(dy, lddy, z, ldz, dz, part, dbias, !together, M, N, act, st);
        if (hipGetLastError() != hipSuccess) return cdae_fail("lin16_bwd: launch failed");
    }
    const u16* d = dz ? dz : (const u16*)dy;
    const long ldd = dz ? up8(N) : lddy;
    LinArgs px{}, pw{};
    if (dbias && together && slope_blocks(M, N) > 1) { pw.sums = part; pw.sum_rows = slope_blocks(M, N); pw.db = dbias; }
    px.A = pw.A = d; px.lda = pw.lda = ldd;
    px.B = (const u16*)w; px.ldb = ldw; pw.B = (const u16*)x; pw.ldb = ldx;
    px.M = M; px.N = K; px.K = N; px.y = (u16*)dx; px.ldy = lddx;
    pw.M = N; pw.N = K; pw.K = M; pw.y = (u16*)dw; pw.ldy = lddw;
    const Operand ow{&px.B, &px.ldb, N, K}, ox{&pw.B, &pw.ldb, M, K};
    if (dx && dw ? prepare({ow, ox}, at, st) : dx ? prepare({ow}, at, st) : dw ? prepare({ox}, at, st) : 0) return -1;
    if (dx && dw) return dt == DT_BF16 ? products<Bf16>(px, pw, pl, at, st) : products<F16>(px, pw, pl, at, st);
    if (dx && (dt == DT_BF16 ? product<Bf16, false, true>(px, pl.x, at, st) : product<F16, false, true>(px, pl.x, at, st))) return -1;
    if (dw && (dt == DT_BF16 ? product<Bf16, true, true>(pw, pl.w, at, st) : product<F16, true, true>(pw, pl.w, at, st))) return -1;
    return 0;
}

}  // extern "C"
