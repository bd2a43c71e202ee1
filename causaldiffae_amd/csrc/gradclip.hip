// gradclip.hip — the global norm of many gradients, and clipping by it (gfx950):
//
//     n = |scale| * sqrt(sum over all tensors of g^2),      out = g * scale * min(1, max_norm / (n + 1e-6))
//
// An HBM stream: the norm reads every gradient once, the clipping reads it again and writes it.  Squares are formed and added in fp64: fp32
// squares leave their range at |g| > 1.8e19 and |g| < 1e-23, and 64-bit adds make the order of summation irrelevant at fp32 accuracy; the
// fp64 pipe has room for it (one fma per 2..4 bytes read).  The order is fixed all the same: each block leaves ONE partial sum in a slot of
// its own, every block of the second launch adds the slots in the same order, so the result is the same in every run.
// Tensors come as kernel arguments, so the calls allocate nothing, copy nothing to the device and can be captured; back-to-back tensors (the
// views of a flat buffer) are joined on the host and cost one table entry together.
#include <hip/hip_runtime.h>
#include <algorithm>
#include <math.h>
#include <vector>

#include "cdae.h"
#include "block_common.h"
#include "cdae_internal.h"

namespace {

constexpr int GC_MAX = 128;                 // table entries of one launch: 128 * 29 + 8 bytes of arguments, below the 4 KB a launch may carry
constexpr int GC_CHUNK = 16384;             // values a block takes at a time: 64 or 32 KB in four or eight passes of its threads' 16-byte loads, unrolled
constexpr int GC_BLOCKS = 1024;             // blocks over all launches of a call, about four per CU
constexpr int GC_SLOTS = 8192;              // partial sums the workspace holds: GC_BLOCKS + one more launch's minimum per table

struct GcTab {
    const void* in[GC_MAX];
    void* out[GC_MAX];
    long n[GC_MAX];
    int first[GC_MAX + 1];                  // first chunk of an entry; first[count] = chunks of the table
    unsigned char types[GC_MAX];            // type of in | type of out << 4
    int count;
};
static_assert(sizeof(GcTab) <= 3800, "kernel arguments");

// sum of the squares of one chunk; PAST: read past the caches
template <class T, bool PAST>
__device__ double sq_chunk(const T* __restrict__ p, int n) {
    constexpr int V = 16 / sizeof(T), U = 8;
    double s0 = 0.0, s1 = 0.0;
    auto add = [&](const Pack<T, V>& r) {
#pragma unroll
        for (int e = 0; e < V; e += 2) {
            const double a = ld1(r.v[e]), b = ld1(r.v[e + 1]);
            s0 = fma(a, a, s0); s1 = fma(b, b, s1);
        }
    };
    int i = threadIdx.x * V;
    if (n == GC_CHUNK) {                                                  // a whole chunk: eight loads on their way together
#pragma unroll 1
        for (int k = 0; k < GC_CHUNK / (256 * V * U); ++k) {
            Pack<T, V> r[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const Pack<T, V>* at = reinterpret_cast<const Pack<T, V>*>(p + i + (k * U + u) * 256 * V);
                r[u] = PAST ? load_past(at) : *at;
            }
#pragma unroll
            for (int u = 0; u < U; ++u) add(r[u]);
        }
        return s0 + s1;
    }
    for (; i + V <= n; i += 256 * V) add(*reinterpret_cast<const Pack<T, V>*>(p + i));
    for (int k = i; k < n && k < i + V; ++k) { const double v = ld1(p[k]); s0 = fma(v, v, s0); }
    return s0 + s1;
}

__device__ double block_sum(double s) {
    __shared__ double part[4];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
    __syncthreads();
    s = (part[0] + part[1]) + (part[2] + part[3]);
    __syncthreads();
    return s;
}

// the entry that chunk c of the table belongs to
__device__ __forceinline__ int entry_of(const GcTab& t, int c) {
    int lo = 0, hi = t.count;
    while (hi - lo > 1) { const int mid = (lo + hi) >> 1; if (t.first[mid] <= c) lo = mid; else hi = mid; }
    return lo;
}

// PAST: the gradients are not read again by this call.  93M fp32 values: 61 us (6.1 TB/s) past the caches, 69 through them; before a clipping pass,
// which reads the last of them from the memory-side cache, the other way round (202 and 188 us for both passes).
template <bool PAST>
__global__ __launch_bounds__(256) void gc_norm_kernel(const GcTab t, double* __restrict__ slots) {
    double s = 0.0;
    const int chunks = t.first[t.count];
    for (int c = blockIdx.x; c < chunks; c += gridDim.x) {
        const int e = entry_of(t, c);
        const long at = (long)(c - t.first[e]) * GC_CHUNK;
        const int n = t.n[e] - at < GC_CHUNK ? (int)(t.n[e] - at) : GC_CHUNK;
        const int ty = t.types[e] & 15;
        if (ty == DT_F32) s += sq_chunk<float, PAST>(reinterpret_cast<const float*>(t.in[e]) + at, n);
        else if (ty == DT_BF16) s += sq_chunk<Bf16, PAST>(reinterpret_cast<const Bf16*>(t.in[e]) + at, n);
        else s += sq_chunk<F16, PAST>(reinterpret_cast<const F16*>(t.in[e]) + at, n);
    }
    s = block_sum(s);
    if (threadIdx.x == 0) slots[blockIdx.x] = s;
}

// every block adds all slots in the same order: norm and factor are the same bits everywhere
__device__ double total(const double* __restrict__ slots, int nslots) {
    double s = 0.0;
    for (int i = threadIdx.x; i < nslots; i += 256) s += slots[i];
    return block_sum(s);
}
__device__ __forceinline__ float clip_factor(double sum, double scale, double max_norm, float* norm) {
    const double n = sqrt(sum) * fabs(scale);
    *norm = (float)n;
    const double c = isinf(max_norm) ? 1.0 : max_norm / (n + 1e-6);
    return (float)(scale * (c >= 1.0 ? 1.0 : c));           // (a norm that is not a number stays one in the factor)
}

__global__ __launch_bounds__(256) void gc_finish_kernel(const double* __restrict__ slots, int nslots, double scale, double max_norm, float* __restrict__ norm) {
    const double s = total(slots, nslots);
    if (threadIdx.x == 0) { float n; const float f = clip_factor(s, scale, max_norm, &n); norm[0] = n; norm[1] = f; }
}

// One chunk times the factor.  In place the input and output are the same addresses, read before they are written by the same thread.
template <class T, class O>
__device__ void mul_chunk(const T* p, O* o, int n, float f) {
    constexpr int V = 16 / sizeof(T), U = 4;
    auto put = [&](int at, const Pack<T, V>& r) {
        Pack<O, V> w;
#pragma unroll
        for (int e = 0; e < V; ++e) st1(w.v[e], ld1(r.v[e]) * f);
        store_past(reinterpret_cast<Pack<O, V>*>(o + at), w);             // (through the caches 219 us instead of 188 for 93M fp32 values)
    };
    int i = threadIdx.x * V;
    if (n == GC_CHUNK) {
#pragma unroll 1
        for (int k = 0; k < GC_CHUNK / (256 * V * U); ++k) {
            Pack<T, V> r[U];
#pragma unroll
            for (int u = 0; u < U; ++u) r[u] = *reinterpret_cast<const Pack<T, V>*>(p + i + (k * U + u) * 256 * V);
#pragma unroll
            for (int u = 0; u < U; ++u) put(i + (k * U + u) * 256 * V, r[u]);
        }
        return;
    }
    for (; i + V <= n; i += 256 * V) put(i, *reinterpret_cast<const Pack<T, V>*>(p + i));
    for (int k = i; k < n && k < i + V; ++k) st1(o[k], ld1(p[k]) * f);
}
template <class T>
__device__ void mul_chunk_to(const T* p, void* o, int ty, long at, int n, float f) {
    if (ty == DT_F32) mul_chunk(p + at, reinterpret_cast<float*>(o) + at, n, f);
    else if (ty == DT_BF16) mul_chunk(p + at, reinterpret_cast<Bf16*>(o) + at, n, f);
    else mul_chunk(p + at, reinterpret_cast<F16*>(o) + at, n, f);
}

__global__ __launch_bounds__(256) void gc_scale_kernel(const GcTab t, const double* __restrict__ slots, int nslots, double scale, double max_norm,
                                                       float* __restrict__ norm) {
    float n;
    const float f = clip_factor(total(slots, nslots), scale, max_norm, &n);
    if (blockIdx.x == 0 && threadIdx.x == 0) { norm[0] = n; norm[1] = f; }
    // from the end: what the norm has read last is still in the memory-side cache
    for (int c = t.first[t.count] - 1 - (int)blockIdx.x; c >= 0; c -= gridDim.x) {
        const int e = entry_of(t, c);
        const long at = (long)(c - t.first[e]) * GC_CHUNK;
        const int ti = t.types[e] & 15, to = t.types[e] >> 4;
        if (f == 1.f && t.in[e] == t.out[e] && ti == to) continue;      // in place and nothing to clip: the values stay
        const int left = t.n[e] - at < GC_CHUNK ? (int)(t.n[e] - at) : GC_CHUNK;
        if (ti == DT_F32) mul_chunk_to(reinterpret_cast<const float*>(t.in[e]), t.out[e], to, at, left, f);
        else if (ti == DT_BF16) mul_chunk_to(reinterpret_cast<const Bf16*>(t.in[e]), t.out[e], to, at, left, f);
        else mul_chunk_to(reinterpret_cast<const F16*>(t.in[e]), t.out[e], to, at, left, f);
    }
}

int bytes_of(int ty) { return ty == DT_F32 ? 4 : 2; }

double bytes_in(const long* n, const int* types, int count) {
    double b = 0.0;
    for (int i = 0; i < count; ++i) b += (double)n[i] * bytes_of(types[i]);
    return b;
}

// The next table of a list: joins entries that lie back to back (in and out, same types), skips empty ones.  -> entries used from `at`
int fill(GcTab& t, const void* const* in, const long* n, const int* types, void* const* out, const int* out_types, int count, int at) {
    t.count = 0;
    int i = at;
    for (; i < count; ++i) {
        if (n[i] == 0) continue;
        const unsigned char ty = (unsigned char)(types[i] | (out ? out_types[i] << 4 : 0));
        if (t.count) {
            const int k = t.count - 1;
            if (t.types[k] == ty && (const char*)t.in[k] + t.n[k] * bytes_of(types[i]) == (const char*)in[i] &&
                (!out || (char*)t.out[k] + t.n[k] * bytes_of(out_types[i]) == (char*)out[i])) {
                t.n[k] += n[i];
                continue;
            }
        }
        if (t.count == GC_MAX) break;
        t.in[t.count] = in[i];
        t.out[t.count] = out ? out[i] : nullptr;
        t.n[t.count] = n[i];
        t.types[t.count] = ty;
        ++t.count;
    }
    t.first[0] = 0;
    for (int k = 0; k < t.count; ++k) t.first[k + 1] = t.first[k] + (int)((t.n[k] + GC_CHUNK - 1) / GC_CHUNK);
    return i;
}

int check_list(const char* what, const void* const* in, const long* n, const int* types, int count) {
    if (count < 0 || (count && (!in || !n || !types))) return cdae_fail(what);
    for (int i = 0; i < count; ++i)
        if (n[i] < 0 || (n[i] && !in[i]) || types[i] < 0 || types[i] > 2) return cdae_fail(what);
    double all = 0.0;                                                     // (chunks of a table are counted in 32 bits; the card holds 2^38 bytes)
    for (int i = 0; i < count; ++i) all += (double)n[i];
    if (all > 1e13) return cdae_fail(what);
    return 0;
}

// Every output must be memory of its own, or exactly its input (in place): blocks write while others read, in no order.
struct Span { const char* lo; const char* hi; int id; bool write; };
int check_overlap(const void* const* in, const long* n, const int* types, void* const* out, const int* out_types, int count) {
    try {
        std::vector<Span> v;
        v.reserve(2 * (size_t)count);
        for (int i = 0; i < count; ++i) {
            if (n[i] == 0) continue;
            const char* a = (const char*)in[i];
            const char* b = (const char*)out[i];
            if (!(a == b && bytes_of(types[i]) == bytes_of(out_types[i]))) v.push_back({a, a + n[i] * bytes_of(types[i]), i, false});
            v.push_back({b, b + n[i] * bytes_of(out_types[i]), i, true});
        }
        std::sort(v.begin(), v.end(), [](const Span& p, const Span& q) { return p.lo < q.lo; });
        const char* wrote = nullptr;             // where the spans so far end: those written, those read
        const char* read = nullptr;
        for (const Span& s : v) {
            if (s.lo < wrote || (s.write && s.lo < read)) return 1;
            const char*& end = s.write ? wrote : read;
            if (s.hi > end) end = s.hi;
        }
        return 0;
    } catch (...) {
        return 2;
    }
}

// blocks for `chunks`, at most `most`, such that all but the last take the same number of them
long even(long chunks, long most) {
    const long each = (chunks + most - 1) / most;
    return (chunks + each - 1) / each;
}

// the norm launches: one partial sum a block, blocks shared out by each table's part of the values.  -> number of slots, or -1
int launch_norm(const void* const* in, const long* n, const int* types, int count, bool past, double* slots, hipStream_t st) {
    double all = 0.0;
    for (int i = 0; i < count; ++i) all += (double)n[i];
    int used = 0, at = 0;
    while (at < count) {
        GcTab t;
        at = fill(t, in, n, types, nullptr, nullptr, count, at);
        if (!t.count) break;
        const long chunks = t.first[t.count];
        double mine = 0.0;
        for (int k = 0; k < t.count; ++k) mine += (double)t.n[k];
        long blocks = (long)(GC_BLOCKS * (mine / all)) + 1;
        blocks = even(chunks, blocks);
        if (used + blocks > GC_SLOTS) blocks = GC_SLOTS - used;
        if (blocks < 1) { cdae_fail("grad_norm: too many tensors in one call"); return -1; }
        auto* kernel = past ? &gc_norm_kernel<true> : &gc_norm_kernel<false>;
        hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(256), 0, st, t, slots + used);
        if (hipGetLastError() != hipSuccess) { cdae_fail("grad_norm launch failed"); return -1; }
        used += (int)blocks;
    }
    return used;
}

}  // namespace

extern "C" {

size_t cdae_grad_workspace_bytes(void) { return sizeof(double) * GC_SLOTS; }

int cdae_grad_norm(const void* const* in, const long* n, const int* types, int count, double scale, double max_norm, float* norm, void* ws, size_t ws_bytes,
                   void* stream) {
    if (check_list("grad_norm: a list of device tensors with sizes >= 0 and types 0 (bf16), 1 (fp16), 2 (fp32)", in, n, types, count)) return -1;
    if (!norm || !ws || ((size_t)ws & 15) || ws_bytes < cdae_grad_workspace_bytes()) return cdae_fail("grad_norm: norm[2] and a workspace of cdae_grad_workspace_bytes() required");
    if (!(max_norm >= 0.0)) return cdae_fail("grad_norm: max_norm must be a number >= 0 (infinity: nothing is clipped)");
    hipStream_t st = (hipStream_t)stream;
    const double bytes = bytes_in(n, types, count);
    const Timed timed(PROF_OPT, bytes, bytes, st);
    double* slots = (double*)ws;
    const int used = launch_norm(in, n, types, count, true, slots, st);
    if (used < 0) return -1;
    hipLaunchKernelGGL(gc_finish_kernel, dim3(1), dim3(256), 0, st, slots, used, scale, max_norm, norm);
    return hipGetLastError() == hipSuccess ? 0 : cdae_fail("grad_norm finish launch failed");
}

int cdae_grad_clip(const void* const* in, const long* n, const int* types, void* const* out, const int* out_types, int count, double scale, double max_norm,
                   float* norm, void* ws, size_t ws_bytes, void* stream) {
    if (check_list("grad_clip: a list of device tensors with sizes >= 0 and types 0 (bf16), 1 (fp16), 2 (fp32)", in, n, types, count)) return -1;
    if (check_list("grad_clip: outputs beside every input, types 0 (bf16), 1 (fp16), 2 (fp32)", (const void* const*)out, n, out_types, count)) return -1;
    if (!norm || !ws || ((size_t)ws & 15) || ws_bytes < cdae_grad_workspace_bytes()) return cdae_fail("grad_clip: norm[2] and a workspace of cdae_grad_workspace_bytes() required");
    if (!(max_norm >= 0.0)) return cdae_fail("grad_clip: max_norm must be a number >= 0 (infinity: nothing is clipped)");
    if (const int rc = check_overlap(in, n, types, out, out_types, count))
        return cdae_fail(rc == 1 ? "grad_clip: two outputs share memory, or an output shares memory with a gradient other than its own" : "grad_clip: out of host memory");
    hipStream_t st = (hipStream_t)stream;
    const double bytes = bytes_in(n, types, count) + bytes_in(n, out_types, count);
    const Timed timed(PROF_OPT, bytes, bytes, st);
    double* slots = (double*)ws;
    const int used = launch_norm(in, n, types, count, false, slots, st);
    if (used < 0) return -1;
    if (!used) {
        hipLaunchKernelGGL(gc_finish_kernel, dim3(1), dim3(256), 0, st, slots, 0, scale, max_norm, norm);
        return hipGetLastError() == hipSuccess ? 0 : cdae_fail("grad_clip finish launch failed");
    }
    int at = 0;
    while (at < count) {
        GcTab t;
        at = fill(t, in, n, types, out, out_types, count, at);
        if (!t.count) break;
        hipLaunchKernelGGL(gc_scale_kernel, dim3((unsigned)even(t.first[t.count], 2 * GC_BLOCKS)), dim3(256), 0, st, t, slots, used, scale, max_norm, norm);
        if (hipGetLastError() != hipSuccess) return cdae_fail("grad_clip launch failed");
    }
    return 0;
}

}  // extern "C"
