// Element access shared by the transformer-block kernels (lin16.hip, resnorm.hip, gradclip.hip): bf16 / f16 / fp32 values as fp32 in registers.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "cdae_internal.h"

enum { DT_BF16 = 0, DT_F16 = 1, DT_F32 = 2 };

struct Bf16 { unsigned short u; };
struct F16 { _Float16 h; };

__device__ __forceinline__ float ld1(Bf16 v) { return __builtin_bit_cast(float, (unsigned)v.u << 16); }
__device__ __forceinline__ float ld1(F16 v) { return (float)v.h; }
__device__ __forceinline__ float ld1(float v) { return v; }
__device__ __forceinline__ void st1(Bf16& d, float v) { d.u = __builtin_bit_cast(unsigned short, (__bf16)v); }       // round to nearest even
__device__ __forceinline__ void st1(F16& d, float v) { d.h = (_Float16)v; }
__device__ __forceinline__ void st1(float& d, float v) { d = v; }

// V consecutive values at ANY element alignment: the vector type carries the element's alignment, so rows of an odd length are read with the
// same wide instructions as aligned ones
template <class T, int V>
struct __attribute__((packed, aligned(sizeof(T)))) Pack { T v[V]; };

template <class T, int V>
__device__ __forceinline__ void ldv(const T* __restrict__ p, float (&o)[V]) {
    const Pack<T, V> t = *reinterpret_cast<const Pack<T, V>*>(p);
#pragma unroll
    for (int i = 0; i < V; ++i) o[i] = ld1(t.v[i]);
}
template <class T, int V>
__device__ __forceinline__ void stv(T* __restrict__ p, const float (&o)[V]) {
    Pack<T, V> t;
#pragma unroll
    for (int i = 0; i < V; ++i) st1(t.v[i], o[i]);
    *reinterpret_cast<Pack<T, V>*>(p) = t;
}
// Past the caches: data that is not read again soon.  (4-byte pieces of unaligned vectors: the instructions stay 16 bytes wide)
typedef unsigned u32x4_any __attribute__((ext_vector_type(4), aligned(2)));
typedef unsigned u32x2_any __attribute__((ext_vector_type(2), aligned(2)));
template <class P>
__device__ __forceinline__ P load_past(const P* p) {
    static_assert(sizeof(P) == 16, "one 16-byte piece");
    return __builtin_bit_cast(P, __builtin_nontemporal_load(reinterpret_cast<const u32x4_any*>(p)));
}
template <class P>
__device__ __forceinline__ void store_past(P* p, const P& v) {
    static_assert(sizeof(P) == 8 || sizeof(P) % 16 == 0, "whole pieces");
    if constexpr (sizeof(P) == 8) __builtin_nontemporal_store(__builtin_bit_cast(u32x2_any, v), reinterpret_cast<u32x2_any*>(p));
    else {
        struct Pieces { u32x4_any q[sizeof(P) / 16]; };
        const Pieces w = __builtin_bit_cast(Pieces, v);
#pragma unroll
        for (int i = 0; i < (int)(sizeof(P) / 16); ++i) __builtin_nontemporal_store(w.q[i], reinterpret_cast<u32x4_any*>(p) + i);
    }
}
// the same with only the first n (0..V) values present; the others read as zero and are not written
template <class T, int V>
__device__ __forceinline__ void ldv_n(const T* __restrict__ p, int n, float (&o)[V]) {
    if (n >= V) { ldv<T, V>(p, o); return; }
#pragma unroll
    for (int i = 0; i < V; ++i) o[i] = i < n ? ld1(p[i]) : 0.f;
}
template <class T, int V>
__device__ __forceinline__ void stv_n(T* __restrict__ p, int n, const float (&o)[V]) {
    if (n >= V) { stv<T, V>(p, o); return; }
#pragma unroll
    for (int i = 0; i < V; ++i) if (i < n) st1(p[i], o[i]);
}
// a value of a vector kept either in the rows' type T or in fp32 (a uniform choice)
template <class T>
__device__ __forceinline__ void st2(void* p, long off, int is32, float v) {
    if (is32) reinterpret_cast<float*>(p)[off] = v;
    else st1(reinterpret_cast<T*>(p)[off], v);
}

// a call's launches in the opt-in profiler (their family, flops or bytes of work, bytes that have to move)
struct Timed {
    const int family; const hipStream_t st;
    Timed(int family_, double work, double bytes, hipStream_t st_) : family(family_), st(st_) { cdae_prof_begin(family, work, st); cdae_prof_note(family, bytes); }
    ~Timed() { cdae_prof_end(family, st); }
};
