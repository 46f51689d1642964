// Element types of the elementwise and 8-bit kernels: fp16, bf16 and fp32 rows read and written in
// groups of eight, computed in fp32. The group types are aligned like one element: rows may start
// anywhere (odd widths, views), and gfx950 takes such 16-byte accesses as one instruction.
#pragma once

#include "dk_internal.h"

namespace dk {

typedef float float8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));

template <int DT>
struct Elem;
template <>
struct Elem<DK_FP16> {
    typedef _Float16 type;
    typedef half8_t vec;
    typedef half8_t loose __attribute__((aligned(2)));
};
template <>
struct Elem<DK_BF16> {
    typedef __bf16 type;
    typedef bf16x8_t vec;
    typedef bf16x8_t loose __attribute__((aligned(2)));
};
template <>
struct Elem<DK_FP32> {
    typedef float type;
    typedef float8_t vec;
    typedef float8_t loose __attribute__((aligned(4)));
};

constexpr int elem_bytes(int dt) { return dt == DK_FP32 ? 4 : 2; }

template <int DT>
__device__ __forceinline__ float8_t widen8(typename Elem<DT>::vec v) {
    return __builtin_convertvector(v, float8_t);
}

template <int DT>
__device__ __forceinline__ typename Elem<DT>::vec load8_raw(const void* p) {
    return *(const typename Elem<DT>::loose*)p;
}

template <int DT>
__device__ __forceinline__ float8_t load8(const void* p) {
    return widen8<DT>(load8_raw<DT>(p));
}

// One rounding (to nearest even). The empty asm keeps a product that feeds it out of the
// mixed-precision multiply-adds, which would round fp16(x * y) once from the exact product.
template <int DT>
__device__ __forceinline__ void store8(void* p, float8_t v) {
    if constexpr (DT == DK_FP16) {
        float a = v[0], b = v[1], c = v[2], d = v[3], e = v[4], f = v[5], g = v[6], h = v[7];
        asm("" : "+v"(a), "+v"(b), "+v"(c), "+v"(d), "+v"(e), "+v"(f), "+v"(g), "+v"(h));
        v = float8_t{a, b, c, d, e, f, g, h};
    }
    *(typename Elem<DT>::loose*)p = __builtin_convertvector(v, typename Elem<DT>::vec);
}

template <int DT>
__device__ __forceinline__ void store1(void* p, float v) {
    asm("" : "+v"(v));
    *(typename Elem<DT>::type*)p = (typename Elem<DT>::type)v;
}

// Element i of an array whose type is known at run time.
__device__ __forceinline__ float load_any(const void* p, int dtype, int64_t i) {
    if (dtype == DK_FP32) return ((const float*)p)[i];
    if (dtype == DK_BF16) return (float)((const __bf16*)p)[i];
    return (float)((const _Float16*)p)[i];
}

}  // namespace dk
