// Element types of the token kernels that take fp32, fp16 or bf16 data (rms_norm.hip, rotary.hip, packed_attn*.hip): arithmetic is
// fp32, values are widened when they are loaded and rounded once (to nearest even) when they are stored.
#pragma once
#include "common.hpp"
#include "../../include/casmtr_hip.h"

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

namespace casmtr {

template <typename T> struct Vec8Of { typedef T type __attribute__((ext_vector_type(8), aligned(sizeof(T)))); };
template <typename T> using vec8_t = typename Vec8Of<T>::type;
// eight consecutive elements at an address aligned to ONE element: global memory takes 16-byte accesses at any alignment on gfx950, so
// rows of odd widths and views that start anywhere need no second path
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&v)[8]) {
    const vec8_t<T> t = *reinterpret_cast<const vec8_t<T>*>(p);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (float)t[i];
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&v)[8]) {
    vec8_t<T> t;
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = (T)v[i];
    *reinterpret_cast<vec8_t<T>*>(p) = t;
}
// the first n (1..8) of them
template <typename T>
__device__ __forceinline__ void load_n(const T* p, float (&v)[8], int n) {
    if (n >= 8) { load8(p, v); return; }
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < n ? (float)p[i] : 0.f;
}
template <typename T>
__device__ __forceinline__ vec8_t<T> load_raw_n(const T* p, int n) {
    if (n >= 8) return *reinterpret_cast<const vec8_t<T>*>(p);
    vec8_t<T> v;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < n ? p[i] : (T)0.f;
    return v;
}
template <typename T>
__device__ __forceinline__ void store_n(T* p, const float (&v)[8], int n) {
    if (n >= 8) { store8(p, v); return; }
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (i < n) p[i] = (T)v[i];
}

// calls f(T{}) for the element type of a CASMTR_F32 / F16 / BF16 code; -> false for any other code
template <typename F>
static inline bool with_type(int dtype, F&& f) {
    if (dtype == CASMTR_F32) f(float{});
    else if (dtype == CASMTR_F16) f(f16_t{});
    else if (dtype == CASMTR_BF16) f(bf16_t{});
    else return false;
    return true;
}
}  // namespace casmtr
