// Element types of the operators that also take 16-bit tensors: widening loads and rounding stores.
// The vector accesses are declared with the alignment of ONE element: gfx950 loads and stores 16
// bytes at any element boundary, so odd row strides and offsets take the same path.
#pragma once

#include "alsmi_common.h"

namespace alsmi {

// The type an element is worked on in.
template <typename T>
struct Elem {
    typedef float wide;
};
template <>
struct Elem<double> {
    typedef double wide;
};

// N consecutive elements from p, widened; those at or behind `valid` are zero and not read.  STREAM: past
// the caches (data that is larger than they are anyway).
template <typename T, int N, bool STREAM = false>
__device__ __forceinline__ void load_n(typename Elem<T>::wide (&v)[N], const T *__restrict__ p,
                                       int64_t valid) {
    typedef typename Elem<T>::wide W;
    typedef T vec_t __attribute__((ext_vector_type(N), aligned(sizeof(T))));
    if (valid >= N) {
        vec_t x;
        if constexpr (STREAM) x = __builtin_nontemporal_load(reinterpret_cast<const vec_t *>(p));
        else x = *reinterpret_cast<const vec_t *>(p);
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = (W)x[i];
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = i < valid ? (W)p[i] : (W)0;
    }
}
template <typename T>
__device__ __forceinline__ void load8(typename Elem<T>::wide (&v)[8], const T *__restrict__ p,
                                      int64_t valid) {
    load_n<T, 8>(v, p, valid);
}

// The first `valid` of N elements to p, rounded to nearest.
template <typename T, int N, bool STREAM = false>
__device__ __forceinline__ void store_n(T *__restrict__ p, const typename Elem<T>::wide (&v)[N],
                                        int64_t valid) {
    typedef T vec_t __attribute__((ext_vector_type(N), aligned(sizeof(T))));
    if (valid >= N) {
        vec_t x;
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = (T)v[i];
        if constexpr (STREAM) __builtin_nontemporal_store(x, reinterpret_cast<vec_t *>(p));
        else *reinterpret_cast<vec_t *>(p) = x;
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (i < valid) p[i] = (T)v[i];
    }
}
template <typename T>
__device__ __forceinline__ void store8(T *__restrict__ p, const typename Elem<T>::wide (&v)[8],
                                       int64_t valid) {
    store_n<T, 8>(p, v, valid);
}

}  // namespace alsmi
