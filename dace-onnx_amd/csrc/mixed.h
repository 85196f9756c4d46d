// Arrays of float32, float16 or bfloat16 whose values are read as float32 and rounded when they are stored.
#pragma once

#include "common.h"

#include <type_traits>

namespace mi355x {

typedef _Float16 f16;
typedef __bf16 bf16;

// E values of T as they lie in memory, at any address of T: the memory unit takes 16-byte accesses at any boundary.
template <class T, int E>
struct Values {
    typedef T vec __attribute__((ext_vector_type(E)));
    typedef vec unaligned __attribute__((aligned(sizeof(T))));
};
template <class T>
struct Values<T, 1> {
    typedef T vec;
    typedef T unaligned;
};

// v[e] = p[e] for e < n, 0 for the others
template <class T, int E>
__device__ __forceinline__ void load_values(float (&v)[E], const T* p, int64_t n) {
    if (n >= E) {
        const typename Values<T, E>::vec x = *reinterpret_cast<const typename Values<T, E>::unaligned*>(p);
#pragma unroll
        for (int e = 0; e < E; ++e) {
            if constexpr (E == 1) v[e] = (float)x;
            else v[e] = (float)x[e];
        }
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = e < n ? (float)p[e] : 0.0f;
    }
}

// p[e] = v[e] for e < n, each rounded once, to the nearest (ties to even)
template <class T, int E, class V>
__device__ __forceinline__ void store_values(T* p, const V (&v)[E], int64_t n) {
    if (n >= E) {
        typename Values<T, E>::vec x;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            if constexpr (E == 1) x = (T)v[e];
            else x[e] = (T)v[e];
        }
        *reinterpret_cast<typename Values<T, E>::unaligned*>(p) = x;
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (e < n) p[e] = (T)v[e];
    }
}

// f(a value of the type that `type`, an element type of the interface, names); false if it is none of these
template <class F>
static bool with_type(int type, F&& f) {
    if (type == MI355X_TYPE_FLOAT) f(float{});
    else if (type == MI355X_TYPE_FLOAT16) f(f16{});
    else if (type == MI355X_TYPE_BFLOAT16) f(bf16{});
    else return false;
    return true;
}
static inline bool is_mixed_type(int type) { return type == MI355X_TYPE_FLOAT || type == MI355X_TYPE_FLOAT16 || type == MI355X_TYPE_BFLOAT16; }

template <int N>
using Int = std::integral_constant<int, N>;

}  // namespace mi355x
