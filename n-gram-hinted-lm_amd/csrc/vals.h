// Element types of the model-side operators (embedded hint rows, the key/value cache, tree attention): loads and stores
// of a few consecutive elements as 32-bit floats, rounded once (half to even) where they are written.
#pragma once
#include "ngram_common.h"

typedef _Float16 f16;
typedef __bf16 b16;

// the element types' numbers in the C ABI
enum { NG_F32 = 0, NG_BF16 = 1, NG_F16 = 2 };
// a cache's codes
enum { KV_INT8 = 0, KV_FP8 = 1, KV_BF16 = 2, KV_F16 = 3 };

template <int BYTES> struct raw_t;
template <> struct raw_t<2> { typedef unsigned short type; };
template <> struct raw_t<4> { typedef u32 type; };
template <> struct raw_t<8> { typedef uint2 type; };
template <> struct raw_t<16> { typedef uint4 type; };

// N consecutive elements of T, moved as one load or store of N * sizeof(T) bytes (p aligned to that)
template <typename T, int N> struct Pack {
    typedef typename raw_t<sizeof(T) * N>::type raw;
    union {
        raw r;
        T v[N];
    };
    __device__ __forceinline__ void load(const T* p) { r = *(const raw*)p; }
    __device__ __forceinline__ void store(T* p) const { *(raw*)p = r; }
};

__device__ __forceinline__ bool finite_f(float x) { return __builtin_fabsf(x) < __builtin_inff(); }  // false for NaN
