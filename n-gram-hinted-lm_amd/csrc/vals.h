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

// N consecutive elements of T, moved as one load or store of N * sizeof(T) bytes, wherever p points (global memory takes
// any alignment; rows whose length is odd run at the wide loads' rate but for the lines that two of them share)
template <int BYTES> struct raw_t { typedef u32 type __attribute__((ext_vector_type(BYTES / 4), aligned(2))); };
template <> struct raw_t<2> { typedef unsigned short type; };
template <> struct raw_t<4> { typedef u32 type __attribute__((aligned(2))); };

template <typename T, int N> struct Pack {
    T v[N];
    typedef typename raw_t<sizeof(T) * N>::type raw;
    __device__ __forceinline__ void load(const T* p) {
        const raw r = *(const raw*)p;
        __builtin_memcpy(v, &r, sizeof(raw));
    }
    __device__ __forceinline__ void store(T* p) const {
        raw r;
        __builtin_memcpy(&r, v, sizeof(raw));
        *(raw*)p = r;
    }
};

__device__ __forceinline__ bool finite_f(float x) { return __builtin_fabsf(x) < __builtin_inff(); }  // false for NaN
