// Choosing the largest of many keys in a block without sorting them: a threshold found by halving, then few keys compared
// with each other.
#pragma once
#include "ngram_common.h"

// Numbers as keys that order as they do (0 and -0 alike); 0 is the key of nothing.
__device__ __forceinline__ u32 key_of(float x) {  // NaN and -inf: nothing
    const u32 u = __float_as_uint(x + 0.f);
    return x > -__builtin_inff() ? (u >> 31 ? ~u : u | 0x80000000u) : 0u;
}
__device__ __forceinline__ float of_key(u32 k) { return __uint_as_float(k >> 31 ? k & 0x7FFFFFFFu : ~k); }
__device__ __forceinline__ u64 key_of(double x) {  // NaN and -inf: nothing
    const u64 u = (u64)__double_as_longlong(x + 0.);
    return x > -__builtin_inf() ? (u >> 63 ? ~u : u | 1ull << 63) : 0ull;
}

// How many of a block's threads' flags are set, over NW waves: one barrier a call (two sets of counts, used in turn).
template <int NW> struct Count {
    int (*at)[NW];
    int turn;
    __device__ __forceinline__ Count(int (*lds)[NW]) : at(lds), turn(0) {}
    __device__ __forceinline__ int sum(int wave_count) {
        if constexpr (NW == 1) return wave_count;
        if (lane_id() == 0) at[turn][threadIdx.x >> 6] = wave_count;
        lds_barrier();
        int n = 0;
#pragma unroll
        for (int w = 0; w < NW; ++w) n += at[turn][w];
        turn ^= 1;
        return __builtin_amdgcn_readfirstlane(n);
    }
    // the keys >= t among E of each thread
    template <int E, typename K> __device__ __forceinline__ int at_least(const K (&k)[E], K t) {
        int n = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) n += __popcll(__ballot(k[e] >= t));
        return sum(n);
    }
    // A threshold t with n(t) = the keys >= t in want .. most; where equal keys leave none, the largest t with n(t) >= want.
    // lo: n(lo) >= want is known (n: it); hi: no key is larger. Each step halves what is between.
    template <int E, typename K> __device__ __forceinline__ K threshold(const K (&k)[E], K lo, K hi, int want, int most, int& n) {
        while (n > most && lo < hi) {
            const K mid = lo + (hi - lo) / 2 + 1;
            const int c = at_least(k, mid);
            if (c >= want) lo = mid, n = c;
            else hi = mid - 1;
        }
        return lo;
    }
};

template <typename K> __device__ __forceinline__ K shfl_key(K x, int o) {
    if constexpr (sizeof(K) == 4) return (K)__shfl_xor((int)x, o, WAVE);
    else return (K)(u32)__shfl_xor((int)(u32)x, o, WAVE) | (K)(u32)__shfl_xor((int)(u32)(x >> 32), o, WAVE) << 32;
}
template <typename K> __device__ __forceinline__ K max_wave(K x) {
#pragma unroll
    for (int o = 32; o; o >>= 1) {
        const K y = shfl_key(x, o);
        x = y > x ? y : x;
    }
    return x;
}
template <typename K> __device__ __forceinline__ K min_wave(K x) { return ~max_wave((K)~x); }
