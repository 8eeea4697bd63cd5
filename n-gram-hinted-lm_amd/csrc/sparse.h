// Attention over chosen pages (sparse.hip has the mathematics and the host's side; a file per cache type instantiates it).
#pragma once
#include "tree.h"

struct SparseArgs {
    TreeArgs a;  // q, the cache, out, lse; a.table: the chosen pages [rows, keep], a.width: keep
    const int2* rows;  // [rows]: a row's keys over its chosen pages (0: none), and whether it is in use
    int T, splits;     // the tokens of a sequence; the blocks a unit
    int b0, t0, nt;    // this pass: tokens t0 .. t0 + nt - 1 of sequences b0 on
    i64 units;         // rows x groups of 16 query heads
};

template <int CODES> int sparse_codes(const SparseArgs& s, int dp, hipStream_t st);
template <int CODES> int bounds_codes(const void* k, const float* ks, i64 pages, int shift, int H, int dim, const int* table,
                                      i64 stride, int width, const int* start, int B, int count, b16* bounds, hipStream_t st);

// A row's sequence, token and head.
struct At {
    i64 b;
    int t, head;
};
__device__ __forceinline__ At at_of(const SparseArgs& s, i64 row) {
    const i64 token = row / s.a.H, b = token / s.nt;
    At p;
    p.b = s.b0 + b, p.t = s.t0 + (int)(token - b * s.nt), p.head = (int)(row - token * s.a.H);
    return p;
}

// The tiles of a unit that its block `split` takes: [t0, t1), and how many of its blocks have any.
struct Share {
    int t0, t1, blocks;
};
__device__ __forceinline__ Share share_of(int keys, int splits, int split) {
    const int tiles = (keys + TILE - 1) / TILE, per = (tiles + splits - 1) / splits;
    Share s;
    s.t0 = split * per, s.t1 = s.t0 + per < tiles ? s.t0 + per : tiles;
    s.blocks = per ? (tiles + per - 1) / per : 0;
    return s;
}

// A block per (row, group of up to 16 query heads, part of its chosen pages): tree attention of one token whose page table is
// the chosen pages'.
template <int CODES, int DP> __global__ __launch_bounds__(256, DP <= 128 ? 2 : 1) void sparse_k(const SparseArgs s) {
    typedef Tree<CODES, DP, 1> W;
    typedef typename W::Lo Lo;
    __shared__ __align__(16) char lds[sizeof(Lo) * 4 > 16 * W::QLD * 2 ? sizeof(Lo) * 4 : 16 * W::QLD * 2];
    Lo* lo = (Lo*)lds;  // the waves' sums at the end; before that the queries
    __shared__ float lm[4][16], ll[4][16];
    __shared__ typename W::Sizes size;
    __shared__ u64 bits[16];
    __shared__ __align__(16) float fac[4][4][32];
    // neighbouring blocks on one XCD (blocks go round the 8 XCDs): rows that share keys meet in its L2
    const i64 blocks = s.units * s.splits, a8 = (blocks + 7) / 8, me = (i64)(blockIdx.x % 8) * a8 + blockIdx.x / 8;
    if ((i64)blockIdx.x / 8 >= a8 || me >= blocks) return;
    const i64 unit = me / s.splits;
    const int split = (int)(me - unit * s.splits), groups = s.a.groups, G = s.a.G;
    const i64 row = unit / groups;
    const int group = (int)(unit - row * groups);
    const At p = at_of(s, row);
    const int2 r = s.rows[row];
    const int n = __builtin_amdgcn_readfirstlane(r.x);
    const Share mine = share_of(n, s.splits, split);
    if (split && mine.t1 <= mine.t0) return;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if constexpr (W::Q8) {
        if (threadIdx.x < 16) size.top[threadIdx.x] = 0;
        lds_barrier();
    }
    TreeArgs a = s.a;
    a.q = (const u16*)a.q + p.b * a.qb + p.t * a.qt, a.T = 1, a.mask = nullptr;
    Seq q;
    q.w = __builtin_amdgcn_readfirstlane(r.y), q.len = n > 0 ? n - 1 : 0, q.n = n, q.tiles = 0, q.span = 0;
    const int base = mine.t0 * TILE + wave * 32, stop = mine.t1 * TILE < n ? mine.t1 * TILE : n;
    typename W::State st;
    typename W::Run run;
    const int* tab = a.table + row * a.width;
    W::begin(a, tab, p.head, base, stop, run);
    const bool own = W::load_q(a, 0, p.head, q, group * 16, (typename W::T*)lds, size, bits, st);
    st.m[0] = -__builtin_inff(), st.l[0] = 0.f;
#pragma unroll
    for (int j = 0; j < W::NJ; ++j) st.o[0][j] = f4{0.f, 0.f, 0.f, 0.f};
    W::keys(a, tab, p.head, q, base, stop, bits, size, own, run, st, fac[wave]);
    float m, sum, o[W::NJ];
    W::join_waves(st, 0, lo, lm, ll, m, sum, o);
    const int at = threadIdx.x >> 4, d0 = (threadIdx.x & 15) * W::NJ, h = group * 16 + at;
    if (h >= G) return;
    if (mine.blocks <= 1) {
        const i64 i = (p.b * s.T + p.t) * a.H * G + p.head * G + h;
        const bool none = sum == 0.f;
        const float inv = none ? 0.f : 1.f / sum;
#pragma unroll
        for (int j = 0; j < W::NJ; ++j) o[j] = none ? 0.f : o[j] * inv;
        put<W::NJ>(a, i * a.dim + d0, a.dim - d0, o);
        if (a.lse && (threadIdx.x & 15) == 0)
            a.lse[i] = none ? -__builtin_inff() : LN2 * (m - W::BIAS + __builtin_amdgcn_logf(sum));
    } else {
        const i64 prow = me * 16 + at;
#pragma unroll
        for (int j = 0; j < W::NJ; ++j) a.po[prow * DP + d0 + j] = o[j];
        if ((threadIdx.x & 15) == 0) a.pm[prow] = m, a.pl[prow] = sum;
    }
}

// A block a unit: its blocks' sums joined.
template <int DP> __global__ __launch_bounds__(256) void sparse_join_k(const SparseArgs s, float bias) {
    constexpr int NJ = DP / 16;
    const TreeArgs& a = s.a;
    const i64 unit = blockIdx.x, row = unit / a.groups;
    const int h = (int)(unit - row * a.groups) * 16 + (threadIdx.x >> 4);
    const At p = at_of(s, row);
    const int parts = share_of(s.rows[row].x, s.splits, 0).blocks;
    if (parts <= 1 || h >= a.G) return;
    const int d0 = (threadIdx.x & 15) * NJ;
    float m = -__builtin_inff(), sum = 0.f, o[NJ];
#pragma unroll
    for (int j = 0; j < NJ; ++j) o[j] = 0.f;
    for (int i = 0; i < parts; ++i) {
        const i64 prow = (unit * s.splits + i) * 16 + (threadIdx.x >> 4);
        const float pm = a.pm[prow], pl = a.pl[prow];
        const float n = fmaxf(m, pm);
        const float ko = m == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(m - n);
        const float kp = pm == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(pm - n);
        sum = (sum == 0.f ? 0.f : sum * ko) + (pl == 0.f ? 0.f : pl * kp);
#pragma unroll
        for (int j = 0; j < NJ; ++j) o[j] = o[j] * ko + a.po[prow * DP + d0 + j] * kp;
        m = n;
    }
    const i64 i = (p.b * s.T + p.t) * a.H * a.G + p.head * a.G + h;
    const bool none = sum == 0.f;
    const float inv = none ? 0.f : 1.f / sum;
#pragma unroll
    for (int j = 0; j < NJ; ++j) o[j] = none ? 0.f : o[j] * inv;
    put<NJ>(a, i * a.dim + d0, a.dim - d0, o);
    if (a.lse && (threadIdx.x & 15) == 0) a.lse[i] = none ? -__builtin_inff() : LN2 * (m - bias + __builtin_amdgcn_logf(sum));
}

template <int CODES, int DP> static int sparse_run(const SparseArgs& s, hipStream_t st) {
    const i64 blocks = (s.units * s.splits + 7) / 8 * 8;
    sparse_k<CODES, DP><<<(unsigned)blocks, 256, 0, st>>>(s);
    const int rc = (int)hipGetLastError();
    if (rc || s.splits == 1) return rc;
    sparse_join_k<DP><<<(unsigned)s.units, 256, 0, st>>>(s, Tree<CODES, DP, 1>::BIAS);
    return (int)hipGetLastError();
}

template <int CODES> int sparse_codes(const SparseArgs& s, int dp, hipStream_t st) {
    switch (dp) {
        case 64: return sparse_run<CODES, 64>(s, st);
        case 128: return sparse_run<CODES, 128>(s, st);
        case 192: return sparse_run<CODES, 192>(s, st);
        default: return sparse_run<CODES, 256>(s, st);
    }
}

// ------------------------------------------------------------------------------------------------------- the bounds

__device__ __forceinline__ b16 outward(float x, bool up) {  // to the next bfloat16 above (or below) where x is none
    const u32 u = __float_as_uint(x), near = u & 0xFFFF0000u;
    if (x != x) return __builtin_bit_cast(b16, (u16)0x7FC0);
    const bool away = up == !(u >> 31);  // its size grows that way
    return __builtin_bit_cast(b16, (u16)((away && u != near ? near + 0x10000u : near) >> 16));
}

// A block per (sequence, page that its tokens touch, head): the elements' smallest and largest over the page's rows, where the
// tokens complete it.
template <int CODES, int DP>
__global__ __launch_bounds__(256) void bounds_k(const void* __restrict__ k, const float* __restrict__ ks, i64 pages, int shift,
                                                int H, int dim, const int* __restrict__ table, i64 stride, int width,
                                                const int* __restrict__ start, int count, int per, b16* __restrict__ bounds) {
    constexpr int L = DP / 8, R = 256 / L;  // lanes a row, rows at a time
    __shared__ float lows[R][DP], highs[R][DP];
    const int h = blockIdx.x % H, at = blockIdx.x / H, b = at / per;
    const i64 from = start[b], column = (from >> shift) + (at - b * per);
    if (column < 0 || (column + 1) << shift > from + count || column >= width) return;
    const int e = table[b * stride + column];
    if ((u32)e >= (u64)pages) return;
    const int r0 = threadIdx.x / L, d0 = threadIdx.x % L * 8;
    const i64 first = ((i64)e * H + h) << shift;
    float lo[8], hi[8];
    u32 bad = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) lo[j] = __builtin_inff(), hi[j] = -__builtin_inff();
    if (r0 < R)
        for (int r = r0; r < 1 << shift; r += R) {
            float x[8];
            if constexpr (CODES == KV_INT8 || CODES == KV_FP8) {
                const float s = ks[first + r];
                const uint2 w = *(const uint2*)((const char*)k + (first + r) * DP + d0);
                if constexpr (CODES == KV_INT8) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) x[j] = (float)(signed char)((j < 4 ? w.x : w.y) >> (8 * (j & 3))) * s;
                } else {
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const auto a = __builtin_amdgcn_cvt_pk_f32_fp8((int)(i ? w.y : w.x), false);
                        const auto c = __builtin_amdgcn_cvt_pk_f32_fp8((int)(i ? w.y : w.x), true);
                        x[4 * i] = a[0] * s, x[4 * i + 1] = a[1] * s, x[4 * i + 2] = c[0] * s, x[4 * i + 3] = c[1] * s;
                    }
                }
            } else {
                typedef typename op_t<CODES>::type T;
                Pack<T, 8> p;
                p.load((const T*)k + (first + r) * DP + d0);
#pragma unroll
                for (int j = 0; j < 8; ++j) x[j] = (float)p.v[j];
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                lo[j] = fminf(lo[j], x[j]), hi[j] = fmaxf(hi[j], x[j]);
                bad |= (x[j] != x[j] ? 1u : 0u) << j;
            }
        }
    if (r0 < R)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            lows[r0][d0 + j] = bad >> j & 1 ? __builtin_nanf("") : lo[j];
            highs[r0][d0 + j] = hi[j];
        }
    __syncthreads();
    const int d = threadIdx.x;
    if (d >= DP) return;
    float l = lows[0][d], g = highs[0][d];
    bool nan = l != l;
#pragma unroll
    for (int r = 1; r < R; ++r) {
        const float x = lows[r][d];
        nan |= x != x;
        l = fminf(l, x), g = fmaxf(g, highs[r][d]);
    }
    if (nan) l = g = __builtin_nanf("");
    if (d >= dim) l = g = 0.f;
    b16* o = bounds + (((i64)e * H + h) * 2) * DP + d;
    o[0] = outward(l, false), o[DP] = outward(g, true);
}

template <int CODES> int bounds_codes(const void* k, const float* ks, i64 pages, int shift, int H, int dim, const int* table,
                                      i64 stride, int width, const int* start, int B, int count, b16* bounds,
                                      hipStream_t st) {
    const int per = ((count - 1) >> shift) + 2;
    const i64 n = (i64)B * per * H;
    if (n >= (i64)1 << 31) return -1;
#define DP_CASE(DP)                                                                                                      \
    bounds_k<CODES, DP><<<(unsigned)n, 256, 0, st>>>(k, ks, pages, shift, H, dim, table, stride, width, start, count, per, bounds)
    switch ((dim + 63) / 64) {
        case 1: DP_CASE(64); break;
        case 2: DP_CASE(128); break;
        case 3: DP_CASE(192); break;
        default: DP_CASE(256);
    }
#undef DP_CASE
    return (int)hipGetLastError();
}
