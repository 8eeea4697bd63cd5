// Attention over chosen pages (sparse.hip has the mathematics and the host's side; a file per cache type instantiates it).
#pragma once
#include "tree.h"
#include <type_traits>

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

// A unit's sequence, token, head and group of 16 query heads. The tokens of a head come one after the other (rows lie by
// sequence, token and head): their pages are the same head's, which an XCD's L2 then holds.
struct At {
    i64 b, row;
    int t, head, group;
};
__device__ __forceinline__ At at_of(const SparseArgs& s, u32 unit) {
    const u32 x = unit / (u32)s.a.groups, bh = x / (u32)s.nt, b = bh / (u32)s.a.H;
    const int t = (int)(x - bh * s.nt);
    At p;
    p.group = (int)(unit - x * s.a.groups), p.head = (int)(bh - b * s.a.H), p.b = s.b0 + (i64)b, p.t = s.t0 + t;
    p.row = ((i64)b * s.nt + t) * s.a.H + p.head;
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
template <int CODES, int DP> __global__ __launch_bounds__(256, DP <= 64 ? 4 : DP <= 128 ? 3 : 1) void sparse_k(const SparseArgs s) {
    typedef Tree<CODES, DP, 1, true> W;
    typedef typename W::Lo Lo;
    // the queries, then the waves' keys, at the end their sums
    __shared__ __align__(16) char lds[sizeof(Lo) > W::STAGE ? sizeof(Lo) * 4 : W::STAGE * 4];
    Lo* lo = (Lo*)lds;
    __shared__ float lm[4][16], ll[4][16];
    __shared__ typename W::Sizes size;
    __shared__ u64 bits[16];
    __shared__ __align__(16) float fac[4][4][32];
    // neighbouring blocks on one XCD (blocks go round the 8 XCDs): rows that share keys meet in its L2
    const i64 blocks = s.units * s.splits, a8 = (blocks + 7) / 8, me = (i64)(blockIdx.x % 8) * a8 + blockIdx.x / 8;
    if ((i64)blockIdx.x / 8 >= a8 || me >= blocks) return;
    const i64 unit = me / s.splits;
    const int split = (int)(me - unit * s.splits), G = s.a.G;
    const At p = at_of(s, (u32)unit);
    const int2 r = s.rows[p.row];
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
    st.stage = lds + wave * W::STAGE;
    const int* tab = a.table + p.row * a.width;
    W::begin(a, tab, p.head, base, stop, run);
    const bool own = W::load_q(a, 0, p.head, q, p.group * 16, (typename W::T*)lds, size, bits, st);
    lds_barrier();  // (each wave has its queries)
    st.m[0] = -__builtin_inff(), st.l[0] = 0.f;
#pragma unroll
    for (int j = 0; j < W::NJ; ++j) st.o[0][j] = f4{0.f, 0.f, 0.f, 0.f};
    W::keys(a, tab, p.head, q, base, stop, bits, size, own, run, st, fac[wave]);
    float m, sum, o[W::NJ];
    W::join_waves(st, 0, lo, lm, ll, m, sum, o);
    const int at = threadIdx.x >> 4, d0 = (threadIdx.x & 15) * W::NJ, h = p.group * 16 + at;
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
    const i64 unit = blockIdx.x;
    const At p = at_of(s, (u32)unit);
    const int h = p.group * 16 + (threadIdx.x >> 4), parts = share_of(s.rows[p.row].x, s.splits, 0).blocks;
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

// To the next bfloat16 above (or below) where x is none: towards zero, after 2^16 - 1 more where its size grows that way.
__device__ __forceinline__ b16 outward(float x, bool up) {
    const u32 u = __float_as_uint(x), negative = (u32)((int)u >> 31);
    return __builtin_bit_cast(b16, (u16)((u + ((up ? ~negative : negative) & 0xFFFFu)) >> 16));
}

// The smaller of two numbers (no NaN), one operation: fminf brings each operand into form first.
__device__ __forceinline__ float least(float a, float b) { return __builtin_amdgcn_fmed3f(a, b, -__builtin_inff()); }

// The smaller of a lane's and its partner's, 32 or 16 lanes on, of two values at once: half of the lanes keep each.
template <int O> __device__ __forceinline__ float halve(float a, float b) {
    const auto r = O == 32 ? __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(b), false, false)
                           : __builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(b), false, false);
    return least(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// WP waves per (sequence, page that its tokens touch, head): the elements' smallest and largest over the page's rows, where
// the tokens complete it. A lane holds E elements of a row, four rows' loads at a time. Of the lanes of one place in a row the
// lower half then keeps the smallest, the upper half the largest (as the smallest of the negatives).
// Pages of 32 rows of 8 heads of 128, 1125 of them: 12.7 us in 8 bits (3.4 TB/s), bound by vector instructions, 640 a wave of 64
// elements a lane (75 % of the time by counters; the sums over lanes at a page's end, 16 elements each, among them); 15.3 in 16
// bits (5.1 TB/s: memory).
template <int CODES, int DP, int WP>
__global__ __launch_bounds__(256) void bounds_k(const void* __restrict__ k, const float* __restrict__ ks, i64 pages, int shift,
                                                int H, int dim, const int* __restrict__ table, i64 stride, int width,
                                                const int* __restrict__ start, u32 items, int count, int per,
                                                b16* __restrict__ bounds) {
    constexpr bool Q8 = CODES == KV_INT8 || CODES == KV_FP8;
    constexpr int E = DP == 192 ? 12 : Q8 ? 16 : 8, L = DP / E, R = 64 / L;  // elements a lane, lanes a row, rows a wave
    constexpr int M = R > 2 ? E / 2 : E;                                     // elements that a lane ends with
    __shared__ float sides[WP == 1 ? 1 : 4][2][WP == 1 ? 1 : DP];
    const int wave = threadIdx.x >> 6, part = wave % WP, l = lane_id();
    const u32 item = blockIdx.x * (4 / WP) + wave / WP, page = item / (u32)H, b = page / (u32)per;
    const int h = (int)(item - page * H);
    int e = -1;
    if (item < items) {
        const i64 from = start[b], column = (from < 0 ? 0 : from >> shift) + (page - b * per);
        if ((column + 1) << shift <= from + count && column < width) e = table[b * stride + column];
    }
    if ((u32)e >= (u64)pages) return;  // (all waves of a page)
    const int r0 = part * R + l / L, d0 = l % L * E;
    const i64 first = ((i64)e * H + h) << shift;
    float x[E], hi[E];
    u32 bad = 0;     // elements that a NaN was seen in
    // Minima pass over NaN. That there may be one is noticed by words (a code of NaN, a scale that is not finite; 16 bits: an
    // element larger than infinity); only then the rows are read again with a look at each element.
    u32 odd = 0;
    auto rows = [&](auto careful) {
        constexpr bool EACH = decltype(careful)::value;
#pragma unroll
        for (int j = 0; j < E; ++j) x[j] = __builtin_inff(), hi[j] = -__builtin_inff();
        for (int r = r0; r < 1 << shift; r += 4 * WP * R) {
            u32 w[4][E * (Q8 ? 1 : 2) / 4];
            float s[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {  // (a row past the page is the first of the four again)
                const int at = r + u * WP * R < 1 << shift ? r + u * WP * R : r;
                load_words<E * (Q8 ? 1 : 2) / 4>((const char*)k + ((first + at) * DP + d0) * (Q8 ? 1 : 2), w[u]);
                s[u] = Q8 ? ks[first + at] : 1.f;
            }
            float v[4][E];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                if constexpr (Q8 && !EACH) odd |= finite_f(s[u]) ? 0u : 1u;
                if constexpr (CODES == KV_FP8) {
#pragma unroll
                    for (int i = 0; i < E / 4; ++i) {
                        const auto p = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[u][i], false);
                        const auto q = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[u][i], true);
                        v[u][4 * i] = p[0], v[u][4 * i + 1] = p[1], v[u][4 * i + 2] = q[0], v[u][4 * i + 3] = q[1];
                        if constexpr (!EACH) odd |= ((w[u][i] & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u;
                    }
                } else
#pragma unroll
                    for (int j = 0; j < E; ++j) {
                        if constexpr (CODES == KV_INT8) v[u][j] = (float)(signed char)(w[u][j / 4] >> (8 * (j & 3)));
                        else v[u][j] = (float)__builtin_bit_cast(typename op_t<CODES>::type, (u16)(w[u][j / 2] >> (16 * (j & 1))));
                        if constexpr (!Q8 && !EACH)
                            if (j & 1) {
                                constexpr u32 INF = CODES == KV_BF16 ? 0x7F80u : 0x7C00u;
                                const u32 size = w[u][j / 2] & 0x7FFF7FFFu;
                                odd |= (size >> 16 > INF) | ((size & 0xFFFFu) > INF);
                            }
                    }
#pragma unroll
                for (int j = 0; j < E; ++j) {
                    if constexpr (Q8) v[u][j] *= s[u];
                    if constexpr (EACH) bad |= (v[u][j] != v[u][j] ? 1u : 0u) << j;
                }
            }
#pragma unroll
            for (int j = 0; j < E; ++j) {
                x[j] = fminf(fminf(x[j], v[0][j]), fminf(v[1][j], fminf(v[2][j], v[3][j])));
                hi[j] = fmaxf(fmaxf(hi[j], v[0][j]), fmaxf(v[1][j], fmaxf(v[2][j], v[3][j])));
            }
        }
    };
    rows(std::false_type());
    if (__any(odd != 0)) {
        rows(std::true_type());
#pragma unroll
        for (int o = L; o < 64; o <<= 1) bad |= (u32)__shfl_xor((int)bad, o, 64);
    }
#pragma unroll
    for (int j = 0; j < E; ++j) x[j] = halve<32>(x[j], -hi[j]);
    if constexpr (R > 2)
#pragma unroll
        for (int j = 0; j < M; ++j) x[j] = halve<16>(x[j], x[M + j]);
    if constexpr (R > 4)
#pragma unroll
        for (int o = 8; o >= L; o >>= 1)
#pragma unroll
            for (int j = 0; j < M; ++j) x[j] = least(x[j], __shfl_xor(x[j], o, 64));
    // lane l: the smallest (l < 32) or the largest of elements d .. d + M - 1
    const int side = l >> 5, skip = R > 2 ? (l >> 4 & 1) * M : 0, d = d0 + skip;
    const bool mine = R <= 4 || (l & 15) < L;
#pragma unroll
    for (int j = 0; j < M; ++j) x[j] = side ? -x[j] : x[j];
    if (__any(bad != 0))
#pragma unroll
        for (int j = 0; j < M; ++j) x[j] = bad >> (skip + j) & 1 ? __builtin_nanf("") : x[j];
    if constexpr (WP > 1)
        if (mine)
#pragma unroll
            for (int j = 0; j < M; ++j) sides[wave][side][d + j] = x[j];
    if constexpr (WP > 1) {
        __syncthreads();
        if (part) return;
#pragma unroll
        for (int j = 0; j < M; ++j) {
#pragma unroll
            for (int w = 1; w < WP; ++w) {
                const float y = sides[wave + w][side][d + j];
                x[j] = x[j] != x[j] || y != y ? __builtin_nanf("") : side ? fmaxf(x[j], y) : fminf(x[j], y);
            }
        }
    }
    if (!mine) return;
    constexpr int N = M % 4 ? 2 : M == 4 ? 4 : 8;  // elements a store
    b16* to = bounds + (((i64)e * H + h) * 2 + side) * DP + d;
#pragma unroll
    for (int i = 0; i < M; i += N) {
        Pack<b16, N> o;
#pragma unroll
        for (int j = 0; j < N; ++j) o.v[j] = d + i + j < dim ? outward(x[i + j], side != 0) : (b16)0.f;
        o.store(to + i);
    }
}

template <int CODES> int bounds_codes(const void* k, const float* ks, i64 pages, int shift, int H, int dim, const int* table,
                                      i64 stride, int width, const int* start, int B, int count, b16* bounds,
                                      hipStream_t st) {
    const int touched = ((count - 1) >> shift) + 2, per = touched < width ? touched : width;  // pages a sequence
    // A wave a page and head, or a block where the page is larger: 64 sequences' pages of 8 heads of 128 in 8 bits take 10.5 us
    // by waves and 13.2 by blocks at 256 rows, 28.2 and 24.8 at 1024; in 16 bits 8.6 and 7.7 at 128.
    const int waves = shift > (CODES == KV_INT8 || CODES == KV_FP8 ? 8 : 6) ? 4 : 1;
    // a launch has fewer than 2^32 threads: so many sequences at a time
    const i64 each = (i64)per * H, most = ((((i64)1 << 26) - 4) / waves) / each;
    if (most < 1) return -1;
    for (i64 b0 = 0; b0 < B; b0 += most, table += most * stride, start += most) {
        const i64 n = (B - b0 < most ? B - b0 : most) * each, grid = (n * waves + 3) / 4;
#define BOUNDS_K(DP, WP) \
    bounds_k<CODES, DP, WP><<<(unsigned)grid, 256, 0, st>>>(k, ks, pages, shift, H, dim, table, stride, width, start, (u32)n, count, per, bounds)
#define DP_CASE(DP)            \
    if (waves == 4) BOUNDS_K(DP, 4); \
    else BOUNDS_K(DP, 1)
        switch ((dim + 63) / 64) {
            case 1: DP_CASE(64); break;
            case 2: DP_CASE(128); break;
            case 3: DP_CASE(192); break;
            default: DP_CASE(256);
        }
        const int rc = (int)hipGetLastError();
        if (rc) return rc;
    }
#undef DP_CASE
#undef BOUNDS_K
    return 0;
}
