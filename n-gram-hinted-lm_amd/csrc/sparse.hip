// Attention of new tokens over the pages of a cache that a cheap score chooses.
//
//   bounds[page, head]   (min, max) over the page's keys of each element, outward to bfloat16
//   score(token, head, page) = sum over the group's query heads g and elements d of max(q[g, d] lo[d], q[g, d] hi[d])
//                            = sum_d (sum_g max(q[g, d], 0)) hi[d] + (sum_g min(q[g, d], 0)) lo[d],  a zero counting nothing
//   kept: of the pages that hold positions 0 .. the token's own, the first and the last ones and the best others
//   o = softmax attention over the kept pages' keys at positions up to the token's own
//
// A page's score is at least the sum over the group of the largest q . k of any of its keys. The second form needs one product
// a page whatever the group's size. It is computed in 64 bits: 16-bit products are exact there and a sum of 512 is off by
// 2^-44 of its terms, so which page is kept does not depend on the order of the sum. Memory bounds it (4 bytes an element).
//
// Choosing: a row's keys lie in registers, and halving the range between the smallest and largest finds the threshold that
// leaves `keep` (equal scores: the lower pages). The kept pages' numbers in the cache, in order, are the page table of a tree
// attention (tree.h) of one token, whose last page is the token's own.
//
// Measured (in a trace, us; 8 heads of 128, groups of 4, but for the last):
//   a token over 5000 positions, 32 of 313 pages of 16        scores 5.4, choice 5.6, attention 10.7: launches and latency
//   32 tokens over up to 32768, 32 of 512 pages of 64         both 18.0 (the longest rows' blocks), attention 29.8 (4.6 TB/s)
//   2 x 4 tokens over 524288, 64 of 8192 pages                scores 22, choice 15.4 (a block a row), attention 16 and 4.9
//   1024 tokens over 16001, 5 heads of 80, groups of 3, 24 of 533 pages of 32
//                                                             scores 32 (the 64-bit products), choice 11, attention 105
// The last one's attention reads 2 GB of pages, 83 % of it from the L2s, for products of which 3 rows in 16 are used.
#include "choose.h"
#include "sparse.h"

#define MOST_PAGES 32768  // of a sequence

struct ScoreArgs {
    const void* q;
    i64 qb, qt, qh;
    const b16* bounds;  // [pages, H, 2, DP], zeros behind dim
    const int* table;
    i64 table_stride, pages;
    const int *lengths, *widths;
    int B, T, H, G, dim, shift, width, keep, first, last, qtype, vec;
    int b0, t0, nt;       // this pass: tokens t0 .. t0 + nt - 1 of sequences b0 on
    i64 rows;             // its rows: (sequence, token, head)
    u64* score;           // [rows, width]
    int* table_out;       // [rows, keep]: the kept pages of the cache
    int2* row_out;        // [rows]
    int* chosen;          // [B, T, H, keep] or NULL: the kept pages' places in the sequence, -1 behind them
    int chunks, per;      // blocks a row, and the pages of each
};

// A row's token: whether it is in use, the pages it sees, and its keys' number over all of them.
struct Place {
    bool is;
    int b, t, h, pages;
    i64 len, keys;  // the tokens before the sequence's first of the call, and those that it sees
};
__device__ __forceinline__ Place place_of(const ScoreArgs& a, u32 row) {  // (a pass has fewer than 2^31 rows)
    Place p;
    const u32 token = row / (u32)a.H, b = token / (u32)a.nt;
    const i64 cap = (i64)a.width << a.shift;
    p.h = (int)(row - token * a.H), p.b = a.b0 + (int)b, p.t = a.t0 + (int)(token - b * a.nt);
    const int l = a.lengths[p.b], w = a.widths ? a.widths[p.b] : a.T;
    p.len = l < 0 ? 0 : l > cap ? cap : l;
    p.is = p.t < w;
    p.keys = p.len + p.t + 1 < cap ? p.len + p.t + 1 : cap;
    p.pages = (int)((p.keys + (1 << a.shift) - 1) >> a.shift);
    return p;
}

__device__ __forceinline__ float query_at(const ScoreArgs& a, u16 e) {
    return a.qtype == NG_BF16 ? __uint_as_float((u32)e << 16) : (float)__builtin_bit_cast(f16, e);
}

// A score as a key, its upper word above 0: a page of none of the cache's ranks last, one whose score is NaN first.
__device__ __forceinline__ u64 score_key(bool is, double x) {
    const u64 u = (u64)__double_as_longlong(x + 0.);
    return !is ? 1ull << 32 : x != x ? ~1ull : u >> 63 ? ~u : u | 1ull << 63;
}

// The pairs of elements of four words, 16 bits each, in 64 bits.
__device__ __forceinline__ double low(u32 w) { return (double)__uint_as_float(w << 16); }
__device__ __forceinline__ double high(u32 w) { return (double)__uint_as_float(w & 0xFFFF0000u); }

// A sum of queries of one sign times a bound. Without such queries nothing of the bound counts: 0 where it is infinite, too
// (its product with 0 is NaN; sums that come out as NaN are taken again so).
__device__ __forceinline__ double times(double q, double x) { return q == 0. && __builtin_isinf(x) ? 0. : q * x; }

// A token's scores of pages from .. stop - 1, by a block of NT: GS lanes a page, each of 8 elements, 4 pages at a time. put
// takes those that are wanted.
template <int DP, int GS, int NT, typename F>
__device__ __forceinline__ void score_one(const ScoreArgs& a, const Place& p, int from, int stop, F put) {
    constexpr int U = 4, STEP = NT / GS;
    const int sub = threadIdx.x % GS, group = threadIdx.x / GS, d0 = sub * 8;
    const int* tab = a.table + p.b * a.table_stride;
    int e[U], next[U];  // (asked for before the sequence's length is known)
#pragma unroll
    for (int u = 0; u < U; ++u) e[u] = from + group + u * STEP < stop ? tab[from + group + u * STEP] : -1;
    double up[8], down[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) up[j] = down[j] = 0.;
    const u16* q = (const u16*)a.q + p.b * a.qb + p.t * a.qt + (i64)p.h * a.G * a.qh + d0;
    if (p.is)
        for (int g = 0; g < a.G; ++g, q += a.qh) {
            union {
                uint4 w;
                u16 e[8];
            } x;
            x.w = make_uint4(0, 0, 0, 0);
            if (a.vec && d0 + 8 <= a.dim) x.w = *(const uint4*)q;
            else
                for (int j = 0; j < 8; ++j)
                    if (d0 + j < a.dim) x.e[j] = q[j];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float f = query_at(a, x.e[j]);
                up[j] += f > 0.f || f != f ? (double)f : 0.;
                down[j] += f < 0.f ? (double)f : 0.;
            }
        }
    const int end = p.pages - a.last < stop ? p.pages - a.last : stop;
    if (!p.is || p.pages <= a.keep || from >= end) return;
    for (int j0 = from + group; j0 < end; j0 += STEP * U) {
        uint4 lo[U], hi[U];
        bool is[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int j = j0 + u * STEP;
            is[u] = (u32)e[u] < (u64)a.pages;
            lo[u] = hi[u] = make_uint4(0, 0, 0, 0);
            if (is[u] && j < end && d0 < DP) {
                const b16* x = a.bounds + ((i64)e[u] * a.H + p.h) * 2 * DP + d0;
                lo[u] = *(const uint4*)x, hi[u] = *(const uint4*)(x + DP);
            }
            next[u] = j + STEP * U < stop ? tab[j + STEP * U] : -1;
        }
        double acc[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            acc[u] = 0.;
            const u32 l[4] = {lo[u].x, lo[u].y, lo[u].z, lo[u].w}, h[4] = {hi[u].x, hi[u].y, hi[u].z, hi[u].w};
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const double x = j & 1 ? high(l[j / 2]) : low(l[j / 2]), y = j & 1 ? high(h[j / 2]) : low(h[j / 2]);
                acc[u] = fma(down[j], x, fma(up[j], y, acc[u]));
            }
        }
        // (the bounds are read again: held for this they would cost every call 20 registers)
        if (__any(acc[0] != acc[0] || acc[1] != acc[1] || acc[2] != acc[2] || acc[3] != acc[3]))
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (!is[u] || acc[u] == acc[u]) continue;
                const b16* x = a.bounds + ((i64)e[u] * a.H + p.h) * 2 * DP + d0;
                acc[u] = 0.;
#pragma unroll
                for (int j = 0; j < 8; ++j) acc[u] += times(down[j], (double)(float)x[j]) + times(up[j], (double)(float)x[DP + j]);
            }
        // the four pages' sums over the lanes, each step for half as many pages: a quarter of the lanes ends with each
        const bool a1 = sub & (GS / 2), a2 = sub & (GS / 4);
        double x = (a1 ? acc[2] : acc[0]) + __shfl_xor(a1 ? acc[0] : acc[2], GS / 2, GS);
        double y = (a1 ? acc[3] : acc[1]) + __shfl_xor(a1 ? acc[1] : acc[3], GS / 2, GS);
        x = (a2 ? y : x) + __shfl_xor(a2 ? x : y, GS / 4, GS);
#pragma unroll
        for (int o = GS / 8; o; o >>= 1) x += __shfl_xor(x, o, GS);
        const int u = (a1 ? 2 : 0) + (a2 ? 1 : 0), j = j0 + u * STEP;
        const bool mine = a1 ? (a2 ? is[3] : is[2]) : (a2 ? is[1] : is[0]);
        if (j >= a.first && j < end && sub % (GS / 4) == 0) put(j, score_key(mine, x));
#pragma unroll
        for (int u = 0; u < U; ++u) e[u] = next[u];
    }
}

// One token a sequence: a block per (row, a.per pages).
template <int DP, int GS> __global__ __launch_bounds__(256) void score_one_k(const ScoreArgs a) {
    const i64 row = blockIdx.x / (u32)a.chunks;
    const int from = (int)(blockIdx.x - row * a.chunks) * a.per, stop = from + a.per < a.width ? from + a.per : a.width;
    score_one<DP, GS, 256>(a, place_of(a, (u32)row), from, stop, [&](int j, u64 x) { a.score[row * a.width + j] = x; });
}

typedef double d4 __attribute__((ext_vector_type(4)));

// Products of TT tokens and 16 pages over 4 elements: a lane's operands are of token lane % TT, page lane % 16 and element
// lane / 16, its sums those of tokens 4 r + lane / 16 and page lane % 16.
template <int TT> struct Sums;
template <> struct Sums<16> {
    typedef d4 type;
    static __device__ __forceinline__ d4 mma(double t, double p, d4 s) { return __builtin_amdgcn_mfma_f64_16x16x4f64(t, p, s, 0, 0, 0); }
    static __device__ __forceinline__ double at(d4 s, int r) { return s[r]; }
};
template <> struct Sums<4> {
    typedef double type;
    static __device__ __forceinline__ double mma(double t, double p, double s) { return __builtin_amdgcn_mfma_f64_4x4x4f64(t, p, s, 0, 0, 0); }
    static __device__ __forceinline__ double at(double s, int) { return s; }
};

// Several tokens a sequence: a block per (TT tokens, 16 or 4, of a sequence and head, a.per pages), on the matrix units: tokens
// x pages, 16 pages a wave at a time (TT = 4: as four products of 4 x 4). A lane's operand is 8 in 32 elements of a page's
// bounds (of one page in 16) and the same ones of a token's sums, which lie in LDS.
template <int DP, int TT> __global__ __launch_bounds__(256, DP <= 128 ? 4 : 2) void score_k(const ScoreArgs a) {
    constexpr int LD = 2 * DP + 2;  // (16 rows' reads of 16 bytes meet no bank twice)
    __shared__ __align__(16) double sums[TT * LD];
    const int c = lane_id() & 15, g = lane_id() >> 4, wave = threadIdx.x >> 6;
    const u32 tiles = (a.nt + TT - 1) / TT, unit = blockIdx.x / (u32)a.chunks, bh = unit / tiles;  // (sequence, head, TT tokens)
    const u32 at = bh / (u32)a.H;
    const int chunk = (int)(blockIdx.x - unit * a.chunks), tile = (int)(unit - bh * tiles) * TT;
    const int h = (int)(bh - at * a.H), b = a.b0 + (int)at, t0 = a.t0 + tile;
    const int n = a.nt - tile < TT ? a.nt - tile : TT;
    const i64 row0 = ((i64)at * a.nt + tile) * a.H + h;
    const Place whole = place_of(a, (u32)(row0 + (i64)(n - 1) * a.H));  // the last token sees the most pages
    const int from = chunk * a.per;
    const int stop = from + a.per < whole.pages - a.last ? from + a.per : whole.pages - a.last;
    if (whole.pages <= a.keep || from >= stop) return;
    const int w = a.widths ? a.widths[b] : a.T;
    if (t0 >= w) return;
    for (int i = threadIdx.x; i < TT * DP / 8; i += 256) {
        const int t = i / (DP / 8), d0 = i % (DP / 8) * 8;
        double up[8], down[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) up[j] = down[j] = 0.;
        if (t < n && t0 + t < w) {
            const u16* q = (const u16*)a.q + b * a.qb + (t0 + t) * a.qt + (i64)h * a.G * a.qh + d0;
            for (int k = 0; k < a.G; ++k, q += a.qh) {
                union {
                    uint4 w;
                    u16 e[8];
                } x;
                x.w = make_uint4(0, 0, 0, 0);
                if (a.vec && d0 + 8 <= a.dim) x.w = *(const uint4*)q;
                else
                    for (int j = 0; j < 8; ++j)
                        if (d0 + j < a.dim) x.e[j] = q[j];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float f = query_at(a, x.e[j]);
                    up[j] += f > 0.f || f != f ? (double)f : 0.;
                    down[j] += f < 0.f ? (double)f : 0.;
                }
            }
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) sums[t * LD + d0 + j] = up[j], sums[t * LD + DP + d0 + j] = down[j];
    }
    __syncthreads();
    const int* tab = a.table + b * a.table_stride;
    const double* mine = sums + c % TT * LD + g * 8;
    const int steps = (a.dim + 31) / 32;
    u64* out = a.score + (row0 + (i64)g * a.H) * a.width;
    int ends[TT / 4];  // behind the last page that a token's score is wanted of
#pragma unroll
    for (int r = 0; r < TT / 4; ++r) {
        const int t = 4 * r + g;
        const i64 keys = whole.len + t0 + t + 1, cap = (i64)a.width << a.shift;
        const int pages = (int)(((keys < cap ? keys : cap) + (1 << a.shift) - 1) >> a.shift);
        ends[r] = t < n && t0 + t < w ? (pages - a.last < stop ? pages - a.last : stop) : 0;
    }
    auto entry = [&](int j) { return j + c < stop ? tab[j + c] : -1; };
    auto page = [&](int e) { return a.bounds + ((i64)((u32)e < (u64)a.pages ? e : 0) * a.H + h) * 2 * DP + g * 8; };
    int e = entry(from + wave * 16), next = entry(from + wave * 16 + 64);
    const b16* x = page(e);
    uint4 lo = *(const uint4*)x, hi = *(const uint4*)(x + DP);
    for (int j0 = from + wave * 16; j0 < stop; j0 += 64) {
        const bool is = (u32)e < (u64)a.pages;
        const b16 *now = page(e) - g * 8, *then = page(next);
        e = next, next = entry(j0 + 128);
        typename Sums<TT>::type acc = {}, more = {};
#pragma unroll 1
        for (int i = 0; i < steps; ++i) {  // (the next eight elements, or the next page's first, are under way)
            const u32 l[4] = {lo.x, lo.y, lo.z, lo.w}, k[4] = {hi.x, hi.y, hi.z, hi.w};
            x = i + 1 < steps ? x + 32 : then;
            lo = *(const uint4*)x, hi = *(const uint4*)(x + DP);
#pragma unroll
            for (int j = 0; j < 8; j += 2) {
                const double2 up = *(const double2*)(mine + i * 32 + j), down = *(const double2*)(mine + DP + i * 32 + j);
                acc = Sums<TT>::mma(up.x, low(k[j / 2]), acc);
                more = Sums<TT>::mma(down.x, low(l[j / 2]), more);
                acc = Sums<TT>::mma(up.y, high(k[j / 2]), acc);
                more = Sums<TT>::mma(down.y, high(l[j / 2]), more);
            }
        }
        const int j = j0 + c;  // this lane's page; its tokens: 4 r + g
#pragma unroll
        for (int r = 0; r < TT / 4; ++r)
            if (j >= a.first && j < ends[r]) {
                double x = Sums<TT>::at(acc, r) + Sums<TT>::at(more, r);
                if (is && x != x) {
                    const double *up = sums + (4 * r + g) * LD, *down = up + DP;
                    x = 0.;
#pragma unroll 1
                    for (int d = 0; d < a.dim; ++d)
                        x += times(down[d], (double)(float)now[d]) + times(up[d], (double)(float)now[DP + d]);
                }
                out[(i64)r * 4 * a.H * a.width + j] = score_key(is, x);
            }
    }
}

// The kept pages of a row, by NW waves that hold E of its scores (score(j)) a lane.
template <int NW, int E, typename F>
__device__ __forceinline__ void choose(const ScoreArgs& a, const Place& p, i64 row, F score) {
    constexpr int NT = NW * 64;
    __shared__ int counts[2][NW], before[NW == 1 ? 1 : E * NW];
    __shared__ u32 ends[2][NW];
    const int tid = NW == 1 ? lane_id() : (int)threadIdx.x, wave = NW == 1 ? 0 : tid >> 6;
    const int* tab = a.table + p.b * a.table_stride;
    int* out = a.table_out + row * a.keep;
    int* chosen = a.chosen ? a.chosen + (((i64)p.b * a.T + p.t) * a.H + p.h) * a.keep : nullptr;
    const int n = p.is ? p.pages : 0, kept = n < a.keep ? n : a.keep;
    if (tid == 0) {
        const int rest = n ? (int)(p.keys - ((i64)(n - 1) << a.shift)) : 0;
        a.row_out[row] = make_int2(n ? ((kept - 1) << a.shift) + rest : 0, p.is);
    }
    for (int i = kept + tid; i < a.keep; i += NT) {
        out[i] = -1;
        if (chosen) chosen[i] = -1;
    }
    if (n <= a.keep) {
        for (int i = tid; i < n; i += NT) {
            out[i] = tab[i];
            if (chosen) chosen[i] = i;
        }
        return;
    }
    // the upper words of the scores decide but where they are equal (a score's first 20 bits): then the lower ones
    u32 key[E], rest[E], lo = ~0u, hi = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int j = e * NT + tid;
        u64 k = 0;
        if (j < n) k = j < a.first || j >= n - a.last ? ~0ull : score(j);
        key[e] = (u32)(k >> 32), rest[e] = (u32)k;
        if (j < n) lo = key[e] < lo ? key[e] : lo;
        if (key[e] != ~0u) hi = key[e] > hi ? key[e] : hi;
    }
    lo = min_wave(lo), hi = max_wave(hi);
    if constexpr (NW > 1) {
        if (lane_id() == 0) ends[0][wave] = lo, ends[1][wave] = hi;
        lds_barrier();
#pragma unroll
        for (int w = 0; w < NW; ++w) lo = ends[0][w] < lo ? ends[0][w] : lo, hi = ends[1][w] > hi ? ends[1][w] : hi;
    }
    Count<NW> count(counts);
    auto few = [&](const u32 (&k)[E], u32 least) {  // the keys from `least` on, no more than lanes: one each, 0 behind them
        __shared__ u32 left[NW == 1 ? 256 : NT];
        __shared__ int fill[4];
        u32* mine = left + (NW == 1 ? threadIdx.x / 64 * 64 : 0);
        int at = 0;
        if constexpr (NW > 1) {
            if (tid == 0) fill[0] = 0;
            mine[tid] = 0;
            __syncthreads();
        } else mine[tid] = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const bool is = k[e] >= least;
            const u64 m = __ballot(is);
            int first = at;
            if constexpr (NW > 1) {
                if (!m) continue;
                if (lane_id() == 0) first = atomicAdd(fill, __popcll(m));
                first = __builtin_amdgcn_readfirstlane(first);
            }
            if (is) mine[first + __popcll(m & lanemask_lt())] = k[e];
            at += __popcll(m);
        }
        if constexpr (NW > 1) __syncthreads();
        else {
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
            __builtin_amdgcn_wave_barrier();
        }
        return mine[tid];
    };
    int c;
    // (an upper word of ones: a page always kept, or a NaN, whose lower word is one less; hi is below both)
    u32 t = ~0u, t2 = 0;
    int equal = E * NT;  // of the scores equal to t and t2, the first so many
    c = count.at_least(key, t);
    if (c < a.keep) {
        c = n;
        // halving with all keys until a key a lane is left, then with those
        t = count.threshold(key, lo, hi, a.keep, a.keep > NT ? a.keep : NT, c);
        if (c > a.keep) {
            if (E > 1 && c <= NT) {
                u32 one[1] = {few(key, t)};
                t = count.threshold(one, t, hi, a.keep, a.keep, c);
            } else t = count.threshold(key, t, hi, a.keep, a.keep, c);
        }
    }
    if (c > a.keep) {
        const int above = t == ~0u ? 0 : count.at_least(key, t + 1);
#pragma unroll
        for (int e = 0; e < E; ++e) rest[e] = key[e] == t ? rest[e] : 0u;
        c -= above;
        t2 = count.threshold(rest, 0u, ~0u, a.keep - above, a.keep - above, c);
        if (c > a.keep - above) equal = a.keep - above - (t2 == ~0u ? 0 : count.at_least(rest, t2 + 1));
    }
    // in order of the pages: first how many of each wave's 64 come before
    auto place = [&](auto is, auto got) {
        int run = 0;
        if constexpr (NW > 1) {
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const u64 m = __ballot(is(e));
                if (lane_id() == 0) before[e * NW + wave] = __popcll(m);
            }
            __syncthreads();
            if (wave == 0) {
                int sum = 0;
                for (int i = 0; i < E * NW; i += 64) {
                    const int x = i + lane_id() < E * NW ? before[i + lane_id()] : 0, inc = scan_wave(x);
                    if (i + lane_id() < E * NW) before[i + lane_id()] = sum + inc - x;
                    sum += __shfl(inc, 63, 64);
                }
            }
            __syncthreads();
        }
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const bool mine = is(e);
            const u64 m = __ballot(mine);
            if (mine) got(e, (NW > 1 ? before[e * NW + wave] : run) + __popcll(m & lanemask_lt()));
            run += __popcll(m);
        }
        if constexpr (NW > 1) __syncthreads();
    };
    u32 take = 0;
    static_assert(E <= 32, "a bit each");
#pragma unroll
    for (int e = 0; e < E; ++e) take |= (key[e] > t || (key[e] == t && rest[e] >= t2) ? 1u : 0u) << e;
    if (equal < E * NT) {
        u32 drop = 0;
        place([&](int e) { return key[e] == t && rest[e] == t2; }, [&](int e, int i) { drop |= (i < equal ? 0u : 1u) << e; });
        take &= ~drop;
    }
    place([&](int e) { return (take >> e & 1) != 0; }, [&](int e, int i) {
        const int j = e * NT + tid;
        out[i] = tab[j];
        if (chosen) chosen[i] = j;
    });
}

// (NW = 1: four rows a block)
template <int NW, int E> __global__ __launch_bounds__(NW == 1 ? 256 : NW * 64) void choose_k(const ScoreArgs a) {
    const i64 row = NW == 1 ? (i64)blockIdx.x * 4 + (threadIdx.x >> 6) : (i64)blockIdx.x;
    if (row >= a.rows) return;
    choose<NW, E>(a, place_of(a, (u32)row), row, [&](int j) { return a.score[row * a.width + j]; });
}

// Both for one token a sequence of few pages, a block a row.
#define FEW_PAGES 1024
template <int DP, int GS> __global__ __launch_bounds__(512) void score_choose_k(const ScoreArgs a) {
    __shared__ u64 scores[FEW_PAGES];
    const i64 row = blockIdx.x;
    const Place p = place_of(a, (u32)row);
    score_one<DP, GS, 512>(a, p, 0, a.width, [&](int j, u64 x) { scores[j] = x; });
    __syncthreads();
    choose<8, FEW_PAGES / 512>(a, p, row, [&](int j) { return scores[j]; });
}

// ------------------------------------------------------------------------------------------------------------ the host

#define SLAB ((i64)256 << 20)  // bytes of scores and kept pages at a time
#define AIM 512                // blocks that fill the card: 2 a CU

struct SparsePlan {
    int dp, groups, splits;
    bool scored;
    int nb, nt;  // sequences and tokens of each at a time
    i64 score, table, rows, po, pm, bytes;  // offsets in the workspace
};

static bool sparse_plan(i64 B, i64 T, i64 H, i64 G, i64 dim, i64 width, i64 page, i64 keep, SparsePlan& p) {
    const i64 lim = (i64)1 << 30;
    if (B < 0 || T < 1 || H < 1 || G < 1 || dim < 1 || dim > 256 || width < 1 || width > MOST_PAGES || keep < 1 || keep > 1024 ||
        B > lim || T > lim || H > lim || G > 1 << 20 || page < 16 || page > 4096 || (page & (page - 1)) ||
        width * page > lim || B * T > lim || H * ((G + 15) / 16) > 1 << 12)
        return false;
    p.dp = (int)(dim + 63) / 64 * 64, p.groups = (int)(G + 15) / 16, p.scored = width > keep;
    // a pass takes as many sequences, or one sequence's tokens, as SLAB holds the scores and kept pages of, fewer than 2^23 units
    // (blocks of up to 512 threads, fewer than 2^32 in a launch)
    const i64 each = H * ((p.scored ? width * 8 : 0) + keep * 4), most_units = (((i64)1 << 23) - 1) / (H * p.groups);
    i64 most = SLAB / each < most_units ? SLAB / each : most_units;
    if (most < 16) most = 16;
    p.nt = (int)(T <= most ? T : most / 16 * 16);
    p.nb = (int)(T <= most ? (B < most / T ? B : most / T) : 1);
    const i64 rows = (B ? (i64)p.nb : 0) * p.nt * H, units = rows * p.groups;
    const i64 tiles = ((keep < width ? keep : width) * page + TILE - 1) / TILE;
    // A block a unit where the units fill the CUs (256: 30.0 us and no joining; in two parts each 28.3 and 4.3), else parts that
    // make AIM blocks, of two tiles at least. Up to six tiles are left whole: joining their parts costs more than they take (8
    // units of four tiles: 10.8 us, in halves 8.7 and 2.6 in two launches).
    i64 splits = units && units < 256 && tiles > 6 ? (AIM + units - 1) / units : 1;
    p.splits = (int)(splits < (tiles + 1) / 2 ? splits : (tiles + 1) / 2);
    const i64 parts = p.splits > 1 ? units * p.splits * 16 : 0;
    p.score = 0;
    p.rows = p.score + (p.scored ? rows * width * 8 : 0);
    p.table = p.rows + rows * 8;
    p.po = (p.table + rows * keep * 4 + 15) / 16 * 16;
    p.pm = p.po + parts * p.dp * 4;
    p.bytes = p.pm + 2 * parts * 4;
    return true;
}

extern "C" i64 ng_sparse_work(i64 B, i64 T, i64 H, i64 G, i64 dim, i64 width, i64 page, i64 keep) {
    SparsePlan p;
    return sparse_plan(B, T, H, G, dim, width, page, keep, p) ? p.bytes : -1;
}

extern template int sparse_codes<KV_INT8>(const SparseArgs&, int, hipStream_t);
extern template int sparse_codes<KV_FP8>(const SparseArgs&, int, hipStream_t);
extern template int sparse_codes<KV_BF16>(const SparseArgs&, int, hipStream_t);
extern template int sparse_codes<KV_F16>(const SparseArgs&, int, hipStream_t);
#define BOUNDS(C)                                                                                                         \
    extern template int bounds_codes<C>(const void*, const float*, i64, int, int, int, const int*, i64, int, const int*, int, \
                                        int, b16*, hipStream_t)
BOUNDS(KV_INT8);
BOUNDS(KV_FP8);
BOUNDS(KV_BF16);
BOUNDS(KV_F16);
#undef BOUNDS

extern "C" int ng_page_bounds(const void* k, const float* ks, i64 pages, int page, int heads, int dim, int codes,
                              const int* table, i64 stride, int width, const int* start, int B, int count, void* bounds,
                              void* stream) {
    if (pages < 1 || pages >= (i64)1 << 31 || page < 16 || page > 4096 || (page & (page - 1)) || heads < 1 || dim < 1 ||
        dim > 256 || codes < KV_INT8 || codes > KV_F16 || width < 1 || B < 0 || count < 0 || count >= 1 << 30 ||
        ((codes == KV_INT8 || codes == KV_FP8) && !ks))
        return -1;
    if (B == 0 || count == 0) return 0;
    hipStream_t st = (hipStream_t)stream;
    const int sh = __builtin_ctz((unsigned)page);
    switch (codes) {
#define CASE(C) \
    case C: return bounds_codes<C>(k, ks, pages, sh, heads, dim, table, stride, width, start, B, count, (b16*)bounds, st)
        CASE(KV_INT8);
        CASE(KV_FP8);
        CASE(KV_BF16);
        default: return bounds_codes<KV_F16>(k, ks, pages, sh, heads, dim, table, stride, width, start, B, count, (b16*)bounds, st);
#undef CASE
    }
}

template <int TT> static void score_tokens(const ScoreArgs& a, int dp, unsigned grid, hipStream_t st) {
    switch (dp) {
        case 64: score_k<64, TT><<<grid, 256, 0, st>>>(a); break;
        case 128: score_k<128, TT><<<grid, 256, 0, st>>>(a); break;
        case 192: score_k<192, TT><<<grid, 256, 0, st>>>(a); break;
        default: score_k<256, TT><<<grid, 256, 0, st>>>(a);
    }
}

// One token a sequence is scored by vector operations (32 over up to 512 pages: 14.7 us, on the matrix units 17.2), more on the
// matrix units, up to four by products of 4 x 4 (2 x 4 over 8192 pages: 21.5 us, by 16 x 16 26.6). A block takes 256 pages, or
// fewer (64 at least) where that leaves fewer than 1024 blocks.
static int score_rows(ScoreArgs& a, int nb, int dp, hipStream_t st) {
    const int tokens = a.T == 1 ? 1 : a.T <= 4 ? 4 : 16;
    const i64 units = (i64)nb * a.H * ((a.nt + tokens - 1) / tokens);
    i64 per = units * a.width / 1024;
    per = per < 256 ? (per + 63) / 64 * 64 : 256;
    a.per = per ? (int)per : 64;
    a.chunks = (a.width + a.per - 1) / a.per;
    const i64 n = units * a.chunks;
    if (n >= (i64)1 << 24) return -1;  // (a pass has fewer)
    if (tokens == 4) score_tokens<4>(a, dp, (unsigned)n, st);
    else if (tokens == 16) score_tokens<16>(a, dp, (unsigned)n, st);
    else switch (dp) {
        case 64: score_one_k<64, 8><<<(unsigned)n, 256, 0, st>>>(a); break;
        case 128: score_one_k<128, 16><<<(unsigned)n, 256, 0, st>>>(a); break;
        case 192: score_one_k<192, 32><<<(unsigned)n, 256, 0, st>>>(a); break;
        default: score_one_k<256, 32><<<(unsigned)n, 256, 0, st>>>(a);
    }
    return (int)hipGetLastError();
}

extern "C" int ng_sparse_attention(const void* q, i64 qb, i64 qt, i64 qh, int qtype, const void* k, const void* v,
                                   const float* ks, const float* vs, const void* bounds, i64 pages, int page, int codes,
                                   const int* table, i64 table_stride, int width, const int* lengths, const int* widths,
                                   int B, int T, int H, int G, int dim, int keep, int first, int last, float scale,
                                   void* out, float* lse, int* chosen, void* work, void* stream) {
    SparsePlan p;
    if (pages < 1 || pages >= (i64)1 << 31 || codes < KV_INT8 || codes > KV_F16 || (qtype != NG_BF16 && qtype != NG_F16) ||
        (codes == KV_BF16 && qtype != NG_BF16) || (codes == KV_F16 && qtype != NG_F16) ||
        ((codes == KV_INT8 || codes == KV_FP8) && (!ks || !vs)) || first < 0 || last < 1 || first > keep - last ||
        !sparse_plan(B, T, H, G, dim, width, page, keep, p))
        return -1;
    if (B == 0) return 0;
    char* w = (char*)work;
    ScoreArgs s;
    s.q = q, s.qb = qb, s.qt = qt, s.qh = qh, s.bounds = (const b16*)bounds, s.table = table, s.table_stride = table_stride;
    s.pages = pages, s.lengths = lengths, s.widths = widths, s.B = B, s.T = T, s.H = H, s.G = G, s.dim = dim;
    s.shift = __builtin_ctz((unsigned)page), s.width = width, s.keep = keep, s.first = first, s.last = last;
    s.qtype = qtype, s.vec = ((u64)q & 15) == 0 && (((qb | qt | qh) * 2) & 15) == 0;
    s.score = (u64*)(w + p.score), s.table_out = (int*)(w + p.table), s.row_out = (int2*)(w + p.rows), s.chosen = chosen;
    SparseArgs r;
    TreeArgs& a = r.a;
    a.q = q, a.qb = qb, a.qt = qt, a.qh = qh, a.k = k, a.v = v, a.ks = ks, a.vs = vs, a.table = s.table_out;
    a.table_stride = keep, a.lengths = nullptr, a.widths = nullptr, a.mask = nullptr, a.out = out, a.lse = lse;
    a.po = (float*)(w + p.po), a.pm = (float*)(w + p.pm), a.pages = pages, a.B = B, a.T = 1, a.H = H, a.G = G, a.dim = dim;
    a.shift = s.shift, a.width = keep, a.groups = p.groups, a.qtype = qtype, a.vec = s.vec, a.scale = scale;
    r.rows = s.row_out, r.T = T, r.splits = p.splits;
    a.pl = a.pm + (p.splits > 1 ? (i64)p.nb * p.nt * H * p.groups * p.splits * 16 : 0);
    hipStream_t st = (hipStream_t)stream;
    for (int b0 = 0; b0 < B; b0 += p.nb)
    for (int t0 = 0; t0 < T; t0 += p.nt) {
        const int nb = B - b0 < p.nb ? B - b0 : p.nb;
        s.b0 = r.b0 = b0, s.t0 = r.t0 = t0, s.nt = r.nt = T - t0 < p.nt ? T - t0 : p.nt;
        s.rows = (i64)nb * s.nt * H;
        int rc;
        // one token a sequence: both at once where the rows fill half the CUs, a block each. At once, and as scores and choice, in
        // us: 128 rows of 313 pages 16.1, 9.1 and 8.2, of 512 18.2, 10.6 and 8.6, of 1024 23.5, 13.9 and 12.1; 96 rows 16.1, 7.0
        // and 7.8, 17.4, 9.5 and 8.4, 23.6, 11.9 and 11.7. (Of few pages the two launches are shorter at 512 rows, too: of 128
        // 17.0, 11.0 and 4.8.)
        if (p.scored && T == 1 && width <= FEW_PAGES && s.rows >= 128) {
            switch (p.dp) {
                case 64: score_choose_k<64, 8><<<(unsigned)s.rows, 512, 0, st>>>(s); break;
                case 128: score_choose_k<128, 16><<<(unsigned)s.rows, 512, 0, st>>>(s); break;
                case 192: score_choose_k<192, 32><<<(unsigned)s.rows, 512, 0, st>>>(s); break;
                default: score_choose_k<256, 32><<<(unsigned)s.rows, 512, 0, st>>>(s);
            }
        } else {
            if (p.scored && (rc = score_rows(s, nb, p.dp, st))) return rc;
            // by the scores that a row can have, the fewest that a lane can hold, in us for 8 and for 5120 rows: 256 scores by
            // 4 a lane 5.3 and 8.1, by 10 6.2 and 10.6; 640 by 10 a lane 7.8 and 13.4, by 16 8.9 and 16.0; 1024 by a wave 10.0
            // and 18.0, by four 11.4 and 47.7. For 8 and 512 rows: 4096 by four waves 12.9 and 15.7, by sixteen 16.5 and 33.3;
            // 16384 by 16 a lane 20.9 and 41.8, by 32 28.4 and 55.8
            if (width <= 256) choose_k<1, 4><<<(unsigned)((s.rows + 3) / 4), 256, 0, st>>>(s);
            else if (width <= 640) choose_k<1, 10><<<(unsigned)((s.rows + 3) / 4), 256, 0, st>>>(s);
            else if (width <= 1024) choose_k<1, 16><<<(unsigned)((s.rows + 3) / 4), 256, 0, st>>>(s);
            else if (width <= 4096) choose_k<4, 16><<<(unsigned)s.rows, 256, 0, st>>>(s);
            else if (width <= 16384) choose_k<16, 16><<<(unsigned)s.rows, 1024, 0, st>>>(s);
            else choose_k<16, 32><<<(unsigned)s.rows, 1024, 0, st>>>(s);
        }
        if ((rc = (int)hipGetLastError())) return rc;
        r.units = s.rows * p.groups;
        switch (codes) {
            case KV_INT8: rc = sparse_codes<KV_INT8>(r, p.dp, st); break;
            case KV_FP8: rc = sparse_codes<KV_FP8>(r, p.dp, st); break;
            case KV_BF16: rc = sparse_codes<KV_BF16>(r, p.dp, st); break;
            default: rc = sparse_codes<KV_F16>(r, p.dp, st);
        }
        if (rc) return rc;
    }
    return 0;
}
