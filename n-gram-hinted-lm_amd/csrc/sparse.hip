// Attention of new tokens over the pages of a cache that a cheap score chooses.
//
//   bounds[page, head]   (min, max) over the page's keys of each element, outward to bfloat16
//   score(token, head, page) = sum over the group's query heads g and elements d of max(q[g, d] lo[d], q[g, d] hi[d])
//                            = sum_d (sum_g max(q[g, d], 0)) hi[d] + (sum_g min(q[g, d], 0)) lo[d]
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
#include "choose.h"
#include "sparse.h"

#define MOST_PAGES 32768  // of a sequence

struct ScoreArgs {
    const void* q;
    i64 qb, qt, qh;
    const b16* bounds;  // [pages, H, 2, DP]
    const int* table;
    i64 table_stride, pages;
    const int *lengths, *widths;
    int B, T, H, G, dim, shift, width, keep, first, last, qtype, vec;
    i64 first_row, rows;  // those of this pass: (sequence, token, head)
    u64* score;           // [rows, width]
    int* table_out;       // [rows, keep]: the kept pages of the cache
    int2* row_out;        // [rows]
    int* chosen;          // [B, T, H, keep] or NULL: the kept pages' places in the sequence, -1 behind them
    int chunks;
};

// A row's token: whether it is in use, the pages it sees, and its keys' number over all of them.
struct Place {
    bool is;
    int b, t, h, pages;
    i64 keys;
};
__device__ __forceinline__ Place place_of(const ScoreArgs& a, i64 row) {
    Place p;
    const i64 at = a.first_row + row, token = at / a.H, cap = (i64)a.width << a.shift;
    p.h = (int)(at - token * a.H), p.b = (int)(token / a.T), p.t = (int)(token - (i64)p.b * a.T);
    const int l = a.lengths[p.b], w = a.widths ? a.widths[p.b] : a.T;
    const i64 len = l < 0 ? 0 : l > cap ? cap : l;
    p.is = p.t < w;
    p.keys = len + p.t + 1 < cap ? len + p.t + 1 : cap;
    p.pages = (int)((p.keys + (1 << a.shift) - 1) >> a.shift);
    return p;
}

// A block per (row, 256 pages); GS lanes a page, each of 8 elements.
template <int DP, int GS> __global__ __launch_bounds__(256) void score_k(const ScoreArgs a) {
    constexpr int U = 4;
    const i64 row = blockIdx.x / a.chunks;
    const int chunk = (int)(blockIdx.x - row * a.chunks);
    const Place p = place_of(a, row);
    const int end = p.pages - a.last, from = chunk * 256 > a.first ? chunk * 256 : a.first;
    const int to = chunk * 256 + 256 < end ? chunk * 256 + 256 : end;
    if (!p.is || p.pages <= a.keep || from >= to) return;
    const int sub = threadIdx.x % GS, group = threadIdx.x / GS, d0 = sub * 8;
    double up[8], down[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) up[j] = down[j] = 0.;
    const u16* q = (const u16*)a.q + p.b * a.qb + p.t * a.qt + (i64)p.h * a.G * a.qh + d0;
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
            const float f = a.qtype == NG_BF16 ? __uint_as_float((u32)x.e[j] << 16) : (float)__builtin_bit_cast(f16, x.e[j]);
            up[j] += f > 0.f || f != f ? (double)f : 0.;
            down[j] += f < 0.f ? (double)f : 0.;
        }
    }
    const int* tab = a.table + p.b * a.table_stride;
    for (int j0 = from + group; j0 < to; j0 += (256 / GS) * U) {
        double acc[U];
        uint4 lo[U], hi[U];
        bool is[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int j = j0 + u * (256 / GS);
            const int e = j < to ? tab[j] : -1;
            is[u] = (u32)e < (u64)a.pages;
            lo[u] = hi[u] = make_uint4(0, 0, 0, 0);
            if (is[u] && d0 < DP) {
                const b16* x = a.bounds + ((i64)e * a.H + p.h) * 2 * DP + d0;
                lo[u] = *(const uint4*)x, hi[u] = *(const uint4*)(x + DP);
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            acc[u] = 0.;
            const u32 l[4] = {lo[u].x, lo[u].y, lo[u].z, lo[u].w}, h[4] = {hi[u].x, hi[u].y, hi[u].z, hi[u].w};
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if (d0 + j >= a.dim) continue;
                const float x = __uint_as_float(j & 1 ? l[j / 2] & 0xFFFF0000u : l[j / 2] << 16);
                const float y = __uint_as_float(j & 1 ? h[j / 2] & 0xFFFF0000u : h[j / 2] << 16);
                acc[u] = fma(down[j], (double)x, fma(up[j], (double)y, acc[u]));
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
#pragma unroll
            for (int o = GS / 2; o; o >>= 1) acc[u] += __shfl_xor(acc[u], o, GS);
            const int j = j0 + u * (256 / GS);
            if (j < to && sub == 0) {
                // a page of none of the cache's ranks last, one whose score is NaN first
                const u64 x = (u64)__double_as_longlong(acc[u] + 0.);
                a.score[row * a.width + j] = !is[u] ? 1ull : acc[u] != acc[u] ? ~1ull : x >> 63 ? ~x : x | 1ull << 63;
            }
        }
    }
}

// The kept pages of a row, by NW waves that hold E of its scores a lane (NW = 1: four rows a block).
template <int NW, int E> __global__ __launch_bounds__(NW == 1 ? 256 : NW * 64) void choose_k(const ScoreArgs a) {
    constexpr int NT = NW * 64;
    __shared__ int counts[2][NW], before[NW == 1 ? 1 : E * NW];
    __shared__ u64 ends[2][NW];
    const i64 row = NW == 1 ? (i64)blockIdx.x * 4 + (threadIdx.x >> 6) : (i64)blockIdx.x;
    if (row >= a.rows) return;
    const int tid = NW == 1 ? lane_id() : (int)threadIdx.x, wave = NW == 1 ? 0 : tid >> 6;
    const Place p = place_of(a, row);
    const int* tab = a.table + p.b * a.table_stride;
    int* out = a.table_out + row * a.keep;
    int* chosen = a.chosen ? a.chosen + (a.first_row + row) * a.keep : nullptr;
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
    u64 key[E], lo = ~0ull, hi = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int j = e * NT + tid;
        key[e] = 0;
        if (j < n) key[e] = j < a.first || j >= n - a.last ? ~0ull : a.score[row * a.width + j];
        if (j < n) lo = key[e] < lo ? key[e] : lo;
        if (key[e] != ~0ull) hi = key[e] > hi ? key[e] : hi;
    }
    lo = min_wave(lo), hi = max_wave(hi);
    if constexpr (NW > 1) {
        if (lane_id() == 0) ends[0][wave] = lo, ends[1][wave] = hi;
        lds_barrier();
#pragma unroll
        for (int w = 0; w < NW; ++w) lo = ends[0][w] < lo ? ends[0][w] : lo, hi = ends[1][w] > hi ? ends[1][w] : hi;
    }
    Count<NW> count(counts);
    int c = n;
    const int forced = a.first + a.last;
    const u64 t = forced == a.keep ? ~0ull : count.threshold(key, lo, hi, a.keep, a.keep, c);
    int equal = E * NT;  // of the scores equal to t, the first so many
    if (forced < a.keep && c > a.keep) equal = a.keep - count.at_least(key, t + 1);
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
    for (int e = 0; e < E; ++e) take |= (key[e] > t || (forced == a.keep && key[e] == t) ? 1u : 0u) << e;
    if (forced < a.keep) place([&](int e) { return key[e] == t; }, [&](int e, int i) { take |= (i < equal ? 1u : 0u) << e; });
    place([&](int e) { return (take >> e & 1) != 0; }, [&](int e, int i) {
        const int j = e * NT + tid;
        out[i] = tab[j];
        if (chosen) chosen[i] = j;
    });
}

// ------------------------------------------------------------------------------------------------------------ the host

#define SLAB ((i64)256 << 20)  // bytes of scores at a time
#define AIM 512                // blocks that fill the card: 2 a CU

struct SparsePlan {
    int dp, groups, splits;
    bool scored;
    i64 tokens;  // at a time
    i64 score, table, rows, po, pm, bytes;  // offsets in the workspace
};

static bool sparse_plan(i64 B, i64 T, i64 H, i64 G, i64 dim, i64 width, i64 page, i64 keep, SparsePlan& p) {
    const i64 lim = (i64)1 << 30;
    if (B < 0 || T < 1 || H < 1 || G < 1 || dim < 1 || dim > 256 || width < 1 || width > MOST_PAGES || keep < 1 || keep > 1024 ||
        B > lim || T > lim || H > lim || G > 1 << 20 || page < 16 || page > 4096 || (page & (page - 1)) ||
        width * page > lim || B * T > lim || H * ((G + 15) / 16) > 1 << 20)
        return false;
    p.dp = (int)(dim + 63) / 64 * 64, p.groups = (int)(G + 15) / 16, p.scored = width > keep;
    const i64 tokens = B * T;
    // a pass takes as many tokens as SLAB holds the scores of, and fewer than 2^24 units
    p.tokens = tokens;
    const i64 each = H * width * 8, most_units = ((i64)1 << 24) / (H * p.groups);
    if (p.scored && p.tokens * each > SLAB) p.tokens = SLAB / each ? SLAB / each : 1;
    if (p.tokens > most_units) p.tokens = most_units ? most_units : 1;
    const i64 rows = p.tokens * H, units = rows * p.groups;
    const i64 tiles = ((keep < width ? keep : width) * page + TILE - 1) / TILE;
    i64 splits = units ? (AIM + units - 1) / units : 1;
    p.splits = (int)(splits < tiles ? splits : tiles);
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

static int score_rows(const ScoreArgs& a, int dp, hipStream_t st) {
    const i64 n = a.rows * a.chunks;
    if (n >= (i64)1 << 31) return -1;
    switch (dp) {
        case 64: score_k<64, 8><<<(unsigned)n, 256, 0, st>>>(a); break;
        case 128: score_k<128, 16><<<(unsigned)n, 256, 0, st>>>(a); break;
        case 192: score_k<192, 32><<<(unsigned)n, 256, 0, st>>>(a); break;
        default: score_k<256, 32><<<(unsigned)n, 256, 0, st>>>(a);
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
    s.chunks = (width + 255) / 256;
    SparseArgs r;
    TreeArgs& a = r.a;
    a.q = q, a.qb = qb, a.qt = qt, a.qh = qh, a.k = k, a.v = v, a.ks = ks, a.vs = vs, a.table = s.table_out;
    a.table_stride = keep, a.lengths = nullptr, a.widths = nullptr, a.mask = nullptr, a.out = out, a.lse = lse;
    a.po = (float*)(w + p.po), a.pm = (float*)(w + p.pm), a.pages = pages, a.B = B, a.T = 1, a.H = H, a.G = G, a.dim = dim;
    a.shift = s.shift, a.width = keep, a.groups = p.groups, a.qtype = qtype, a.vec = s.vec, a.scale = scale;
    r.rows = s.row_out, r.T = T, r.splits = p.splits;
    a.pl = a.pm + (p.splits > 1 ? p.tokens * H * p.groups * p.splits * 16 : 0);
    hipStream_t st = (hipStream_t)stream;
    const i64 tokens = (i64)B * T;
    for (i64 t0 = 0; t0 < tokens; t0 += p.tokens) {
        const i64 n = tokens - t0 < p.tokens ? tokens - t0 : p.tokens;
        s.first_row = t0 * H, s.rows = n * H;
        int rc;
        if (p.scored && (rc = score_rows(s, p.dp, st))) return rc;
        // by the scores that a row can have: 1024 are a wave's, 4096 four waves'
        if (width <= 1024) choose_k<1, 16><<<(unsigned)((s.rows + 3) / 4), 256, 0, st>>>(s);
        else if (width <= 4096) choose_k<4, 16><<<(unsigned)s.rows, 256, 0, st>>>(s);
        else choose_k<16, 32><<<(unsigned)s.rows, 1024, 0, st>>>(s);
        if ((rc = (int)hipGetLastError())) return rc;
        r.first_row = s.first_row, r.units = s.rows * p.groups;
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
