// Hint rows embedded, and the table's gradient.
//
//   out[n] = scale * sum_j w[n, j] * table[tok[n, j]]     over the entries j = (slot, candidate) of position n that count:
//            w[n, j] != 0 and cell[n, slot] > 0; without weights one entry of weight 1
//   grad[v] = scale * sum over the counted entries of token v of w[n, j] * dout[n]
//   dw[n, j] = scale * <table[tok[n, j]], dout[n]> where the slot has a cell, else 0; also where w[n, j] = 0: the slope at 0
//
// An entry that does not count is not read by the output and the table's gradient (its table row may hold anything); the
// weights' gradient reads the row of an entry of weight 0 that has a cell, and is 0 where its token is outside the table. A
// counted token outside the table is never read: its position's output is NaN, its dw NaN, and it adds to no gradient. Sums
// are held in 32 bits, in a fixed order, and rounded once.
#include "vals.h"
#include <type_traits>

struct Rows {
    const void* tokens;  // int64, int32 or uint16 (tsize 8, 4, 2), [n, m]
    const float* w;      // [n, m] or NULL
    const void* cell;    // [n, m / entries], int64, int32 or int16 (csize 8, 4, 2), or NULL
    i64 n;
    int m, entries, tsize, csize;
    i64 V;
};

__device__ __forceinline__ i64 int_at(const void* p, int size, i64 i) {
    return size == 8 ? ((const i64*)p)[i] : size == 4 ? ((const int*)p)[i] : (i64)((const u16*)p)[i];
}

__device__ __forceinline__ bool has_cell(const Rows& r, i64 i) {
    if (!r.cell) return true;
    const i64 c = i / r.entries;
    return (r.csize == 2 ? (i64)((const short*)r.cell)[c] : int_at(r.cell, r.csize, c)) > 0;
}

// the counted weight of entry i (0: it does not count)
__device__ __forceinline__ float weight_of(const Rows& r, i64 i) {
    if (!r.w) return has_cell(r, i) ? 1.f : 0.f;
    const float w = r.w[i];
    return w != 0.f && has_cell(r, i) ? w : 0.f;
}

template <typename T, int VEC> struct Acc {
    float v[VEC];
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[j] = 0.f;
    }
    __device__ __forceinline__ void add(const Pack<T, VEC>& p, float w) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[j] = fmaf(w, (float)p.v[j], v[j]);
    }
    __device__ __forceinline__ void store(T* o, float scale) const {
        Pack<T, VEC> p;
#pragma unroll
        for (int j = 0; j < VEC; ++j) p.v[j] = (T)(v[j] * scale);
        p.store(o);
    }
};

// The columns of a lane, [at, at + VEC) of the row: where the row ends inside them, or before, the row's last VEC columns
// (dim >= VEC). So every load is a whole one: a row's last lane may compute columns of the lane before it once more, to the
// same values, and a lane with nothing to do (in false) only stores nothing.
template <int VEC> struct Cols {
    int at, again;  // again: the first `again` of its columns are another lane's
    bool in;
    __device__ __forceinline__ Cols(int lane, int dim) {
        const int col = lane * VEC;
        in = col < dim, at = col < dim - VEC ? col : dim - VEC, again = in ? col - at : VEC;
    }
};

__device__ __forceinline__ float lane_f(float x, int l) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), l)); }
__device__ __forceinline__ int lane_i(int x, int l) { return __builtin_amdgcn_readlane(x, l); }

// The rows that the lanes of `live` name (`row` of a lane, weighted `w`), added up in order at this lane's column: U rows'
// loads in flight together.
template <typename T, int VEC, int U>
__device__ __forceinline__ void sum_rows(const T* __restrict__ base, i64 ld, int col, u64 live, int row, float w,
                                         Acc<T, VEC>& acc) {
    while (live) {
        int at[U];
        Pack<T, VEC> p[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            at[u] = live ? __builtin_ctzll(live) : -1;
            live &= live - 1;
            if (at[u] >= 0) p[u].load(base + (i64)(u32)lane_i(row, at[u]) * ld + col);
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (at[u] >= 0) acc.add(p[u], lane_f(w, at[u]));
    }
}

// A wave per (position, chunk of 64 * VEC columns). Its lanes hold a position's entries while it adds their rows, so an entry
// is read once, and four rows' loads are in flight. Memory bounds it: 65536 positions of 8 entries (2.25 counted) at 768
// columns in bfloat16 64 us, 5.3 TB/s of rows and entries read and rows written; 16 positions 3.8 us, a launch.
template <typename T, int VEC>
__global__ __launch_bounds__(256) void embed_rows_k(const Rows r, const T* __restrict__ table, i64 ld, int dim, float scale,
                                                    T* __restrict__ out, int chunks) {
    const i64 items = r.n * chunks, step = (i64)gridDim.x * 4;
    for (i64 it = (i64)blockIdx.x * 4 + (threadIdx.x >> 6); it < items; it += step) {
        const i64 n = it / chunks;
        const Cols<VEC> col((int)(it - n * chunks) * 64 + lane_id(), dim);
        Acc<T, VEC> acc;
        acc.zero();
        bool bad = false;
        for (int base = 0; base < r.m; base += 64) {
            const int j = base + lane_id();
            float w = 0.f;
            i64 tok = 0;
            if (j < r.m) {
                w = weight_of(r, n * r.m + j);
                if (w != 0.f) tok = int_at(r.tokens, r.tsize, n * r.m + j);
            }
            const bool out_of = (u64)tok >= (u64)r.V;
            bad |= __ballot(out_of && w != 0.f) != 0;
            sum_rows<T, VEC, 4>(table, ld, col.at, __ballot(w != 0.f && !out_of), (int)tok, w, acc);
        }
        if (bad)
#pragma unroll
            for (int j = 0; j < VEC; ++j) acc.v[j] = __builtin_nanf("");
        if (col.in) acc.store(out + n * dim + col.at, scale);
    }
}

// Without weights: a thread per VEC columns of a position, four of them in flight. Memory: 131072 tokens at 1024 columns in
// bfloat16 78 us, 6.9 TB/s read and written (frequent tokens' rows come from the caches).
template <typename T, int VEC>
__global__ __launch_bounds__(256) void embed_tokens_k(const Rows r, const T* __restrict__ table, i64 ld, int dim,
                                                      float scale, T* __restrict__ out, int per) {
    const i64 items = r.n * per, step = (i64)gridDim.x * 256;
    for (i64 i0 = (i64)blockIdx.x * 256 + threadIdx.x; i0 < items; i0 += 4 * step) {
        Pack<T, VEC> p[4];
        bool ok[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const i64 i = i0 + u * step;
            ok[u] = false;
            if (i < items) {
                const i64 n = i / per;
                const i64 tok = int_at(r.tokens, r.tsize, n);
                ok[u] = (u64)tok < (u64)r.V;
                if (ok[u]) p[u].load(table + tok * ld + Cols<VEC>((int)(i - n * per), dim).at);
            }
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const i64 i = i0 + u * step;
            if (i < items) {
                const i64 n = i / per;
                Acc<T, VEC> acc;
                acc.zero();
                if (ok[u]) acc.add(p[u], 1.f);
                else
#pragma unroll
                    for (int j = 0; j < VEC; ++j) acc.v[j] = __builtin_nanf("");
                acc.store(out + n * dim + Cols<VEC>((int)(i - n * per), dim).at, scale);
            }
        }
    }
}

// ------------------------------------------------------------------------------------------------ the table's gradient
//
// The counted entries are sorted by token, stably, by digits of 8 bits, the first pass leaving out the others: an entry is
// one 64-bit word, token << 32 | index. A pass is three launches over `tiles` spans of the list: the spans' digit counts,
// their sums, and the words put in their places. A list of at most ONE entries is sorted by one block in one launch.
// Launches and the entries' scattered words bound it: 524288 entries of which 147456 count, two passes, 39 us (first pass
// 7.8 + 3.4 + 10.9, second 4.6 + 3.4 + 6.3, starts 2.9). The workspace is sized by all entries, since the host does not
// know how many count: 16 bytes an entry and two float rows per 64 of them.

#define ONE 8192

struct Source {  // what a pass reads: the entries themselves (list NULL), or the list of the pass before, count words long
    Rows r;
    const u64* list;
    const u32* count;
};

template <bool FIRST> __device__ __forceinline__ u32 source_size(const Source& s) {
    return FIRST ? (u32)(s.r.n * s.r.m) : *s.count;
}

template <bool FIRST> __device__ __forceinline__ bool word_at(const Source& s, u32 i, u64& w) {
    if (!FIRST) {
        w = s.list[i];
        return true;
    }
    if (weight_of(s.r, i) == 0.f) return false;
    const i64 t = int_at(s.r.tokens, s.r.tsize, i);
    w = (u64)t << 32 | i;
    return (u64)t < (u64)s.r.V;
}

// the wave's part of tile b: whole rounds of 64 words
__device__ __forceinline__ void part_of(u32 n, u32 tile, int b, int waves, int wave, u32& lo, u32& hi) {
    const u64 a = (u64)b * tile + (u64)(tile / waves) * wave, z = a + tile / waves;
    lo = a < n ? (u32)a : n, hi = z < n ? (u32)z : n;
}

template <bool FIRST>
__global__ __launch_bounds__(256) void embed_count_k(const Source s, u32 tile, int shift, int tiles, u32* __restrict__ hist) {
    __shared__ u32 cnt[256];
    cnt[threadIdx.x] = 0;
    __syncthreads();
    const u32 n = source_size<FIRST>(s);
    const u64 a = (u64)blockIdx.x * tile, z = a + tile < n ? a + tile : n;
    for (u64 i = a + threadIdx.x; i < z; i += 256) {
        u64 w;
        if (word_at<FIRST>(s, (u32)i, w)) atomicAdd(&cnt[(w >> 32 >> shift) & 255], 1u);
    }
    __syncthreads();
    hist[(i64)threadIdx.x * tiles + blockIdx.x] = cnt[threadIdx.x];
}

// a block a digit: its counts become the sums before each tile, total[digit] their sum
__global__ __launch_bounds__(256) void embed_sums_k(u32* __restrict__ hist, int tiles, u32* __restrict__ total) {
    __shared__ u32 part[4];
    u32* h = hist + (i64)blockIdx.x * tiles;
    u32 run = 0;
    for (int t0 = 0; t0 < tiles; t0 += 256) {
        const int t = t0 + threadIdx.x;
        const u32 x = t < tiles ? h[t] : 0;
        u32 inc = x;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const u32 up = (u32)__shfl_up((int)inc, o, 64);
            if (lane_id() >= o) inc += up;
        }
        __syncthreads();
        if (lane_id() == 63) part[threadIdx.x >> 6] = inc;
        __syncthreads();
        u32 before = run;
        for (int w = 0; w < (int)(threadIdx.x >> 6); ++w) before += part[w];
        if (t < tiles) h[t] = before + inc - x;
        run += part[0] + part[1] + part[2] + part[3];
    }
    if (threadIdx.x == 0) total[blockIdx.x] = run;
}

// the 256 digits' starts from their totals (every thread below 256 of the block: its digit's), and their sum
__device__ __forceinline__ u32 digit_start(u32 mine, u32* lds, u32& sum) {
    u32 inc = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const u32 up = (u32)__shfl_up((int)inc, o, 64);
        if (lane_id() >= o) inc += up;
    }
    if (threadIdx.x < 256 && lane_id() == 63) lds[threadIdx.x >> 6] = inc;
    __syncthreads();
    u32 before = 0;
    for (int w = 0; w < 4; ++w) before += w < (int)(threadIdx.x >> 6) ? lds[w] : 0;
    sum = lds[0] + lds[1] + lds[2] + lds[3];
    return before + inc - mine;
}

// a wave's words [lo, hi) to their places: next[digit] the place of its next word of that digit
template <bool FIRST>
__device__ __forceinline__ void place_words(const Source& s, u32 lo, u32 hi, int shift, u32* next, u64* __restrict__ out) {
    for (u32 i0 = lo; i0 < hi; i0 += 64) {
        const u32 i = i0 + lane_id();
        u64 w = 0;
        const bool ok = i < hi && word_at<FIRST>(s, i, w);
        const u32 d = (u32)(w >> 32 >> shift) & 255;
        u64 same = __ballot(ok);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const u64 one = __ballot(d >> k & 1);
            same &= d >> k & 1 ? one : ~one;
        }
        const u32 at = ok ? next[d] : 0;
        __builtin_amdgcn_wave_barrier();
        if (ok && (same & lanemask_lt()) == 0) next[d] = at + (u32)__popcll(same);  // the first lane of each digit
        __builtin_amdgcn_wave_barrier();
        if (ok) out[at + (u32)__popcll(same & lanemask_lt())] = w;
    }
}

template <bool FIRST>
__device__ __forceinline__ void count_words(const Source& s, u32 lo, u32 hi, int shift, u32* cnt) {
    for (u32 i = lo + lane_id(); i < hi; i += 64) {
        u64 w;
        if (word_at<FIRST>(s, i, w)) atomicAdd(&cnt[(w >> 32 >> shift) & 255], 1u);
    }
}

template <bool FIRST>
__global__ __launch_bounds__(256) void embed_place_k(const Source s, u32 tile, int shift, int tiles,
                                                     const u32* __restrict__ hist, const u32* __restrict__ total,
                                                     u64* __restrict__ out, u32* __restrict__ count) {
    __shared__ u32 next[4][256];
    __shared__ u32 part[4];
    const int wave = threadIdx.x >> 6, d = threadIdx.x;
#pragma unroll
    for (int w = 0; w < 4; ++w) next[w][d] = 0;
    u32 sum;
    u32 at = digit_start(total[d], part, sum) + hist[(i64)d * tiles + blockIdx.x];
    if (FIRST && blockIdx.x == 0 && d == 0) *count = sum;
    __syncthreads();
    u32 lo, hi;
    part_of(source_size<FIRST>(s), tile, blockIdx.x, 4, wave, lo, hi);
    count_words<FIRST>(s, lo, hi, shift, next[wave]);
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        const u32 c = next[w][d];
        next[w][d] = at;
        at += c;
    }
    __syncthreads();
    place_words<FIRST>(s, lo, hi, shift, next[wave], out);
}

// The whole sort of at most ONE entries by one block, the lists in LDS; the last pass writes out.
__global__ __launch_bounds__(1024) void embed_sort_one_k(const Source src, int passes, u64* __restrict__ out,
                                                         u32* __restrict__ count) {
    __shared__ u64 list[ONE];
    __shared__ u32 next[16][256];
    __shared__ u32 part[4];
    __shared__ u32 size;
    const int wave = threadIdx.x >> 6, d = threadIdx.x & 255;
    Source s = src;
    for (int p = 0; p < passes; ++p) {
        for (int i = threadIdx.x; i < 16 * 256; i += 1024) next[i >> 8][i & 255] = 0;
        __syncthreads();
        const u32 n = p ? size : (u32)(s.r.n * s.r.m);
        const u32 tile = (n + 1023) / 1024 * 1024;
        u32 lo, hi;
        part_of(n, tile, 0, 16, wave, lo, hi);
        u64 keep[ONE / 1024];  // the wave's words: they are written over the list they come from
#pragma unroll
        for (int k = 0; k < ONE / 1024; ++k) {
            const u32 i = lo + k * 64 + lane_id();
            keep[k] = ~0ull;
            if (i < hi) {
                if (p) keep[k] = list[i];
                else if (u64 w; word_at<true>(s, i, w)) keep[k] = w;
            }
            if (keep[k] != ~0ull) atomicAdd(&next[wave][(keep[k] >> 32 >> (8 * p)) & 255], 1u);
        }
        __syncthreads();
        u32 mine = 0;
        if (threadIdx.x < 256)
            for (int w = 0; w < 16; ++w) mine += next[w][d];
        u32 sum, at = digit_start(mine, part, sum);
        if (threadIdx.x < 256)
            for (int w = 0; w < 16; ++w) {
                const u32 c = next[w][d];
                next[w][d] = at;
                at += c;
            }
        if (p == 0 && threadIdx.x == 0) size = sum, *count = sum;
        __syncthreads();
        u64* to = p == passes - 1 ? out : list;
#pragma unroll
        for (int k = 0; k < ONE / 1024; ++k) {
            const u64 w = keep[k];
            const bool ok = w != ~0ull;
            const u32 b = (u32)(w >> 32 >> (8 * p)) & 255;
            u64 same = __ballot(ok);
#pragma unroll
            for (int q = 0; q < 8; ++q) {
                const u64 one = __ballot(b >> q & 1);
                same &= b >> q & 1 ? one : ~one;
            }
            const u32 to_at = ok ? next[wave][b] : 0;
            __builtin_amdgcn_wave_barrier();
            if (ok && (same & lanemask_lt()) == 0) next[wave][b] = to_at + (u32)__popcll(same);
            __builtin_amdgcn_wave_barrier();
            if (ok) to[to_at + (u32)__popcll(same & lanemask_lt())] = w;
        }
        __syncthreads();
    }
}

// start[v] = the first sorted word whose token is >= v, v in [0, V]. Many words: each opens its token and the absent ones
// before it (a gap of many tokens is filled by the whole wave).
__global__ __launch_bounds__(256) void embed_starts_k(const u64* __restrict__ list, const u32* __restrict__ count, i64 V,
                                                      u32* __restrict__ start) {
    const i64 M = *count;
    for (i64 w0 = (i64)blockIdx.x * 256 + (threadIdx.x & ~63); w0 <= M; w0 += (i64)gridDim.x * 256) {
        const i64 i = w0 + lane_id();
        i64 lo = 0, hi = 0;  // this word opens the tokens [lo, hi)
        if (i <= M) {
            lo = i ? (i64)(list[i - 1] >> 32) + 1 : 0;
            hi = (i < M ? (i64)(list[i] >> 32) : V) + 1;
        }
        u64 wide = __ballot(hi - lo > 16);
        if (hi - lo <= 16)
            for (i64 v = lo; v < hi; ++v) start[v] = (u32)i;
        while (wide) {
            const int l = __builtin_ctzll(wide);
            const i64 a = (i64)bcast_u64((u64)lo, l), b = (i64)bcast_u64((u64)hi, l);
            for (i64 v = a + lane_id(); v < b; v += 64) start[v] = (u32)(w0 + l);
            wide &= wide - 1;
        }
    }
}

// Few words (at most ONE): every token looks for its own, in LDS.
__global__ __launch_bounds__(256) void embed_starts_one_k(const u64* __restrict__ list, const u32* __restrict__ count, i64 V,
                                                          u32* __restrict__ start) {
    __shared__ u32 tok[ONE];
    const u32 M = *count;
    for (u32 i = threadIdx.x; i < M; i += 256) tok[i] = (u32)(list[i] >> 32);
    __syncthreads();
    for (i64 v = (i64)blockIdx.x * 256 + threadIdx.x; v <= V; v += (i64)gridDim.x * 256) {
        u32 lo = 0, hi = M;
        while (lo < hi) {
            const u32 mid = (lo + hi) / 2;
            if ((i64)tok[mid] < v) lo = mid + 1;
            else hi = mid;
        }
        start[v] = lo;
    }
}

// The sums. The sorted list is cut into chunks of 64 entries, a wave per chunk (and chunk of columns), whatever the tokens:
// the work is even, and 8 rows' loads are in flight together whichever token they belong to. A token whose entries all lie
// in one chunk has its gradient row stored there; one that crosses a chunk's end leaves a partial sum in each chunk that it
// touches, slot 2 * chunk where it holds the chunk's first entry, else slot 2 * chunk + 1 (it then holds the last one), and
// they are joined in a fixed order. Rows without entries are zeroed by a pass of their own. Waiting for rows bounds the sums
// (their waves wait 90 % of the time; no more than 8 rows are asked for before they are added): 147456 entries at 768
// columns in bfloat16 57 us (4.0 TB/s), 131072 at 1024 103 us (2.6).
#define CHUNK 64

template <typename T, int VEC>
__global__ __launch_bounds__(256) void embed_runs_k(const u64* __restrict__ list, const u32* __restrict__ count,
                                                    const float* __restrict__ w, int m, const T* __restrict__ dout, i64 ld,
                                                    int dim, int chunks, float scale, i64 spans, float* __restrict__ part,
                                                    T* __restrict__ grad) {
    constexpr int U = 8;
    const u32 M = *count;
    const i64 items = spans * chunks;
    for (i64 it = (i64)blockIdx.x * 4 + (threadIdx.x >> 6); it < items; it += (i64)gridDim.x * 4) {
        const i64 c = it / chunks;
        const u32 c0 = (u32)(c * CHUNK);
        if (c0 >= M) return;
        const int last = M - c0 < CHUNK ? (int)(M - c0) - 1 : CHUNK - 1;
        const Cols<VEC> col((int)(it - c * chunks) * 64 + lane_id(), dim);
        const u32 i = c0 + (lane_id() < last ? lane_id() : last);
        const u64 word = list[i];
        const u32 tok = (u32)(word >> 32), before = i ? (u32)(list[i - 1] >> 32) : ~0u, after = i + 1 < M ? (u32)(list[i + 1] >> 32) : ~0u;
        const int n = (int)((u32)word / (u32)m);
        const float x = w ? w[(u32)word] : 1.f;
        const u64 ends = __ballot(after != tok) | 1ull << last;
        const bool from = lane_i((int)before, 0) == lane_i((int)tok, 0), on = lane_i((int)after, last) == lane_i((int)tok, last);
        bool first = true;
        Acc<T, VEC> acc;
        acc.zero();
        for (int l0 = 0; l0 <= last; l0 += U) {
            Pack<T, VEC> r[U];
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (l0 + u <= last) r[u].load(dout + (i64)(u32)lane_i(n, l0 + u) * ld + col.at);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int l = l0 + u;
                if (l > last) break;
                acc.add(r[u], lane_f(x, l));
                if (ends >> l & 1) {
                    if ((first && from) || (l == last && on)) {
                        Pack<float, VEC> o;
#pragma unroll
                        for (int j = 0; j < VEC; ++j) o.v[j] = acc.v[j];
                        if (col.in) o.store(part + (2 * c + (first ? 0 : 1)) * dim + col.at);
                    } else if (col.in) acc.store(grad + (i64)(u32)lane_i((int)tok, l) * dim + col.at, scale);
                    acc.zero();
                    first = false;
                }
            }
        }
    }
}

// A block per (chunk, chunk of columns) in which a token begins that goes on in the next: its partial sums joined, each of
// the eight waves in order, then the waves' sums. 16 us beside the 57 above, 14 beside the 103.
template <typename T, int VEC>
__global__ __launch_bounds__(512) void embed_join_k(const u64* __restrict__ list, const u32* __restrict__ count,
                                                    const u32* __restrict__ start, int dim, int chunks, i64 spans, float scale,
                                                    const float* __restrict__ part, T* __restrict__ grad) {
    constexpr int U = 8;
    __shared__ float sums[8][64 * VEC];
    const u32 M = *count;
    const i64 items = spans * chunks;
    const int wave = threadIdx.x >> 6;
    for (i64 it = blockIdx.x; it < items; it += gridDim.x) {
        const i64 c = it / chunks;
        const u32 c0 = (u32)(c * CHUNK);
        if (c0 >= M) return;
        const u32 c1 = M - c0 < CHUNK ? M : c0 + CHUNK;
        const u32 t = (u32)(list[c1 - 1] >> 32), s = start[t], e = start[t + 1];
        if (e <= c1 || s < c0) continue;
        const Cols<VEC> col((int)(it - c * chunks) * 64 + lane_id(), dim);
        const i64 end = (e - 1) / CHUNK;
        float acc[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) acc[j] = 0.f;
        for (i64 k = c + wave; k <= end; k += 8 * U) {
            Pack<float, VEC> x[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const i64 q = k + 8 * u;
                if (q <= end) x[u].load(part + (2 * q + (q == c && s != c0 ? 1 : 0)) * dim + col.at);
            }
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (k + 8 * u <= end)
#pragma unroll
                    for (int j = 0; j < VEC; ++j) acc[j] += x[u].v[j];
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < VEC; ++j) sums[wave][j * 64 + lane_id()] = acc[j];
        __syncthreads();
        if (wave == 0 && col.in) {
            Acc<T, VEC> r;
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                r.v[j] = sums[0][j * 64 + lane_id()];
#pragma unroll
                for (int k = 1; k < 8; ++k) r.v[j] += sums[k][j * 64 + lane_id()];
            }
            r.store(grad + t * (i64)dim + col.at, scale);
        }
    }
}

// A thread per VEC columns of a row: rows without entries are zeros. 13 us for 50257 rows of 768 in bfloat16.
template <typename T, int VEC>
__global__ __launch_bounds__(256) void embed_zero_k(const u32* __restrict__ start, i64 V, int dim, int per, T* __restrict__ grad) {
    const i64 items = V * per;
    for (i64 i = (i64)blockIdx.x * 256 + threadIdx.x; i < items; i += (i64)gridDim.x * 256) {
        const i64 v = i / per;
        if (start[v] != start[v + 1]) continue;
        Pack<T, VEC> z;
#pragma unroll
        for (int j = 0; j < VEC; ++j) z.v[j] = (T)0.f;
        z.store(grad + v * dim + Cols<VEC>((int)(i - v * per), dim).at);
    }
}

// A wave per position: the slopes of its weights, 8 entries at a time. 20011 positions of 16 entries at 333 columns in
// float32: 32 us, bound by the dots' reductions over the lanes (six shuffles each) beside the rows' loads.
template <typename T, int VEC>
__global__ __launch_bounds__(256) void embed_dw_k(const Rows r, const T* __restrict__ table, i64 ld, const T* __restrict__ dout,
                                                  i64 dld, int dim, float scale, float* __restrict__ dw) {
    for (i64 n = (i64)blockIdx.x * 4 + (threadIdx.x >> 6); n < r.n; n += (i64)gridDim.x * 4) {
        for (int base = 0; base < r.m; base += 64) {
            const int j = base + lane_id();
            i64 tok = -1;
            bool has = false, counts = false;
            if (j < r.m) {
                has = has_cell(r, n * r.m + j);
                if (has) tok = int_at(r.tokens, r.tsize, n * r.m + j), counts = !r.w || r.w[n * r.m + j] != 0.f;
            }
            const bool ok = has && (u64)tok < (u64)r.V;
            float mine = counts && !ok ? __builtin_nanf("") : 0.f;
            u64 live = __ballot(ok);
            while (live) {
                int at[8];
                float dot[8];
#pragma unroll
                for (int u = 0; u < 8; ++u) {
                    at[u] = live ? __builtin_ctzll(live) : -1;
                    live &= live - 1;
                    dot[u] = 0.f;
                }
                for (int k = 0; k * 64 * VEC < dim; ++k) {
                    const Cols<VEC> col(k * 64 + lane_id(), dim);
                    Pack<T, VEC> d, p[8];
                    d.load(dout + n * dld + col.at);
#pragma unroll
                    for (int u = 0; u < 8; ++u)
                        if (at[u] >= 0) p[u].load(table + (i64)(u32)lane_i((int)tok, at[u]) * ld + col.at);
                    float f[VEC];
#pragma unroll
                    for (int j = 0; j < VEC; ++j) f[j] = j < col.again ? 0.f : (float)d.v[j];
#pragma unroll
                    for (int u = 0; u < 8; ++u)
                        if (at[u] >= 0)
#pragma unroll
                            for (int j = 0; j < VEC; ++j) dot[u] = j < col.again ? dot[u] : fmaf(f[j], (float)p[u].v[j], dot[u]);
                }
#pragma unroll
                for (int u = 0; u < 8; ++u) {
                    if (at[u] < 0) break;
#pragma unroll
                    for (int o = 32; o; o >>= 1) dot[u] += __shfl_xor(dot[u], o, 64);
                    if (lane_id() == at[u]) mine = dot[u] * scale;
                }
            }
            if (j < r.m) dw[n * r.m + j] = mine;
        }
    }
}

// ------------------------------------------------------------------------------------------------------------ the host

static bool rows_ok(const Rows& r, int dim) {
    return r.n >= 0 && r.m >= 1 && r.entries >= 1 && r.m % r.entries == 0 && r.V >= 1 && r.V < (i64)1 << 31 && dim >= 1 &&
           r.n <= (((i64)1 << 31) - 64) / r.m && (r.tsize == 8 || r.tsize == 4 || r.tsize == 2) &&
           (!r.cell || r.csize == 8 || r.csize == 4 || r.csize == 2);
}

static inline int wave_grid(i64 waves) {
    const i64 g = (waves + 3) / 4;
    return (int)(g < 65536 ? (g > 0 ? g : 1) : 65536);
}

// The elements a lane takes of a row: 16 bytes of them, or fewer where a short row would leave over half of a wave's lanes
// without work.
template <typename T> static int vec_of(int dim, int lanes = 32) {
    int v = 16 / (int)sizeof(T);
    while (v > 1 && ((dim + v - 1) / v <= lanes || dim < v)) v >>= 1;
    return v;
}

template <typename T, typename F> static int with_vec(int v, F f) {
    if constexpr (sizeof(T) == 2) {
        if (v == 8) return f(std::integral_constant<int, 8>{});
    }
    if (v == 4) return f(std::integral_constant<int, 4>{});
    if (v == 2) return f(std::integral_constant<int, 2>{});
    return f(std::integral_constant<int, 1>{});
}

template <typename T>
static int embed_fwd(const Rows& r, const T* table, i64 ld, int dim, float scale, T* out, hipStream_t st) {
    const bool plain = !r.w && !r.cell && r.m == 1;
    return with_vec<T>(vec_of<T>(dim, plain ? 0 : 32), [&](auto c) {
        constexpr int VEC = decltype(c)::value;
        if (plain) {
            const int per = (dim + VEC - 1) / VEC;
            const i64 g = (r.n * per + 1023) / 1024;
            embed_tokens_k<T, VEC><<<(int)(g < 65536 ? g : 65536), 256, 0, st>>>(r, table, ld, dim, scale, out, per);
        } else {
            const int chunks = (dim + 64 * VEC - 1) / (64 * VEC);
            embed_rows_k<T, VEC><<<wave_grid(r.n * chunks), 256, 0, st>>>(r, table, ld, dim, scale, out, chunks);
        }
        return (int)hipGetLastError();
    });
}

struct GradWork {
    u64 *la, *lb;
    u32 *hist, *total, *count, *start;
    float* part;
    u32 tile;   // entries of a span, a multiple of 256
    int tiles;  // at most 2048 of them
    i64 bytes;
    GradWork(void* base, i64 M, i64 V, int dim) {
        char* p = (char*)base;
        const auto take = [&](i64 n) {
            char* q = p;
            p += (n + 255) / 256 * 256;
            return (void*)q;
        };
        // spans of 1024 entries or more: 524288 entries fill the 256 compute units twice
        const i64 t = (M + 2047) / 2048;
        tile = (u32)((t < 1024 ? 1024 : t) + 255) / 256 * 256;
        tiles = M > ONE ? (int)((M + tile - 1) / tile) : 0;
        la = (u64*)take(8 * M), lb = (u64*)take(M > ONE ? 8 * M : 0);
        hist = (u32*)take(1024ll * tiles), total = (u32*)take(1024), count = (u32*)take(4);
        start = (u32*)take(4 * (V + 1));
        part = (float*)take(M > CHUNK ? (M + CHUNK - 1) / CHUNK * 2 * dim * 4 : 0);
        bytes = p - (char*)base;
    }
};

template <typename T>
static int embed_grad(const Rows& r, const T* dout, i64 ld, int dim, float scale, T* grad, void* work, hipStream_t st) {
    const i64 M = r.n * r.m;
    const GradWork g(work, M, r.V, dim);
    int passes = 1;
    while (passes < 4 && (r.V - 1) >> (8 * passes)) ++passes;
    u64* list = g.la;
    Source s;
    s.r = r, s.list = nullptr, s.count = g.count;
    if (M <= ONE) {
        embed_sort_one_k<<<1, 1024, 0, st>>>(s, passes, list, g.count);
        const int sg = grid_for(r.V + 1, 256);
        embed_starts_one_k<<<sg > 1024 ? 1024 : sg, 256, 0, st>>>(list, g.count, r.V, g.start);
    } else {
        for (int p = 0; p < passes; ++p) {
            u64* to = p & 1 ? g.lb : g.la;
            if (p == 0) embed_count_k<true><<<g.tiles, 256, 0, st>>>(s, g.tile, 0, g.tiles, g.hist);
            else embed_count_k<false><<<g.tiles, 256, 0, st>>>(s, g.tile, 8 * p, g.tiles, g.hist);
            embed_sums_k<<<256, 256, 0, st>>>(g.hist, g.tiles, g.total);
            if (p == 0) embed_place_k<true><<<g.tiles, 256, 0, st>>>(s, g.tile, 0, g.tiles, g.hist, g.total, to, g.count);
            else embed_place_k<false><<<g.tiles, 256, 0, st>>>(s, g.tile, 8 * p, g.tiles, g.hist, g.total, to, g.count);
            s.list = list = to;
        }
        const int sg = grid_for(M + 1, 256);
        embed_starts_k<<<sg > 4096 ? 4096 : sg, 256, 0, st>>>(list, g.count, r.V, g.start);
    }
    return with_vec<T>(vec_of<T>(dim), [&](auto c) {
        constexpr int VEC = decltype(c)::value;
        const int chunks = (dim + 64 * VEC - 1) / (64 * VEC), per = (dim + VEC - 1) / VEC;
        const i64 spans = (M + CHUNK - 1) / CHUNK, items = spans * chunks;
        const int zg = grid_for(r.V * per, 256);
        embed_zero_k<T, VEC><<<zg > 65536 ? 65536 : zg, 256, 0, st>>>(g.start, r.V, dim, per, grad);
        if (M > 0)
            embed_runs_k<T, VEC><<<wave_grid(items), 256, 0, st>>>(list, g.count, r.w, r.m, dout, ld, dim, chunks, scale, spans,
                                                                   g.part, grad);
        if (M > CHUNK)
            embed_join_k<T, VEC><<<(int)(items < 2048 ? items : 2048), 512, 0, st>>>(list, g.count, g.start, dim, chunks, spans,
                                                                                       scale, g.part, grad);
        return (int)hipGetLastError();
    });
}

template <typename T>
static int embed_dw(const Rows& r, const T* table, i64 ld, const T* dout, i64 dld, int dim, float scale, float* dw,
                    hipStream_t st) {
    return with_vec<T>(vec_of<T>(dim), [&](auto c) {
        constexpr int VEC = decltype(c)::value;
        embed_dw_k<T, VEC><<<wave_grid(r.n), 256, 0, st>>>(r, table, ld, dout, dld, dim, scale, dw);
        return (int)hipGetLastError();
    });
}

static Rows rows_of(const void* tokens, int tsize, const float* w, const void* cell, int csize, i64 n, int m, int entries,
                    i64 V) {
    Rows r;
    r.tokens = tokens, r.w = w, r.cell = cell, r.n = n, r.m = m, r.entries = entries, r.tsize = tsize, r.csize = csize;
    r.V = V;
    return r;
}

extern "C" int ng_embed(const void* table, i64 ld, i64 V, int dim, int dtype, const void* tokens, int tsize, const float* w,
                        const void* cell, int csize, i64 n, int m, int entries, float scale, void* out, void* stream) {
    const Rows r = rows_of(tokens, tsize, w, cell, csize, n, m, entries, V);
    if (!rows_ok(r, dim)) return -1;
    if (n == 0) return 0;
    hipStream_t st = (hipStream_t)stream;
    switch (dtype) {
        case NG_F32: return embed_fwd<float>(r, (const float*)table, ld, dim, scale, (float*)out, st);
        case NG_BF16: return embed_fwd<b16>(r, (const b16*)table, ld, dim, scale, (b16*)out, st);
        case NG_F16: return embed_fwd<f16>(r, (const f16*)table, ld, dim, scale, (f16*)out, st);
        default: return -1;
    }
}

extern "C" i64 ng_embed_grad_work(i64 entries, i64 V, i64 dim) {
    if (entries < 0 || V < 1 || dim < 1) return -1;
    return GradWork(nullptr, entries, V, (int)dim).bytes;
}

extern "C" int ng_embed_grad(const void* dout, i64 ld, i64 V, int dim, int dtype, const void* tokens, int tsize,
                             const float* w, const void* cell, int csize, i64 n, int m, int entries, float scale, void* grad,
                             void* work, void* stream) {
    const Rows r = rows_of(tokens, tsize, w, cell, csize, n, m, entries, V);
    if (!rows_ok(r, dim)) return -1;
    hipStream_t st = (hipStream_t)stream;
    switch (dtype) {
        case NG_F32: return embed_grad<float>(r, (const float*)dout, ld, dim, scale, (float*)grad, work, st);
        case NG_BF16: return embed_grad<b16>(r, (const b16*)dout, ld, dim, scale, (b16*)grad, work, st);
        case NG_F16: return embed_grad<f16>(r, (const f16*)dout, ld, dim, scale, (f16*)grad, work, st);
        default: return -1;
    }
}

extern "C" int ng_embed_slopes(const void* table, i64 ld, const void* dout, i64 dld, i64 V, int dim, int dtype,
                               const void* tokens, int tsize, const float* w, const void* cell, int csize, i64 n, int m,
                               int entries, float scale, float* dw, void* stream) {
    const Rows r = rows_of(tokens, tsize, w, cell, csize, n, m, entries, V);
    if (!rows_ok(r, dim)) return -1;
    if (n == 0) return 0;
    hipStream_t st = (hipStream_t)stream;
    switch (dtype) {
        case NG_F32: return embed_dw<float>(r, (const float*)table, ld, (const float*)dout, dld, dim, scale, dw, st);
        case NG_BF16: return embed_dw<b16>(r, (const b16*)table, ld, (const b16*)dout, dld, dim, scale, dw, st);
        case NG_F16: return embed_dw<f16>(r, (const f16*)table, ld, (const f16*)dout, dld, dim, scale, dw, st);
        default: return -1;
    }
}

extern "C" int ng_embed_weight_grad(const void* table, i64 ld, const void* dout, i64 dld, i64 V, int dim, int dtype,
                                    const void* tokens, int tsize, const void* cell, int csize, i64 n, int m, int entries,
                                    float scale, float* dw, void* stream) {
    return ng_embed_slopes(table, ld, dout, dld, V, dim, dtype, tokens, tsize, nullptr, cell, csize, n, m, entries, scale, dw,
                           stream);
}
