// Hint rows embedded, and the table's gradient.
//
//   out[n] = scale * sum_j w[n, j] * table[tok[n, j]]     over the entries j = (slot, candidate) of position n that count:
//            w[n, j] != 0 and cell[n, slot] > 0; without weights one entry of weight 1
//   grad[v] = scale * sum over the counted entries of token v of w[n, j] * dout[n]
//   dw[n, j] = scale * <table[tok[n, j]], dout[n]> where the slot has a cell, else 0
//
// An entry that does not count is not read (its table row may hold anything). A counted token outside the table is never
// read either: its position's output is NaN, its dw NaN, and it adds to no gradient. Sums are held in 32 bits, in a fixed
// order, and rounded once.
#include "prim.h"
#include "vals.h"

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

__device__ __forceinline__ float lane_f(float x, int l) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), l)); }
__device__ __forceinline__ int lane_i(int x, int l) { return __builtin_amdgcn_readlane(x, l); }

// The rows that the lanes of `live` name (`row` of a lane, weighted `w`), added up at this lane's column: U rows' loads in
// flight together.
template <typename T, int VEC, int U>
__device__ __forceinline__ void sum_rows(const T* __restrict__ base, i64 ld, int col, bool in, u64 live, int row, float w,
                                         Acc<T, VEC>& acc) {
    while (live) {
        const int have = __popcll(live);
        int at[U];
        u64 rest = live;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            at[u] = rest ? __builtin_ctzll(rest) : at[0];
            rest &= rest - 1;
        }
        if (have >= U) {
            Pack<T, VEC> p[U];
            if (in)
#pragma unroll
                for (int u = 0; u < U; ++u) p[u].load(base + (i64)(u32)lane_i(row, at[u]) * ld + col);
            if (in)
#pragma unroll
                for (int u = 0; u < U; ++u) acc.add(p[u], lane_f(w, at[u]));
            live = rest;
        } else {
            const float x = lane_f(w, at[0]);
            const i64 r = (u32)lane_i(row, at[0]);
            if (in) {
                Pack<T, VEC> p;
                p.load(base + r * ld + col);
                acc.add(p, x);
            }
            live &= live - 1;
        }
    }
}

// A wave per (position, chunk of 64 * VEC columns).
template <typename T, int VEC>
__global__ __launch_bounds__(256) void embed_rows_k(const Rows r, const T* __restrict__ table, i64 ld, int dim, float scale,
                                                    T* __restrict__ out, int chunks) {
    const i64 items = r.n * chunks, step = (i64)gridDim.x * 4;
    for (i64 it = (i64)blockIdx.x * 4 + (threadIdx.x >> 6); it < items; it += step) {
        const i64 n = it / chunks;
        const int col = ((int)(it - n * chunks) * 64 + lane_id()) * VEC;
        const bool in = col < dim;
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
            sum_rows<T, VEC, 4>(table, ld, col, in, __ballot(w != 0.f && !out_of), (int)tok, w, acc);
        }
        if (bad)
#pragma unroll
            for (int j = 0; j < VEC; ++j) acc.v[j] = __builtin_nanf("");
        if (in) acc.store(out + n * dim + col, scale);
    }
}

// Without weights: a thread per VEC columns of a position, four of them in flight.
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
                if (ok[u]) p[u].load(table + tok * ld + (i - n * per) * VEC);
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
                acc.store(out + n * dim + (i - n * per) * VEC, scale);
            }
        }
    }
}

// ------------------------------------------------------------------------------------------------ the table's gradient

__global__ __launch_bounds__(256) void embed_emit_k(const Rows r, u64* __restrict__ keys, u32* __restrict__ vals) {
    const i64 M = r.n * r.m;
    for (i64 i = (i64)blockIdx.x * 256 + threadIdx.x; i < M; i += (i64)gridDim.x * 256) {
        u64 k = (u64)r.V;
        if (weight_of(r, i) != 0.f) {
            const i64 t = int_at(r.tokens, r.tsize, i);
            if ((u64)t < (u64)r.V) k = (u64)t;
        }
        keys[i] = k;
        vals[i] = (u32)i;
    }
}

// start[v] = the first sorted entry whose token is >= v, v in [0, V]; a gap of many tokens is filled by the whole wave
__global__ __launch_bounds__(256) void embed_starts_k(const u64* __restrict__ keys, i64 M, i64 V, u32* __restrict__ start) {
    for (i64 w0 = (i64)blockIdx.x * 256 + (threadIdx.x & ~63); w0 <= M; w0 += (i64)gridDim.x * 256) {
        const i64 i = w0 + lane_id();
        i64 lo = 0, hi = 0;  // this entry opens the tokens [lo, hi)
        if (i <= M) {
            lo = i ? (i64)keys[i - 1] + 1 : 0;
            hi = (i < M ? (i64)keys[i] : V) + 1;
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

#define PIECE 64  // a token with more entries than this is summed in pieces of the sorted list's chunks of this many

// The sum over sorted entries [a, b) (at most 64) at this lane's column.
template <typename T, int VEC>
__device__ __forceinline__ void sum_entries(const u32* __restrict__ vals, u32 a, u32 b, const float* __restrict__ w, int m,
                                            const T* __restrict__ dout, i64 ld, int col, bool in, Acc<T, VEC>& acc) {
    const u32 i = a + lane_id();
    int n = 0;
    float x = 0.f;
    if (i < b) {
        const u32 e = vals[i];
        x = w ? w[e] : 1.f;
        n = (int)(e / (u32)m);
    }
    sum_rows<T, VEC, 4>(dout, ld, col, in, __ballot(i < b), n, x, acc);
}

// A wave per (chunk of PIECE sorted entries, chunk of columns): the sums of a frequent token's part at the chunk's start
// (slot 2 * chunk) and at its end (slot 2 * chunk + 1). A token with more than PIECE entries holds a chunk's first entry or
// its last one wherever it touches it, so there are no others.
template <typename T, int VEC>
__global__ __launch_bounds__(256) void embed_pieces_k(const u64* __restrict__ keys, const u32* __restrict__ vals,
                                                      const u32* __restrict__ start, i64 V, const float* __restrict__ w,
                                                      int m, const T* __restrict__ dout, i64 ld, int dim, int chunks,
                                                      i64 pieces, float* __restrict__ part) {
    const u32 M = start[V];
    const i64 items = pieces * chunks;
    for (i64 it = (i64)blockIdx.x * 4 + (threadIdx.x >> 6); it < items; it += (i64)gridDim.x * 4) {
        const i64 c = it / chunks;
        const u32 c0 = (u32)(c * PIECE);
        if (c0 >= M) return;
        const u32 c1 = M - c0 < PIECE ? M : c0 + PIECE;
        const int col = ((int)(it - c * chunks) * 64 + lane_id()) * VEC;
        const u32 t[2] = {(u32)keys[c0], (u32)keys[c1 - 1]};
#pragma unroll
        for (int side = 0; side < 2; ++side) {
            if (side && t[1] == t[0]) break;
            const u32 s = start[t[side]], e = start[t[side] + 1];
            if (e - s <= PIECE) continue;
            Acc<T, VEC> acc;
            acc.zero();
            sum_entries<T, VEC>(vals, s > c0 ? s : c0, e < c1 ? e : c1, w, m, dout, ld, col, col < dim, acc);
            if (col < dim) {
                float* o = part + (2 * c + side) * dim + col;
#pragma unroll
                for (int j = 0; j < VEC; ++j) o[j] = acc.v[j];
            }
        }
    }
}

// A wave per (token, chunk of columns): its gradient row, from its entries or from its pieces.
template <typename T, int VEC>
__global__ __launch_bounds__(256) void embed_grad_k(const u32* __restrict__ vals, const u32* __restrict__ start, i64 V,
                                                    const float* __restrict__ w, int m, const T* __restrict__ dout, i64 ld,
                                                    int dim, int chunks, float scale, const float* __restrict__ part,
                                                    T* __restrict__ grad) {
    const i64 items = V * chunks;
    for (i64 it = (i64)blockIdx.x * 4 + (threadIdx.x >> 6); it < items; it += (i64)gridDim.x * 4) {
        const i64 v = it / chunks;
        const int col = ((int)(it - v * chunks) * 64 + lane_id()) * VEC;
        const bool in = col < dim;
        const u32 s = start[v], e = start[v + 1];
        Acc<T, VEC> acc;
        acc.zero();
        if (e - s <= PIECE) {
            if (e > s) sum_entries<T, VEC>(vals, s, e, w, m, dout, ld, col, in, acc);
        } else if (in) {
            const i64 c0 = s / PIECE, c1 = (e - 1) / PIECE;
            for (i64 c = c0; c <= c1; ++c) {
                const float* p = part + (2 * c + (c == c0 && s % PIECE ? 1 : 0)) * dim + col;
#pragma unroll
                for (int j = 0; j < VEC; ++j) acc.v[j] += p[j];
            }
        }
        if (in) acc.store(grad + v * dim + col, scale);
    }
}

// A wave per position: the slopes of its weights, 8 entries at a time.
template <typename T, int VEC>
__global__ __launch_bounds__(256) void embed_dw_k(const Rows r, const T* __restrict__ table, i64 ld, const T* __restrict__ dout,
                                                  i64 dld, int dim, float scale, float* __restrict__ dw) {
    for (i64 n = (i64)blockIdx.x * 4 + (threadIdx.x >> 6); n < r.n; n += (i64)gridDim.x * 4) {
        for (int base = 0; base < r.m; base += 64) {
            const int j = base + lane_id();
            i64 tok = -1;
            bool counts = false;
            if (j < r.m) {
                counts = has_cell(r, n * r.m + j);
                if (counts) tok = int_at(r.tokens, r.tsize, n * r.m + j);
            }
            const bool ok = counts && (u64)tok < (u64)r.V;
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
                for (int col = lane_id() * VEC; col < dim; col += 64 * VEC) {
                    Pack<T, VEC> d, p[8];
                    d.load(dout + n * dld + col);
#pragma unroll
                    for (int u = 0; u < 8; ++u)
                        if (at[u] >= 0) p[u].load(table + (i64)(u32)lane_i((int)tok, at[u]) * ld + col);
#pragma unroll
                    for (int u = 0; u < 8; ++u)
                        if (at[u] >= 0)
#pragma unroll
                            for (int k = 0; k < VEC; ++k) dot[u] = fmaf((float)d.v[k], (float)p[u].v[k], dot[u]);
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

// The most elements of 16 bytes or fewer that a row's loads may take: every pointer and row stride a multiple of them, the
// row a whole number of them, and (where a wave takes one row) more than `lanes` lanes with work.
template <typename T> static int vec_of(u64 where, int dim, int lanes = 32) {
    int v = 16 / (int)sizeof(T);
    while (v > 1 && ((where & (v * sizeof(T) - 1)) || dim % v || dim / v <= lanes)) v >>= 1;
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
    const u64 where = (u64)table | (u64)out | (u64)(ld * sizeof(T));
    const bool plain = !r.w && !r.cell && r.m == 1;
    return with_vec<T>(vec_of<T>(where, dim, plain ? 0 : 32), [&](auto c) {
        constexpr int VEC = decltype(c)::value;
        if (plain) {
            const int per = dim / VEC;
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
    u64 *ka, *kb;
    u32 *va, *vb, *start;
    void* sort;
    size_t sort_bytes;
    float* part;
    i64 bytes;
    GradWork(void* base, i64 M, i64 V, int dim) {
        char* p = (char*)base;
        const auto take = [&](i64 n) {
            char* q = p;
            p += (n + 255) / 256 * 256;
            return (void*)q;
        };
        sort_bytes = prim::radix_sort_temp_bytes(M, true);
        ka = (u64*)take(8 * M), kb = (u64*)take(8 * M), va = (u32*)take(4 * M), vb = (u32*)take(4 * M);
        start = (u32*)take(4 * (V + 1));
        sort = take((i64)sort_bytes);
        part = (float*)take((M + PIECE - 1) / PIECE * 2 * dim * 4);
        bytes = p - (char*)base;
    }
};

template <typename T>
static int embed_grad(const Rows& r, const T* dout, i64 ld, int dim, float scale, T* grad, void* work, hipStream_t st) {
    const i64 M = r.n * r.m;
    const GradWork g(work, M, r.V, dim);
    int bits = 1;
    while (bits < 32 && (r.V >> bits)) ++bits;
    const int eg = grid_for(M, 256);
    embed_emit_k<<<eg > 4096 ? 4096 : eg, 256, 0, st>>>(r, g.ka, g.va);
    int rc = prim::radix_sort_pairs(g.ka, g.kb, g.va, g.vb, M, 0, bits, g.sort, g.sort_bytes, st);
    if (rc) return rc;
    const int sg = grid_for(M + 1, 256);
    embed_starts_k<<<sg > 4096 ? 4096 : sg, 256, 0, st>>>(g.kb, M, r.V, g.start);
    const u64 where = (u64)dout | (u64)grad | (u64)(ld * sizeof(T));
    return with_vec<T>(vec_of<T>(where, dim), [&](auto c) {
        constexpr int VEC = decltype(c)::value;
        const int chunks = (dim + 64 * VEC - 1) / (64 * VEC);
        const i64 pieces = (M + PIECE - 1) / PIECE;
        embed_pieces_k<T, VEC><<<wave_grid(pieces * chunks), 256, 0, st>>>(g.kb, g.vb, g.start, r.V, r.w, r.m, dout, ld, dim,
                                                                           chunks, pieces, g.part);
        embed_grad_k<T, VEC><<<wave_grid(r.V * chunks), 256, 0, st>>>(g.vb, g.start, r.V, r.w, r.m, dout, ld, dim, chunks,
                                                                      scale, g.part, grad);
        return (int)hipGetLastError();
    });
}

template <typename T>
static int embed_dw(const Rows& r, const T* table, i64 ld, const T* dout, i64 dld, int dim, float scale, float* dw,
                    hipStream_t st) {
    const u64 where = (u64)table | (u64)dout | (u64)((ld | dld) * sizeof(T));
    return with_vec<T>(vec_of<T>(where, dim), [&](auto c) {
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

extern "C" int ng_embed_weight_grad(const void* table, i64 ld, const void* dout, i64 dld, i64 V, int dim, int dtype,
                                    const void* tokens, int tsize, const void* cell, int csize, i64 n, int m, int entries,
                                    float scale, float* dw, void* stream) {
    const Rows r = rows_of(tokens, tsize, nullptr, cell, csize, n, m, entries, V);
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
