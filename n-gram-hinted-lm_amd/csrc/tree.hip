// Attention for a tree of drafted tokens over a paged key/value cache.
//
//   o[i] = sum_p softmax_p(scale * q[i] . k[p]) v[p]   over the positions p that tree token i sees: the sequence's cached
//          tokens, and the tree token j (position length + j) where bit j of mask[i] is set; a row that sees nothing: 0
//
// Mathematics. One pass over the keys with a running maximum M and sum l per row, in base 2 and 32 bits. A cache held in
// 8 bits is not dequantised: the key's scale multiplies the finished score, and the value's scale joins the exponent,
// P = exp2(score + log2(vscale) - M), so that P stays in (0, 1] whatever the scales are and the product P V runs on the
// codes; the sum of the softmax then takes P / vscale. Codes of 8 bits are exact in 16-bit floats. The 8-bit caches run
// on f16 products (queries scaled by a power of two to f16's range), 16-bit caches on their own type.
//
// Layout. The scores are computed transposed (keys x rows), so that a lane holds 8 keys of one row: its maximum, sum and
// rescaling are its own, and its P are the next product's operand as they stand, without a move between lanes. The output
// is transposed too (dims x rows). Keys and values go from memory straight into the operand registers: which key an
// operand row means, and which dimension, is chosen so that a lane's loads are contiguous (keys: a quarter of a row;
// values: a sixteenth of 8 rows).
//
// Split. The work of every (sequence, kv head, group of rows) is laid end to end in tiles of 128 keys, and each block
// takes an equal share, wherever that begins and ends: ragged lengths balance, and the lengths are read on the device
// only. A share that ends inside a unit leaves its rows' M, l and sums in the workspace, and a second kernel joins them.
// The four waves of a block take 32 keys of a tile each and join in LDS at a unit's end.
#include "vals.h"

typedef float f4 __attribute__((ext_vector_type(4)));
typedef f16 h8 __attribute__((ext_vector_type(8)));
typedef b16 b8 __attribute__((ext_vector_type(8)));

#define TILE 128  // keys of a block's step: 32 a wave
#define LOG2E 1.4426950408889634f
#define LN2 0.6931471805599453f

struct TreeArgs {
    const void* q;
    i64 qb, qt, qh;  // strides of q [B, T, H * G, dim] in elements
    const void *k, *v;
    const float *ks, *vs;
    const int* table;
    i64 table_stride;
    const int *lengths, *widths;
    const u64* mask;
    void* out;   // [B, T, H * G, dim]
    float* lse;  // [B, T, H * G] or NULL
    float *po, *pm, *pl;  // partial sums [2 * blocks, rows a block, DP], maxima and sums [2 * blocks, rows a block]
    i64 pages;
    int B, T, H, G, dim, shift, width;  // width: the table's entries a sequence
    int groups;  // row groups of a kv head
    int qtype, vec;
    float scale;
};

struct Seq {
    int len, w, n, tiles;
};

__device__ __forceinline__ Seq seq_of(const TreeArgs& a, int b) {
    Seq s;
    const i64 cap = (i64)a.width << a.shift;
    const int l = a.lengths[b], w = a.widths ? a.widths[b] : a.T;
    s.len = l < 0 ? 0 : (i64)l > cap ? (int)cap : l;
    s.w = w < 0 ? 0 : w > a.T ? a.T : w;
    const i64 n = (i64)s.len + s.w;
    s.n = (int)(n < cap ? n : cap);
    s.tiles = s.n > 0 ? (s.n + TILE - 1) / TILE : 1;
    return s;
}

// The tiles of the sequences before b (b = B: of all), by one wave.
__device__ __forceinline__ i64 tiles_before(const TreeArgs& a, int b) {
    i64 t = 0;
    for (int i = lane_id(); i < b; i += 64) t += seq_of(a, i).tiles;
#pragma unroll
    for (int o = 32; o; o >>= 1) t += (i64)__shfl_xor((long long)t, o, 64);
    return t * a.H * a.groups;
}

// The sequence that holds flat tile x, and the tiles before it.
__device__ __forceinline__ int seq_at(const TreeArgs& a, i64 x, i64& before) {
    const i64 per = (i64)a.H * a.groups;
    i64 run = 0;
    for (int b0 = 0; b0 < a.B; b0 += 64) {
        const int b = b0 + lane_id();
        const i64 mine = b < a.B ? seq_of(a, b).tiles * per : 0;
        i64 inc = mine;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const i64 up = (i64)__shfl_up((long long)inc, o, 64);
            if (lane_id() >= o) inc += up;
        }
        const u64 past = __ballot(run + inc > x);
        if (past) {
            const int l = __builtin_ctzll(past);
            before = run + (i64)__shfl((long long)(inc - mine), l, 64);
            return b0 + l;
        }
        run += (i64)__shfl((long long)inc, 63, 64);
    }
    before = run;
    return a.B;
}

// ---------------------------------------------------------------------------------------------- codes to operands

template <int CODES> struct op_t { typedef f16 type; };
template <> struct op_t<KV_BF16> { typedef b16 type; };

__device__ __forceinline__ f4 mma(h8 a, h8 b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f4 mma(b8 a, b8 b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }

template <int CODES> __device__ __forceinline__ f16 code_f16(u32 w, int byte) {
    if constexpr (CODES == KV_INT8) return (f16)(float)(signed char)(w >> (8 * byte));
    else {
        const auto x = byte < 2 ? __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false) : __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
        return (f16)x[byte & 1];
    }
}

// Eight consecutive elements of a row (8-bit: two words; 16-bit: four) as an operand.
template <int CODES, typename V8> __device__ __forceinline__ V8 row_operand(const u32* w) {
    V8 r;
    if constexpr (CODES == KV_INT8 || CODES == KV_FP8) {
#pragma unroll
        for (int i = 0; i < 8; ++i) r[i] = code_f16<CODES>(w[i >> 2], i & 3);
    } else {
        union {
            u32 u[4];
            V8 v;
        } x;
#pragma unroll
        for (int i = 0; i < 4; ++i) x.u[i] = w[i];
        r = x.v;
    }
    return r;
}

// Element j of eight rows (v[row][words]) as an operand.
template <int CODES, typename V8, int VW> __device__ __forceinline__ V8 col_operand(const u32 (&v)[8][VW], int j) {
    V8 r;
    if constexpr (CODES == KV_INT8 || CODES == KV_FP8) {
#pragma unroll
        for (int i = 0; i < 8; ++i) r[i] = code_f16<CODES>(v[i][j >> 2], j & 3);
    } else {
        union {
            u32 u[4];
            V8 v;
        } x;
        const u32 sel = j & 1 ? 0x07060302u : 0x05040100u;
#pragma unroll
        for (int i = 0; i < 4; ++i) x.u[i] = __builtin_amdgcn_perm(v[2 * i + 1][j >> 1], v[2 * i][j >> 1], sel);
        r = x.v;
    }
    return r;
}

// N words at p, which is aligned to a word at least (rows of 192 put a lane's values at multiples of 12 bytes)
typedef u32 w4 __attribute__((ext_vector_type(4), aligned(4)));
typedef u32 w2 __attribute__((ext_vector_type(2), aligned(4)));
template <int N> __device__ __forceinline__ void load_words(const char* p, u32* w) {
#pragma unroll
    for (int i = 0; i + 4 <= N; i += 4) {
        const w4 x = *(const w4*)(p + 4 * i);
        w[i] = x[0], w[i + 1] = x[1], w[i + 2] = x[2], w[i + 3] = x[3];
    }
    if constexpr (N % 4 >= 2) {
        const w2 x = *(const w2*)(p + 4 * (N / 4 * 4));
        w[N / 4 * 4] = x[0], w[N / 4 * 4 + 1] = x[1];
    }
    if constexpr (N % 2 == 1) w[N - 1] = *(const u32*)(p + 4 * (N - 1));
}

__device__ __forceinline__ float max_quarters(float x) {  // over the lanes of one row: lane, lane ^ 16, lane ^ 32, ^ 48
    x = fmaxf(x, __shfl_xor(x, 16, 64));
    return fmaxf(x, __shfl_xor(x, 32, 64));
}
__device__ __forceinline__ float sum_quarters(float x) {
    x += __shfl_xor(x, 16, 64);
    return x + __shfl_xor(x, 32, 64);
}

__device__ __forceinline__ float q_at(const TreeArgs& a, i64 i) {
    return a.qtype == NG_BF16 ? (float)((const b16*)a.q)[i] : (float)((const f16*)a.q)[i];
}

__device__ __forceinline__ void put(const TreeArgs& a, i64 i, float x) {
    if (a.qtype == NG_BF16) ((b16*)a.out)[i] = (b16)x;
    else ((f16*)a.out)[i] = (f16)x;
}

// CODES: the cache's; DP: its padded row; R: rows a block / 16.
template <int CODES, int DP, int R> struct Tree {
    typedef typename op_t<CODES>::type T;
    typedef T V8 __attribute__((ext_vector_type(8)));
    static constexpr bool Q8 = CODES == KV_INT8 || CODES == KV_FP8;
    static constexpr int ES = Q8 ? 1 : 2;       // bytes a code
    static constexpr int KW = DP * ES / 16;     // words of a lane's quarter of a key row
    static constexpr int VW = DP * ES / 64;     // words of a lane's sixteenth of a value row
    static constexpr int KS = DP / 32;          // product steps over the dimension
    static constexpr int NJ = DP / 16;          // 16-dimension tiles of the output
    static constexpr float BIAS = Q8 ? 8.f : 0.f;   // P's exponent is raised by this: f16 holds 2^-24 of the largest
    static constexpr float SLACK = 4.f;             // M follows the maximum only when that passes it by 2^SLACK

    struct Frag {
        u32 k[2][KW], v[8][VW];
        float ks[8], vs[8];
        bool ok;  // this lane's value keys lie in a page of the cache
        bool okk;  // ... and the group of eight whose keys it loads
        i64 row;   // its first value row
    };

    struct State {
        V8 q[R][KS];
        f4 o[R][NJ];
        float m[R], l[R];
        float c;  // scale * log2(e) / the queries' power of two
    };

    static __device__ __forceinline__ void load_q(const TreeArgs& a, int b, int head, int row0, State& s) {
        const int c = lane_id() & 15, g = lane_id() >> 4, rows = a.T * a.G;
        float x[R][KS][8];
        float top = 0.f;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int row = row0 + r * 16 + c, t = row / a.G, h = row - t * a.G;
            const i64 at = b * a.qb + t * a.qt + (i64)(head * a.G + h) * a.qh;
#pragma unroll
            for (int st = 0; st < KS; ++st) {
                const int d0 = g * (DP / 4) + st * 8;
                if (row < rows && a.vec && d0 + 8 <= a.dim) {
                    if (a.qtype == NG_BF16) {
                        Pack<b16, 8> p;
                        p.load((const b16*)a.q + at + d0);
#pragma unroll
                        for (int i = 0; i < 8; ++i) x[r][st][i] = (float)p.v[i];
                    } else {
                        Pack<f16, 8> p;
                        p.load((const f16*)a.q + at + d0);
#pragma unroll
                        for (int i = 0; i < 8; ++i) x[r][st][i] = (float)p.v[i];
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i) x[r][st][i] = row < rows && d0 + i < a.dim ? q_at(a, at + d0 + i) : 0.f;
                }
                if constexpr (Q8)
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if (finite_f(x[r][st][i])) top = fmaxf(top, __builtin_fabsf(x[r][st][i]));
            }
        }
        float up = 1.f;
        s.c = a.scale * LOG2E;
        if constexpr (Q8) {  // the largest query element of these rows at 2^14 .. 2^15
#pragma unroll
            for (int o = 32; o; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
            if (top > 0.f) {
                int e = 15 - __builtin_amdgcn_frexp_expf(top);
                e = e > 100 ? 100 : e;
                up = __builtin_amdgcn_ldexpf(1.f, e);
                s.c *= __builtin_amdgcn_ldexpf(1.f, -e);
            }
        }
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int st = 0; st < KS; ++st)
#pragma unroll
                for (int i = 0; i < 8; ++i) s.q[r][st][i] = (T)(Q8 ? x[r][st][i] * up : x[r][st][i]);
    }

    // the table's entry of the page that holds position p (any entry of the sequence where p is past the table)
    static __device__ __forceinline__ int page_of(const TreeArgs& a, const int* tab, int p) {
        int e = p >> a.shift;
        e = e < a.width ? e : a.width - 1;
        return tab[e];
    }

    // this wave's 32 keys at `base`: their pages pk (of the key group c >> 2) and pv (of the value group g)
    static __device__ __forceinline__ void fetch(const TreeArgs& a, int head, int base, int pk, int pv, Frag& f) {
        const int c = lane_id() & 15, g = lane_id() >> 4, mask = (1 << a.shift) - 1;
        f.okk = (u32)pk < (u64)a.pages;
        f.ok = (u32)pv < (u64)a.pages;
        const i64 rk = ((((i64)(f.okk ? pk : 0)) * a.H + head) << a.shift) + ((base + (c >> 2) * 8) & mask) + (c & 3);
        const i64 rv = ((((i64)(f.ok ? pv : 0)) * a.H + head) << a.shift) + ((base + g * 8) & mask);
        f.row = rv;
        const char* k = (const char*)a.k + rk * (DP * ES) + g * (DP * ES / 4);
        load_words<KW>(k, f.k[0]);
        load_words<KW>(k + 4 * DP * ES, f.k[1]);
        if constexpr (Q8) {
            load_words<8>((const char*)(a.ks + rv), (u32*)f.ks);
            load_words<8>((const char*)(a.vs + rv), (u32*)f.vs);
        }
        const char* v = (const char*)a.v + rv * (DP * ES) + c * (DP * ES / 16);
#pragma unroll
        for (int i = 0; i < 8; ++i) load_words<VW>(v + i * DP * ES, f.v[i]);
    }

    // the tree tokens that a row sees
    static __device__ __forceinline__ u64 bits_of(const TreeArgs& a, int b, const Seq& q, int row) {
        const int t = row / a.G;
        if (t >= q.w) return 0;
        return a.mask ? a.mask[(i64)b * a.T + t] : (2ull << t) - 1;
    }

    // Values of a 16-bit cache that are not finite, in keys that only some rows see: they are 0 in the product (a masked
    // key's P of 0 would make NaN of them) and are added here to the rows that do see them.
    static __device__ __forceinline__ u32 take_out(Frag& f) {
        constexpr u32 E = CODES == KV_BF16 ? 0x7F80u : 0x7C00u;
        u32 bad = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int w = 0; w < VW; ++w) {
                const bool lo = (f.v[i][w] & E) == E, hi = (f.v[i][w] >> 16 & E) == E;
                bad |= (lo || hi ? 1u : 0u) << i;
                f.v[i][w] &= (lo ? 0u : 0xFFFFu) | (hi ? 0u : 0xFFFF0000u);
            }
        return bad;
    }
    static __device__ __forceinline__ void put_back(const TreeArgs& a, int b, const Seq& q, int base, int row0, const Frag& f,
                                                    u32 bad, const V8 (&p)[R], State& s) {
        const int c = lane_id() & 15, g = lane_id() >> 4;
        for (int from = 0; from < 4; ++from) {
            const i64 first = (i64)__shfl((long long)f.row, from * 16, 64);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (!__any(g == from && (bad >> i & 1))) continue;
                const T* v = (const T*)a.v + (first + i) * DP;
                const int j0 = base + from * 8 + i - q.len;
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    const float w = __shfl((float)p[r][i], from * 16 + c, 64);
                    const bool sees = j0 < 0 || (bits_of(a, b, q, row0 + r * 16 + c) >> j0 & 1);
#pragma unroll
                    for (int j = 0; j < NJ; ++j)
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const float x = (float)v[(4 * g + k) * NJ + j];
                            if (sees && !finite_f(x)) s.o[r][j][k] += w * x;
                        }
                }
            }
        }
    }

    static __device__ __forceinline__ void step(const TreeArgs& a, int b, const Seq& q, int base, int row0, Frag& f, State& s) {
        const int c = lane_id() & 15, g = lane_id() >> 4;
        const bool whole = base + 32 <= q.len && __all(f.ok);
        float kf[8], lv[8], rv[8];
        if constexpr (Q8) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                kf[i] = f.ks[i] * s.c;
                const float x = f.vs[i] == 0.f ? 1.f : f.vs[i];
                lv[i] = __builtin_amdgcn_logf(x);
                rv[i] = __builtin_amdgcn_rcpf(x);
            }
        }
        if (!whole) {  // keys past the end or without a page: nothing of them enters the products
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const bool in = f.ok && base + g * 8 + i < q.n;
#pragma unroll
                for (int w = 0; w < VW; ++w) f.v[i][w] = in ? f.v[i][w] : 0u;
                if constexpr (Q8) rv[i] = in ? rv[i] : 1.f;
            }
        }
        u32 bad = 0;
        if constexpr (!Q8)
            if (!whole) bad = take_out(f);
        f4 sc[R][2];
#pragma unroll
        for (int r = 0; r < R; ++r) sc[r][0] = sc[r][1] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int st = 0; st < KS; ++st) {
                const V8 k = row_operand<CODES, V8>(f.k[t] + st * (Q8 ? 2 : 4));
#pragma unroll
                for (int r = 0; r < R; ++r) sc[r][t] = mma(k, s.q[r][st], sc[r][t]);
            }
        V8 p[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float x[8];
#pragma unroll
            for (int i = 0; i < 8; ++i)
                x[i] = Q8 ? fmaf(sc[r][i >> 2][i & 3], kf[i], lv[i]) : sc[r][i >> 2][i & 3] * s.c;
            if (!whole) {
                const u64 bits = bits_of(a, b, q, row0 + r * 16 + c);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int at = base + g * 8 + i, j = at - q.len;
                    const bool sees = f.ok && at < q.n && (j < 0 || (j < 64 && (bits >> j & 1)));
                    x[i] = sees ? x[i] : -__builtin_inff();
                }
            }
            float top = x[0];
#pragma unroll
            for (int i = 1; i < 8; ++i) top = fmaxf(top, x[i]);
            if (__any(top > s.m[r] + SLACK)) {
                const float m = fmaxf(s.m[r], max_quarters(top));
                const float down = s.m[r] == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(s.m[r] - m);
                s.m[r] = m;
                s.l[r] *= down;
#pragma unroll
                for (int j = 0; j < NJ; ++j) s.o[r][j] *= down;
            }
            const float m0 = s.m[r] == -__builtin_inff() ? 0.f : s.m[r] - BIAS;
            float add = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float e = __builtin_amdgcn_exp2f(x[i] - m0);
                // a masked key's scale may be NaN: it does not enter the sum
                if constexpr (Q8) add = fmaf(e, !whole && e == 0.f ? 0.f : rv[i], add);
                else add += e;
                p[r][i] = (T)e;
            }
            s.l[r] += add;
        }
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            const V8 v = col_operand<CODES, V8, VW>(f.v, j);
#pragma unroll
            for (int r = 0; r < R; ++r) s.o[r][j] = mma(v, p[r], s.o[r][j]);
        }
        if constexpr (!Q8)
            if (__any(bad != 0)) put_back(a, b, q, base, row0, f, bad, p, s);
    }
};

__device__ __forceinline__ i64 share(i64 i, i64 total, i64 blocks) { return i * total / blocks; }

template <int CODES, int DP, int R> __global__ __launch_bounds__(256) void tree_k(const TreeArgs a, int blocks) {
    typedef Tree<CODES, DP, R> W;
    constexpr int LD = DP + 4;
    __shared__ float lo[4][16][LD];
    __shared__ float lm[4][16], ll[4][16];
    // neighbouring shares on one XCD (blocks go round the 8 XCDs): units that share keys meet in its L2
    const i64 me = blocks % 8 == 0 ? (i64)(blockIdx.x % 8) * (blocks / 8) + blockIdx.x / 8 : blockIdx.x;
    const int wave = threadIdx.x >> 6, c = lane_id() & 15, g = lane_id() >> 4;
    const i64 total = tiles_before(a, a.B);
    i64 x = share(me, total, blocks);
    const i64 end = share(me + 1, total, blocks);
    if (x >= end) return;
    i64 before;
    int b = seq_at(a, x, before);
    Seq q = seq_of(a, b);
    while (x < end) {
        while (x >= before + (i64)q.tiles * a.H * a.groups) {
            before += (i64)q.tiles * a.H * a.groups;
            q = seq_of(a, ++b);
        }
        const int unit = (int)((x - before) / q.tiles), t0 = (int)(x - before - (i64)unit * q.tiles);
        const int t1 = (int)(end - x < q.tiles - t0 ? t0 + (end - x) : q.tiles);
        const int head = unit / a.groups, row0 = (unit - head * a.groups) * 16 * R;
        const int* tab = a.table + (i64)b * a.table_stride;
        typename W::State s;
        W::load_q(a, b, head, row0, s);
#pragma unroll
        for (int r = 0; r < R; ++r) {
            s.m[r] = -__builtin_inff(), s.l[r] = 0.f;
#pragma unroll
            for (int j = 0; j < W::NJ; ++j) s.o[r][j] = f4{0.f, 0.f, 0.f, 0.f};
        }
        int base = t0 * TILE + wave * 32;
        const int stop = t1 * TILE < q.n ? t1 * TILE : q.n;
        for (; base < stop; base += TILE) {
            typename W::Frag f;
            W::fetch(a, head, base, W::page_of(a, tab, base + (c >> 2) * 8), W::page_of(a, tab, base + g * 8), f);
            W::step(a, b, q, base, row0, f, s);
        }
        const bool all = t0 == 0 && t1 == q.tiles;
        const i64 slot = 2 * me + (t0 == 0 ? 1 : 0);
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const float l = sum_quarters(s.l[r]);
            __syncthreads();
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < W::NJ; ++j) lo[wave][c][(4 * g + i) * W::NJ + j] = s.o[r][j][i];
            if (g == 0) lm[wave][c] = s.m[r], ll[wave][c] = l;
            __syncthreads();
            const int row = threadIdx.x >> 4, d0 = (threadIdx.x & 15) * W::NJ;
            float m = lm[0][row];
#pragma unroll
            for (int w = 1; w < 4; ++w) m = fmaxf(m, lm[w][row]);
            float sum = 0.f, o[W::NJ];
#pragma unroll
            for (int j = 0; j < W::NJ; ++j) o[j] = 0.f;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const float k = lm[w][row] == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(lm[w][row] - m);
                // a wave without a key that counts: sum and o are 0, or NaN where a NaN was seen
                sum = ll[w][row] == 0.f ? sum : fmaf(ll[w][row], lm[w][row] == -__builtin_inff() ? 1.f : k, sum);
#pragma unroll
                for (int j = 0; j < W::NJ; ++j) o[j] = fmaf(lo[w][row][d0 + j], k, o[j]);
            }
            const int at = row0 + r * 16 + row, t = at / a.G, h = at - t * a.G;
            if (all) {
                if (t < a.T) {
                    const i64 i = ((i64)b * a.T + t) * a.H * a.G + head * a.G + h;
                    const bool none = sum == 0.f || t >= q.w;
                    const float inv = none ? 0.f : 1.f / sum;
#pragma unroll
                    for (int j = 0; j < W::NJ; ++j)
                        if (d0 + j < a.dim) put(a, i * a.dim + d0 + j, none ? 0.f : o[j] * inv);
                    if (a.lse && (threadIdx.x & 15) == 0)
                        a.lse[i] = none ? -__builtin_inff() : LN2 * (m - W::BIAS + __builtin_amdgcn_logf(sum));
                }
            } else {
                const i64 prow = slot * (16 * R) + r * 16 + row;
#pragma unroll
                for (int j = 0; j < W::NJ; ++j) a.po[prow * DP + d0 + j] = o[j];
                if ((threadIdx.x & 15) == 0) a.pm[prow] = m, a.pl[prow] = sum;
            }
        }
        x += t1 - t0;
    }
}

// A block per (unit, 16 rows): the shares that hold part of the unit joined.
template <int DP> __global__ __launch_bounds__(256) void tree_join_k(const TreeArgs a, int blocks, int rpb, float bias) {
    constexpr int NJ = DP / 16;
    const int sub = rpb / 16;
    const i64 u = blockIdx.x / sub;
    const int r16 = (int)(blockIdx.x - u * sub) * 16;
    const int per = a.H * a.groups, b = (int)(u / per), unit = (int)(u - (i64)b * per);
    const i64 total = tiles_before(a, a.B), before = tiles_before(a, b);
    const Seq q = seq_of(a, b);
    const i64 x0 = before + (i64)unit * q.tiles, x1 = x0 + q.tiles;
    const i64 i0 = ((x0 + 1) * blocks - 1) / total, i1 = (x1 * blocks - 1) / total;
    if (i0 == i1) return;
    const int head = unit / a.groups, row0 = (unit - head * a.groups) * rpb;
    const int row = threadIdx.x >> 4, d0 = (threadIdx.x & 15) * NJ;
    const int at = row0 + r16 + row, t = at / a.G, h = at - t * a.G;
    if (t >= a.T) return;
    float m = -__builtin_inff(), sum = 0.f, o[NJ];
#pragma unroll
    for (int j = 0; j < NJ; ++j) o[j] = 0.f;
    for (i64 x = x0; x < x1;) {  // share by share (a share is empty where there are more blocks than tiles)
        const i64 i = ((x + 1) * blocks - 1) / total, slot = 2 * i + (i == i0 ? 1 : 0);
        x = share(i + 1, total, blocks);
        const i64 prow = slot * rpb + r16 + row;
        const float pm = a.pm[prow], pl = a.pl[prow];
        const float n = fmaxf(m, pm);
        const float ko = m == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(m - n);
        const float kp = pm == -__builtin_inff() ? (pl == 0.f ? 0.f : 1.f) : __builtin_amdgcn_exp2f(pm - n);
        sum = sum * (sum == 0.f ? 0.f : m == -__builtin_inff() ? 1.f : ko) + pl * kp;
#pragma unroll
        for (int j = 0; j < NJ; ++j) o[j] = o[j] * ko + a.po[prow * DP + d0 + j] * kp;
        m = n;
    }
    const i64 i = ((i64)b * a.T + t) * a.H * a.G + head * a.G + h;
    const bool none = sum == 0.f || t >= q.w;
    const float inv = none ? 0.f : 1.f / sum;
#pragma unroll
    for (int j = 0; j < NJ; ++j)
        if (d0 + j < a.dim) put(a, i * a.dim + d0 + j, none ? 0.f : o[j] * inv);
    if (a.lse && (threadIdx.x & 15) == 0) a.lse[i] = none ? -__builtin_inff() : LN2 * (m - bias + __builtin_amdgcn_logf(sum));
}

// bits[b, i]: tree token i sees itself and its ancestors; parents [B, T], below 0 (or not before the token): the context
__global__ __launch_bounds__(64) void tree_mask_k(const int* __restrict__ parents, int T, u64* __restrict__ bits) {
    const int b = blockIdx.x, i = lane_id();
    int p = i < T ? parents[(i64)b * T + i] : -1;
    if (p >= i || p < 0) p = -1;
    u64 m = 1ull << i;
#pragma unroll
    for (int k = 0; k < 6; ++k) {  // ancestors 1, 2, 4, .. 32 steps up
        const u64 pm = bcast_u64(m, p < 0 ? 0 : p);
        const int pp = __shfl(p, p < 0 ? 0 : p, 64);
        if (p >= 0) m |= pm, p = pp;
    }
    if (i < T) bits[(i64)b * T + i] = m;
}

// ------------------------------------------------------------------------------------------------------------ the host

#define MAX_BLOCKS 512

struct TreePlan {
    int rpb, groups, dp;
    i64 blocks;
    bool join;
    i64 po, pm, bytes;  // offsets in the workspace
};

static bool tree_plan(int B, int T, int H, int G, int dim, int codes, i64 cap, TreePlan& p) {
    if (B < 0 || T < 1 || T > 64 || H < 1 || G < 1 || dim < 1 || dim > 256 || codes < KV_INT8 || codes > KV_F16 || cap < 1 ||
        cap > (i64)1 << 30 || (i64)T * G > 1 << 20)
        return false;
    p.dp = (dim + 63) / 64 * 64;
    const int rows = T * G;
    p.rpb = rows <= 16 ? 16 : rows <= 32 || p.dp > 128 ? 32 : 64;
    p.groups = (rows + p.rpb - 1) / p.rpb;
    const i64 units = (i64)B * H * p.groups;
    if (units > (i64)1 << 30) return false;
    const i64 most = units * ((cap + TILE - 1) / TILE);
    p.blocks = most < MAX_BLOCKS ? most : MAX_BLOCKS;
    p.join = cap > TILE;
    const i64 slots = p.join ? 2 * p.blocks * p.rpb : 0;
    p.po = 0, p.pm = slots * p.dp * 4, p.bytes = p.pm + 2 * slots * 4;
    return true;
}

extern "C" i64 ng_tree_attention_work(i64 B, i64 T, i64 H, i64 G, i64 dim, i64 codes, i64 cap) {
    TreePlan p;
    const i64 lim = 1 << 30;
    if (B > lim || T > lim || H > lim || G > lim || dim > lim) return -1;
    return tree_plan((int)B, (int)T, (int)H, (int)G, (int)dim, (int)codes, cap, p) ? p.bytes : -1;
}

template <int CODES, int DP, int R> static int tree_run(const TreeArgs& a, const TreePlan& p, hipStream_t st) {
    tree_k<CODES, DP, R><<<(int)p.blocks, 256, 0, st>>>(a, (int)p.blocks);
    int rc = (int)hipGetLastError();
    if (rc || !p.join) return rc;
    const i64 g = (i64)a.B * a.H * a.groups * R;
    tree_join_k<DP><<<(int)g, 256, 0, st>>>(a, (int)p.blocks, 16 * R, Tree<CODES, DP, R>::BIAS);
    return (int)hipGetLastError();
}

template <int CODES, int DP> static int tree_rows(const TreeArgs& a, const TreePlan& p, hipStream_t st) {
    if (p.rpb == 16) return tree_run<CODES, DP, 1>(a, p, st);
    if (p.rpb == 32) return tree_run<CODES, DP, 2>(a, p, st);
    if constexpr (DP <= 128) return tree_run<CODES, DP, 4>(a, p, st);
    return -1;
}

template <int CODES> static int tree_dim(const TreeArgs& a, const TreePlan& p, hipStream_t st) {
    switch (p.dp) {
        case 64: return tree_rows<CODES, 64>(a, p, st);
        case 128: return tree_rows<CODES, 128>(a, p, st);
        case 192: return tree_rows<CODES, 192>(a, p, st);
        default: return tree_rows<CODES, 256>(a, p, st);
    }
}

extern "C" int ng_tree_attention(const void* q, i64 qb, i64 qt, i64 qh, int qtype, const void* k, const void* v,
                                 const float* ks, const float* vs, i64 pages, int page, int codes, const int* table,
                                 i64 table_stride, int width, const int* lengths, const int* widths, const u64* mask,
                                 int B, int T, int H, int G, int dim, float scale, void* out, float* lse, void* work,
                                 void* stream) {
    if (page < 16 || page > 4096 || (page & (page - 1)) || pages < 1 || pages > (i64)1 << 31 || width < 1) return -1;
    if (qtype != NG_BF16 && qtype != NG_F16) return -1;
    if ((codes == KV_BF16 && qtype != NG_BF16) || (codes == KV_F16 && qtype != NG_F16)) return -1;
    if ((codes == KV_INT8 || codes == KV_FP8) && (!ks || !vs)) return -1;
    TreePlan p;
    if (!tree_plan(B, T, H, G, dim, codes, (i64)width * page, p)) return -1;
    if (B == 0) return 0;
    TreeArgs a;
    a.q = q, a.qb = qb, a.qt = qt, a.qh = qh, a.k = k, a.v = v, a.ks = ks, a.vs = vs, a.table = table;
    a.table_stride = table_stride, a.lengths = lengths, a.widths = widths, a.mask = mask, a.out = out, a.lse = lse;
    a.po = (float*)((char*)work + p.po), a.pm = (float*)((char*)work + p.pm);
    a.pl = a.pm + (p.join ? 2 * p.blocks * p.rpb : 0);
    a.pages = pages, a.B = B, a.T = T, a.H = H, a.G = G, a.dim = dim, a.shift = __builtin_ctz((unsigned)page);
    a.width = width, a.groups = p.groups, a.qtype = qtype, a.scale = scale;
    a.vec = ((u64)q & 15) == 0 && (((qb | qt | qh) * 2) & 15) == 0;
    hipStream_t st = (hipStream_t)stream;
    switch (codes) {
        case KV_INT8: return tree_dim<KV_INT8>(a, p, st);
        case KV_FP8: return tree_dim<KV_FP8>(a, p, st);
        case KV_BF16: return tree_dim<KV_BF16>(a, p, st);
        default: return tree_dim<KV_F16>(a, p, st);
    }
}

extern "C" int ng_tree_mask(const int* parents, int B, int T, u64* bits, void* stream) {
    if (B < 0 || T < 1 || T > 64) return -1;
    if (B == 0) return 0;
    tree_mask_k<<<B, 64, 0, (hipStream_t)stream>>>(parents, T, bits);
    return (int)hipGetLastError();
}
