// The tree attention kernel (tree.hip has the mathematics and the host's side; a file per cache type instantiates it).
#pragma once
#include "vals.h"

typedef float f4 __attribute__((ext_vector_type(4)));
typedef f16 h2 __attribute__((ext_vector_type(2)));
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

struct TreePlan {
    int rpb, groups, dp;
    int blocks;
    bool join;
    i64 po, pm, bytes;  // offsets in the workspace
};

// the launches for one cache type
template <int CODES> int tree_codes(const TreeArgs& a, const TreePlan& p, hipStream_t st);

// A sequence's cached tokens, tree tokens, both, its tiles, and its units' span on the line: a unit costs its tiles and
// START more, what its beginning and end take (queries, masks, the waves' joining) in tiles' time: a share of many short
// units would else be a long one.
#define START 3
struct Seq {
    int len, w, n, tiles, span;
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
    s.span = s.tiles + START;
    return s;
}

__device__ __forceinline__ Seq uniform(Seq s) {
    s.len = __builtin_amdgcn_readfirstlane(s.len), s.w = __builtin_amdgcn_readfirstlane(s.w);
    s.n = __builtin_amdgcn_readfirstlane(s.n), s.tiles = __builtin_amdgcn_readfirstlane(s.tiles);
    s.span = s.tiles + START;
    return s;
}

__device__ __forceinline__ int scan_wave(int x) {  // inclusive sum over the lanes
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int up = __shfl_up(x, o, 64);
        if (lane_id() >= o) x += up;
    }
    return x;
}

// The work laid end to end: sequence by sequence, in each its units (kv head, group of rows), in each its span. A share is
// `per` places. Each wave finds its place by itself: one load and one scan for 64 sequences.
struct Line {
    Seq mine;  // of sequence lane_id()
    int inc;   // places up to and with it
    int total, per, shares;

    __device__ __forceinline__ Line(const TreeArgs& a, int blocks) {
        const int units = a.H * a.groups;
        const int b = lane_id() < a.B ? lane_id() : a.B - 1;
        mine = seq_of(a, b);
        inc = scan_wave(lane_id() < a.B ? mine.span * units : 0);
        total = lane(inc, 63);
        for (int b0 = 64; b0 < a.B; b0 += 64) {
            int t = b0 + lane_id() < a.B ? seq_of(a, b0 + lane_id()).span * units : 0;
            total += lane(scan_wave(t), 63);
        }
        per = (total + blocks - 1) / blocks;
        shares = (total + per - 1) / per;
    }

    // the sequence that holds place x < total, and the places before it
    __device__ __forceinline__ int at(const TreeArgs& a, int x, int& before, Seq& q) const {
        const int units = a.H * a.groups;
        u64 past = __ballot(inc > x);
        if (past) {
            const int l = __builtin_ctzll(past);
            q = pick(mine, l);
            before = lane(inc, l) - q.span * units;
            return l;
        }
        int run = lane(inc, 63);
        for (int b0 = 64;; b0 += 64) {
            Seq s;
            s.len = s.w = s.n = s.tiles = s.span = 0;
            if (b0 + lane_id() < a.B) s = seq_of(a, b0 + lane_id());
            const int i = scan_wave(s.span * units);
            past = __ballot(run + i > x);
            if (past || b0 + 64 >= a.B) {
                const int l = past ? __builtin_ctzll(past) : 63;
                q = pick(s, l);
                before = run + lane(i, l) - q.span * units;
                return b0 + l;
            }
            run += lane(i, 63);
        }
    }

    // the places before sequence b
    __device__ __forceinline__ int before(const TreeArgs& a, int b, Seq& q) const {
        const int units = a.H * a.groups;
        int run = 0;
        for (int b0 = 0;; b0 += 64) {
            Seq s = mine;
            int i = inc;
            if (b0) {
                s.len = s.w = s.n = s.tiles = s.span = 0;
                if (b0 + lane_id() < a.B) s = seq_of(a, b0 + lane_id());
                i = scan_wave(s.span * units);
            }
            if (b < b0 + 64) {
                const int l = b - b0;
                q = pick(s, l);
                return run + lane(i, l) - q.span * units;
            }
            run += lane(i, 63);
        }
    }
    static __device__ __forceinline__ Seq pick(const Seq& s, int l) {
        Seq q;
        q.len = lane(s.len, l), q.w = lane(s.w, l), q.n = lane(s.n, l), q.tiles = lane(s.tiles, l), q.span = q.tiles + START;
        return q;
    }
    static __device__ __forceinline__ int lane(int x, int l) { return __builtin_amdgcn_readlane(x, l); }
};

// ---------------------------------------------------------------------------------------------- codes to operands

template <int CODES> struct op_t { typedef f16 type; };
template <> struct op_t<KV_BF16> { typedef b16 type; };

__device__ __forceinline__ f4 mma(h8 a, h8 b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f4 mma(b8 a, b8 b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }

template <typename V8> union Words {
    u32 u[4];
    V8 v;
};

// Eight consecutive codes of a row (8 bits: two words; 16 bits: four) as an operand. int8 (its words' sign bits flipped
// where they were loaded: c + 128): the byte under 0x64 is the f16 1024 + (c + 128), exactly, and less 1152 it is c. (The
// sum over c + 128, less 128 sum(q) at the end, saves that subtraction, but a key of small codes loses its sum in 128's.)
template <int CODES, typename V8> __device__ __forceinline__ V8 row_operand(const u32* w) {
    Words<V8> x;
    if constexpr (CODES == KV_INT8) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const h2 o = {(f16)-1152.f, (f16)-1152.f};
            x.u[2 * i] = __builtin_bit_cast(u32, __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, w[i], 0x04010400u)) + o);
            x.u[2 * i + 1] = __builtin_bit_cast(u32, __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, w[i], 0x04030402u)) + o);
        }
    } else if constexpr (CODES == KV_FP8) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            x.u[2 * i] = __builtin_bit_cast(u32, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w[i], 1.f, false));
            x.u[2 * i + 1] = __builtin_bit_cast(u32, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w[i], 1.f, true));
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) x.u[i] = w[i];
    }
    return x.v;
}

// Elements 2 p and 2 p + 1 of eight rows (v[row][words]) as two operands. int8: the bytes are taken for f16 as they stand,
// which are (c + 128) 2^-24 exactly, then one multiply-add to c 2^-9 (the outputs are multiplied by 2^9 at the end).
template <int CODES, typename V8, int VW>
__device__ __forceinline__ void col_operands(const u32 (&v)[8][VW], int p, V8& lo, V8& hi) {
    Words<V8> x, y;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (CODES == KV_INT8) {
            const u32 a = v[2 * i][p >> 1], b = v[2 * i + 1][p >> 1], by = 2 * (p & 1);
            const h2 k = {(f16)32768.f, (f16)32768.f}, o = {(f16)-0.25f, (f16)-0.25f};
            const u32 s = 0x0c040c00u + by * 0x00010001u;
            x.u[i] = __builtin_bit_cast(u32, __builtin_elementwise_fma(__builtin_bit_cast(h2, __builtin_amdgcn_perm(b, a, s)), k, o));
            y.u[i] = __builtin_bit_cast(u32, __builtin_elementwise_fma(__builtin_bit_cast(h2, __builtin_amdgcn_perm(b, a, s + 0x00010001u)), k, o));
        } else if constexpr (CODES == KV_FP8) {
            const u32 by = 2 * (p & 1);
            const u32 t = __builtin_amdgcn_perm(v[2 * i + 1][p >> 1], v[2 * i][p >> 1], 0x05010400u + by * 0x01010101u);
            x.u[i] = __builtin_bit_cast(u32, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(t, 1.f, false));
            y.u[i] = __builtin_bit_cast(u32, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(t, 1.f, true));
        } else {
            x.u[i] = __builtin_amdgcn_perm(v[2 * i + 1][p], v[2 * i][p], 0x05040100u);
            y.u[i] = __builtin_amdgcn_perm(v[2 * i + 1][p], v[2 * i][p], 0x07060302u);
        }
    }
    lo = x.v, hi = y.v;
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

// N outputs at element i of out, of which the first `have` exist
template <int N> __device__ __forceinline__ void put(const TreeArgs& a, i64 i, int have, const float* x) {
    u16 e[N];
#pragma unroll
    for (int j = 0; j < N; ++j)
        e[j] = a.qtype == NG_BF16 ? __builtin_bit_cast(u16, (b16)x[j]) : __builtin_bit_cast(u16, (f16)x[j]);
    u16* o = (u16*)a.out + i;
#pragma unroll
    for (int j = 0; j < N; j += 4) {
        if (a.dim % 4 == 0) {
            if (j < have) *(uint2*)(o + j) = make_uint2(e[j] | (u32)e[j + 1] << 16, e[j + 2] | (u32)e[j + 3] << 16);
        } else
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (j + k < have) o[j + k] = e[j + k];
    }
}

// CODES: the cache's; DP: its padded row; R: rows a block / 16, 1 or 2.
template <int CODES, int DP, int R> struct Tree {
    typedef typename op_t<CODES>::type T;
    typedef T V8 __attribute__((ext_vector_type(8)));
    static constexpr bool Q8 = CODES == KV_INT8 || CODES == KV_FP8;
    static constexpr int ES = Q8 ? 1 : 2;       // bytes a code
    static constexpr int KW = DP * ES / 16;     // words of a lane's quarter of a key row
    static constexpr int VW = DP * ES / 64;     // words of a lane's sixteenth of a value row
    static constexpr int KS = DP / 32;          // product steps over the dimension
    static constexpr int NJ = DP / 16;          // 16-dimension tiles of the output
    static constexpr float BIAS = Q8 ? 8.f : 0.f;   // P's exponent is raised by this: f16 holds 2^-32 of the largest
    // The scale taken for value rows of a smaller one, zeros among them; their weights in the product with the values then
    // take the rest, scale / NONE. So such a row counts in the softmax's sum (2^-64 * 2^64: the inverse of a scale near the
    // smallest float would overflow it), and the maximum follows it only where its weight is 2^64 of the others' weighted
    // values, which are then nothing: it takes none of their bits, as a row of zeros with a scale of 1 would.
    static constexpr float NONE = 0x1p-64f;
    static constexpr float SLACK = 4.f;             // M follows the maximum only when that passes it by 2^SLACK
    static constexpr bool WILD = CODES != KV_INT8;  // codes can be NaN or infinite
    static constexpr float V_UP = CODES == KV_INT8 ? 512.f : 1.f;

    struct Pages {
        int k, v, s;  // of the keys this lane loads: key group c >> 2, value group g, scale group
    };
    struct Keys {
        u32 k[2][KW];
        float s;   // lanes 0 .. 31: the key scale of key lane; 32 .. 63: the value scale of key lane - 32
    };
    struct Values {
        u32 v[8][VW];
        bool ok;   // this lane's keys lie in a page of the cache
        i64 row;   // its first value row
    };
    static constexpr bool QLDS = R == 2;  // the queries are read from LDS for every tile: registers go to loads in flight

    struct State {
        V8 q[QLDS ? 1 : R][KS];
        const T* ql;  // the queries in LDS, at this lane's row and quarter
        f4 o[R][NJ];
        float m[R], l[R];
        float c;  // the scores' factor: scale * log2(e) / the queries' power of two (own: without powers of two)
    };

    // A block's rows' largest elements (as bits: the largest of floats >= 0), zero between units, and their shifts.
    struct Sizes {
        u32 top[16 * R];
        int shift[16 * R];
    };
    static constexpr int APART = 8;  // rows whose largest elements lie within 2^APART share one power of two

    static constexpr int QLD = DP + 8;                    // a query row in LDS (16 rows' reads meet no bank twice)
    static constexpr int NQ = (16 * R * DP / 8 + 255) / 256;  // groups of 8 query elements a thread brings

    // The block's query rows in use, through LDS: each read once; a row past the tree's width is zeros, whatever it holds.
    // For 8-bit caches the products run on f16: rows are scaled by the power of two that puts their largest finite element
    // at 2^14 .. 2^15. Rows of about one size share it, the largest's (an element then keeps its bits down to 2^-22 of its
    // own row's largest, and is off by 2^-31 of that below); where a row is over 2^APART smaller than another, or their size
    // is far from 1 (its power of two times the scale or a key's scale could overflow), each has its own, and its scores
    // take one more operation. bits: the tree tokens that each row sees.
    // Returns whether each row has its own power of two (a score then takes 2^shift[row]).
    static __device__ __forceinline__ bool load_q(const TreeArgs& a, int b, int head, const Seq& q, int row0, T* lds, Sizes& size,
                                                  u64* bits, State& s) {
        const int c = lane_id() & 15, g = lane_id() >> 4;
        u64 seen = 0;
        if (threadIdx.x < 16 * R) {
            const int t = (row0 + threadIdx.x) / a.G;
            if (t < q.w) seen = a.mask ? a.mask[(i64)b * a.T + t] : (2ull << t) - 1;
        }
        union Eight {
            uint4 w;
            u16 e[8];
        } x[NQ];
#pragma unroll
        for (int k = 0; k < NQ; ++k) {
            const int i = threadIdx.x + 256 * k, row = row0 + i / (DP / 8), d0 = i % (DP / 8) * 8;
            const int t = row / a.G, h = row - t * a.G;
            const u16* p = (const u16*)a.q + b * a.qb + t * a.qt + (i64)(head * a.G + h) * a.qh + d0;
            x[k].w = make_uint4(0, 0, 0, 0);
            if (i < 16 * R * DP / 8 && t < q.w) {
                if (a.vec && d0 + 8 <= a.dim) x[k].w = *(const uint4*)p;
                else
                    for (int j = 0; j < 8; ++j)
                        if (d0 + j < a.dim) x[k].e[j] = p[j];
            }
        }
        if constexpr (Q8)
#pragma unroll
            for (int k = 0; k < NQ; ++k) {  // (apart from the loads, which are all asked for first)
                const int i = threadIdx.x + 256 * k;
                float top = 0.f;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float f = __builtin_fabsf(value(a, x[k].e[j]));
                    top = finite_f(f) ? fmaxf(top, f) : top;
                }
                if (i < 16 * R * DP / 8) atomicMax(&size.top[i / (DP / 8)], __float_as_uint(top));
            }
        lds_barrier();  // what LDS held before has been read, too
        if (threadIdx.x < 16 * R) bits[threadIdx.x] = seen;
        s.c = a.scale * LOG2E;
        bool own = false;
        int up = 0;  // the shared power of two
        if constexpr (Q8) {
            u32 hi = size.top[lane_id() & (16 * R - 1)], lo = hi ? hi : ~0u;
#pragma unroll
            for (int o = 8 * R; o; o >>= 1) {
                const u32 h = (u32)__shfl_xor((int)hi, o, 64), l = (u32)__shfl_xor((int)lo, o, 64);
                hi = h > hi ? h : hi, lo = l < lo ? l : lo;
            }
            hi = __builtin_amdgcn_readfirstlane(hi), lo = __builtin_amdgcn_readfirstlane(lo);
            if (hi) {
                const int eh = __builtin_amdgcn_frexp_expf(__uint_as_float(hi));
                own = eh - __builtin_amdgcn_frexp_expf(__uint_as_float(lo)) > APART || eh > 40 || eh < -40;
                up = 15 - eh;
            }
            if (own) {
                if (threadIdx.x < 16 * R)
                    size.shift[threadIdx.x] = __builtin_amdgcn_frexp_expf(s.c) - up_of(size.top[threadIdx.x]);
                s.c = __builtin_amdgcn_frexp_mantf(s.c);
            } else s.c = __builtin_amdgcn_ldexpf(s.c, -up);
        }
#pragma unroll
        for (int k = 0; k < NQ; ++k) {
            const int i = threadIdx.x + 256 * k;
            if (i < 16 * R * DP / 8) {
                union {
                    T e[8];
                    uint4 w;
                } y;
                if constexpr (Q8) {
                    if (own) up = up_of(size.top[i / (DP / 8)]);
#pragma unroll
                    for (int j = 0; j < 8; ++j) y.e[j] = (T)__builtin_amdgcn_ldexpf(value(a, x[k].e[j]), up);
                } else y.w = x[k].w;
                *(uint4*)(lds + i / (DP / 8) * QLD + i % (DP / 8) * 8) = y.w;
            }
        }
        lds_barrier();
        if constexpr (Q8)
            if (threadIdx.x < 16 * R) size.top[threadIdx.x] = 0;  // (the next unit's maxima come after the joining's barriers)
        s.ql = lds + c * QLD + g * (DP / 4);
        if constexpr (!QLDS)
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int st = 0; st < KS; ++st) s.q[r][st] = *(const V8*)(s.ql + r * 16 * QLD + st * 8);
        return own;
    }
    // the power of two that puts a row's largest element at 2^14 .. 2^15
    static __device__ __forceinline__ int up_of(u32 top) {
        return top ? 15 - __builtin_amdgcn_frexp_expf(__uint_as_float(top)) : 0;
    }
    static __device__ __forceinline__ float value(const TreeArgs& a, u16 e) {
        return a.qtype == NG_BF16 ? __uint_as_float((u32)e << 16) : (float)__builtin_bit_cast(f16, e);
    }

    // the pages of this wave's 32 keys at `base` (any entry of the sequence where a key is past the table)
    static __device__ __forceinline__ Pages pages_of(const TreeArgs& a, const int* tab, int base) {
        const int c = lane_id() & 15, g = lane_id() >> 4, w = a.width - 1;
        Pages p;
        int e = (base + (c >> 2) * 8) >> a.shift;
        p.k = tab[e < w ? e : w];
        e = (base + g * 8) >> a.shift;
        p.v = tab[e < w ? e : w];
        e = (base + (lane_id() & 31)) >> a.shift;
        p.s = Q8 ? tab[e < w ? e : w] : 0;
        return p;
    }

    // A tile's keys and factors, and its values. Both are asked for in the middle of the tile before: the keys into the
    // registers that its keys have just left, the values into the other of two sets.
    static __device__ __forceinline__ void fetch_keys(const TreeArgs& a, int head, int base, const Pages& p, Keys& f) {
        const int c = lane_id() & 15, g = lane_id() >> 4, in = (1 << a.shift) - 1;
        const i64 pk = (u32)p.k < (u64)a.pages ? p.k : 0, ps = (u32)p.s < (u64)a.pages ? p.s : 0;
        const i64 rk = ((pk * a.H + head) << a.shift) + ((base + (c >> 2) * 8) & in) + (c & 3);
        const char* k = (const char*)a.k + rk * (DP * ES) + g * (DP * ES / 4);
        load_words<KW>(k, f.k[0]);
        load_words<KW>(k + 4 * DP * ES, f.k[1]);
        if constexpr (Q8) {
            const i64 rs = ((ps * a.H + head) << a.shift) + ((base + (lane_id() & 31)) & in);
            f.s = (lane_id() < 32 ? a.ks : a.vs)[rs];
        }
    }
    static __device__ __forceinline__ void fetch_values(const TreeArgs& a, int head, int base, const Pages& p, Values& f) {
        const int c = lane_id() & 15, g = lane_id() >> 4, in = (1 << a.shift) - 1;
        f.ok = (u32)p.v < (u64)a.pages;
        const i64 rv = ((((i64)(f.ok ? p.v : 0)) * a.H + head) << a.shift) + ((base + g * 8) & in);
        if constexpr (WILD) f.row = rv;
        const char* v = (const char*)a.v + rv * (DP * ES) + c * (DP * ES / 16);
#pragma unroll
        for (int i = 0; i < 8; ++i) load_words<VW>(v + i * DP * ES, f.v[i]);
    }


    // Values that are not finite (codes of NaN: fp8), in keys that only some rows see: they are 0 in the product (a masked
    // key's P of 0 would make NaN of them) and are added here to the rows that do see them.
    static __device__ __forceinline__ u32 take_out(Values& f) {
        constexpr u32 E = CODES == KV_BF16 ? 0x7F80u : 0x7C00u;
        u32 bad = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int w = 0; w < VW; ++w) {
                if constexpr (CODES == KV_FP8) {  // 0x7F and 0xFF
                    const u32 nan = ((f.v[i][w] & 0x7F7F7F7Fu) + 0x01010101u) >> 7 & 0x01010101u;
                    bad |= (nan ? 1u : 0u) << i;
                    f.v[i][w] &= ~(nan * 0xFFu);
                } else {
                    const bool lo = (f.v[i][w] & E) == E, hi = (f.v[i][w] >> 16 & E) == E;
                    bad |= (lo || hi ? 1u : 0u) << i;
                    f.v[i][w] &= (lo ? 0u : 0xFFFFu) | (hi ? 0u : 0xFFFF0000u);
                }
            }
        return bad;
    }
    // element `at` of the values held, where it is not finite (else anything finite)
    static __device__ __forceinline__ float wild(const TreeArgs& a, i64 at) {
        if constexpr (CODES == KV_FP8) return (((const unsigned char*)a.v)[at] & 0x7F) == 0x7F ? __builtin_nanf("") : 0.f;
        else return (float)((const T*)a.v)[at];
    }
    static __device__ __forceinline__ void put_back(const TreeArgs& a, const Seq& q, int base, const u64* bits, const Values& f,
                                                    u32 bad, const V8 (&p)[R], State& s) {
        const int c = lane_id() & 15, g = lane_id() >> 4;
        for (int from = 0; from < 4; ++from) {
            const i64 first = (i64)__shfl((long long)f.row, from * 16, 64);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (!__any(g == from && (bad >> i & 1))) continue;
                const int j0 = base + from * 8 + i - q.len;
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    const float w = __shfl((float)p[r][i], from * 16 + c, 64);
                    const bool sees = j0 < 0 || (bits[r * 16 + c] >> j0 & 1);
#pragma unroll
                    for (int j = 0; j < NJ; ++j)
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const float x = wild(a, (first + i) * DP + (4 * g + k) * NJ + j);
                            if (sees && !finite_f(x)) s.o[r][j][k] += w * x;
                        }
                }
            }
        }
    }

    struct Run {
        Keys k;
        Values v;
        Pages next;  // the pages of the tile whose loads come next
    };

    // The factors of a tile's keys, computed by one lane each and handed through LDS to the lanes that hold their scores:
    // the score's factor, the logarithm and the inverse of the value scale.
    // True where a value scale is below NONE, or negative: the weights then take fac[3] more.
    static __device__ __forceinline__ bool factors(float scale, bool in, const State& s, float (*fac)[32]) {
        const int key = lane_id() & 31;
        const bool low = in && lane_id() >= 32 && scale < NONE;
        if (lane_id() < 32) fac[0][key] = scale * s.c;
        else {
            float x = low ? fmaxf(__builtin_fabsf(scale), NONE) : scale;
            x = in ? x : 1.f;
            fac[1][key] = __builtin_amdgcn_logf(x);
            fac[2][key] = __builtin_amdgcn_rcpf(x);
            if (__any(low)) fac[3][key] = low && finite_f(scale) ? scale * fac[2][key] : 1.f;  // (-inf: 0 times it is no 0)
        }
        __builtin_amdgcn_wave_barrier();
        return __any(low);
    }

    static __device__ __forceinline__ void scores(Keys& k, const State& s, const Sizes& size, bool own, float (*fac)[32],
                                                  f4 (&sc)[R][2]) {
        const int c = lane_id() & 15, g = lane_id() >> 4;
#pragma unroll
        for (int r = 0; r < R; ++r) sc[r][0] = sc[r][1] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int st = 0; st < KS; ++st) {
            V8 x[R];
#pragma unroll
            for (int r = 0; r < R; ++r) x[r] = QLDS ? *(const V8*)(s.ql + r * 16 * QLD + st * 8) : s.q[QLDS ? 0 : r][st];
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                if constexpr (CODES == KV_INT8) k.k[t][2 * st] ^= 0x80808080u, k.k[t][2 * st + 1] ^= 0x80808080u;
                const V8 e = row_operand<CODES, V8>(k.k[t] + st * (Q8 ? 2 : 4));
#pragma unroll
                for (int r = 0; r < R; ++r) sc[r][t] = mma(e, x[r], sc[r][t]);
            }
        }
        if (Q8 && own) {  // (in this order nothing overflows that the score itself does not)
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    sc[r][i >> 2][i & 3] = __builtin_amdgcn_ldexpf(sc[r][i >> 2][i & 3] * fac[0][g * 8 + i], size.shift[r * 16 + c]) +
                                           fac[1][g * 8 + i];
            return;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float kf = Q8 ? fac[0][g * 8 + i] : s.c, lv = Q8 ? fac[1][g * 8 + i] : 0.f;
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const float x = sc[r][i >> 2][i & 3];
                sc[r][i >> 2][i & 3] = Q8 ? fmaf(x, kf, lv) : x * kf;
            }
        }
    }

    // The running maximum, and the scores as weights, their sum (rv: the inverses of the value scales).
    static __device__ __forceinline__ void weights(f4 (&sc)[R][2], const float (&rv)[8], V8 (&p)[R], State& s) {
        bool grow = false;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float top = sc[r][0][0];
#pragma unroll
            for (int i = 1; i < 8; ++i) top = fmaxf(top, sc[r][i >> 2][i & 3]);
            grow |= top > s.m[r] + SLACK;
        }
        if (__any(grow)) {
#pragma unroll
            for (int r = 0; r < R; ++r) {
                float top = sc[r][0][0];
#pragma unroll
                for (int i = 1; i < 8; ++i) top = fmaxf(top, sc[r][i >> 2][i & 3]);
                const float m = fmaxf(s.m[r], max_quarters(top));
                const float down = s.m[r] == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(s.m[r] - m);
                s.m[r] = m;
                s.l[r] *= down;
#pragma unroll
                for (int j = 0; j < NJ; ++j) s.o[r][j] *= down;
            }
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const float m0 = s.m[r] == -__builtin_inff() ? 0.f : s.m[r] - BIAS;
            float add = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float e = __builtin_amdgcn_exp2f(sc[r][i >> 2][i & 3] - m0);
                if constexpr (Q8) add = fmaf(e, rv[i], add);
                else add += e;
                p[r][i] = (T)e;
            }
            s.l[r] += add;
        }
    }

    // The weights of value rows whose scale is below NONE, or negative.
    static __device__ __forceinline__ void lower(const float (*fac)[32], V8 (&p)[R]) {
        const int g = lane_id() >> 4;
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int r = 0; r < R; ++r) p[r][i] = (T)((float)p[r][i] * fac[3][g * 8 + i]);
    }

    static __device__ __forceinline__ void values(Values& f, const V8 (&p)[R], State& s) {
        if constexpr (CODES == KV_INT8)
#pragma unroll
            for (int i = 0; i < 8; ++i)
#pragma unroll
                for (int k = 0; k < VW; ++k) f.v[i][k] ^= 0x80808080u;
#pragma unroll
        for (int j = 0; j < NJ; j += 2) {
            V8 v0, v1;
            col_operands<CODES, V8, VW>(f.v, j / 2, v0, v1);
#pragma unroll
            for (int r = 0; r < R; ++r) {
                s.o[r][j] = mma(v0, p[r], s.o[r][j]);
                s.o[r][j + 1] = mma(v1, p[r], s.o[r][j + 1]);
            }
        }
    }

    // The first tile's loads.
    static __device__ __forceinline__ void begin(const TreeArgs& a, int b, int head, int base, int stop, Run& w) {
        if (base >= stop) return;
        const int* tab = a.table + (i64)b * a.table_stride;
        w.next = pages_of(a, tab, base);
        fetch_keys(a, head, base, w.next, w.k);
        fetch_values(a, head, base, w.next, w.v);
        w.next = pages_of(a, tab, base + TILE);
    }

    // This wave's keys from base up to stop, a tile of 32 in every TILE; the first one's loads are under way. Only its last
    // tile can hold keys past the cached tokens: the tree and the rest of a tile before it are at most 3 tiles in a row.
    static __device__ __forceinline__ void keys(const TreeArgs& a, int b, int head, const Seq& q, int base, int stop,
                                                const u64* bits, const Sizes& size, bool own, Run& w, State& s,
                                                float (*fac)[32]) {
        if (base >= stop) return;
        const int g = lane_id() >> 4;
        const int* tab = a.table + (i64)b * a.table_stride;
        const int last = base + (stop - 1 - base) / TILE * TILE;
        const int whole = stop < q.len - 31 ? stop : q.len - 31;
        if (base < whole) do {
            f4 sc[R][2];
            V8 p[R];
            float rv[8];
            bool low = false;
            if constexpr (Q8) low = factors(w.k.s, true, s, fac);
            scores(w.k, s, size, own, fac, sc);
#pragma unroll
            for (int i = 0; i < 8; ++i) rv[i] = Q8 ? fac[2][g * 8 + i] : 1.f;
            __builtin_amdgcn_wave_barrier();
            const int nb = base + TILE < last ? base + TILE : last;  // past the last tile: that one again
            const Pages pg = w.next;
            fetch_keys(a, head, nb, pg, w.k);
            w.next = pages_of(a, tab, nb + TILE < last ? nb + TILE : last);
            if (!__all(w.v.ok)) {  // keys without a page: masked, nothing of them enters a product
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    rv[i] = w.v.ok ? rv[i] : 1.f;
#pragma unroll
                    for (int k = 0; k < VW; ++k) w.v.v[i][k] = w.v.ok ? w.v.v[i][k] : 0u;
#pragma unroll
                    for (int r = 0; r < R; ++r) sc[r][i >> 2][i & 3] = w.v.ok ? sc[r][i >> 2][i & 3] : -__builtin_inff();
                }
            }
            weights(sc, rv, p, s);
            if (Q8 && low) lower(fac, p);
            values(w.v, p, s);
            fetch_values(a, head, nb, pg, w.v);
            base += TILE;
        } while (base < whole);
        if (base < stop) any_tile(a, q, base, bits, size, own, w, s, fac);
    }

    // A tile with keys that some row does not see.
    static __device__ __forceinline__ void any_tile(const TreeArgs& a, const Seq& q, int base, const u64* bits, const Sizes& size,
                                                    bool own, Run& w, State& s, float (*fac)[32]) {
        const int c = lane_id() & 15, g = lane_id() >> 4;
        f4 sc[R][2];
        V8 p[R];
        float rv[8];
        bool low = false;
        if constexpr (Q8) low = factors(w.k.s, base + (lane_id() & 31) < q.n, s, fac);
        scores(w.k, s, size, own, fac, sc);
#pragma unroll
        for (int i = 0; i < 8; ++i) rv[i] = Q8 ? fac[2][g * 8 + i] : 1.f;
        __builtin_amdgcn_wave_barrier();
        const int j0 = base + g * 8 - q.len, left = q.n - base - g * 8;  // this lane's first key's place in the tree
        const u32 in = !w.v.ok || left <= 0 ? 0u : left >= 8 ? 0xFFu : (1u << left) - 1;
        const u32 cached = j0 >= 0 ? 0u : j0 <= -8 ? 0xFFu : (1u << -j0) - 1;
#pragma unroll
        for (int i = 0; i < 8; ++i)  // nothing of a key past the end or without a page enters a product
#pragma unroll
            for (int k = 0; k < VW; ++k) w.v.v[i][k] = in >> i & 1 ? w.v.v[i][k] : 0u;
        u32 bad = 0;
        if constexpr (WILD) bad = take_out(w.v);
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const u64 see = bits[r * 16 + c];
            const u32 tree = j0 >= 64 || j0 <= -8 ? 0u : j0 >= 0 ? (u32)(see >> j0) : (u32)(see << -j0);
            const u32 sees = in & (cached | tree);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                sc[r][i >> 2][i & 3] = sees >> i & 1 ? sc[r][i >> 2][i & 3] : -__builtin_inff();
                // a masked key's scale may be NaN: it does not enter the sum (a row that sees it has P of NaN)
                if constexpr (Q8) rv[i] = (sees >> i & 1) | finite_f(rv[i]) ? rv[i] : 1.f;
            }
        }
        weights(sc, rv, p, s);
        if (Q8 && low) lower(fac, p);
        values(w.v, p, s);
        if constexpr (WILD)
            if (__any(bad != 0)) put_back(a, q, base, bits, w.v, bad, p, s);
    }
};

template <int CODES, int DP, int R>
__global__ __launch_bounds__(256, DP <= 128 ? 2 : 1) void tree_k(const TreeArgs a, int blocks) {
    typedef Tree<CODES, DP, R> W;
    constexpr int LD = DP + 4;
    typedef float Lo[16][LD];
    __shared__ __align__(16) char lds[sizeof(Lo) * 4 > 16 * R * W::QLD * 2 ? sizeof(Lo) * 4 : 16 * R * W::QLD * 2];
    Lo* lo = (Lo*)lds;  // the waves' sums at a unit's end; before that the queries
    __shared__ float lm[4][16], ll[4][16];
    __shared__ typename W::Sizes size;
    __shared__ u64 bits[16 * R];
    __shared__ __align__(16) float fac[4][4][32];
    const Line line(a, blocks);
    // neighbouring shares on one XCD (blocks go round the 8 XCDs): units that share keys meet in its L2
    const int a8 = (line.shares + 7) / 8, me = (int)(blockIdx.x % 8) * a8 + (int)blockIdx.x / 8;
    if ((int)blockIdx.x / 8 >= a8 || me >= line.shares) return;
    // (uniform, and the compiler is to know it: a loop that lanes left one by one would keep two sets of sums)
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane_id() & 15, g = lane_id() >> 4, units = a.H * a.groups;
    if constexpr (W::Q8) {
        if (threadIdx.x < 16 * R) size.top[threadIdx.x] = 0;
        lds_barrier();
    }
    int x = me * line.per;
    const int end = line.total - x < line.per ? line.total : x + line.per;
    int before;
    Seq q;
    int b = line.at(a, x, before, q);
    while (x < end) {
        while (x - before >= q.span * units) {
            before += q.span * units;
            q = uniform(seq_of(a, ++b));
        }
        const int unit = (x - before) / q.span, from = x - before - unit * q.span;
        const int to = end - x < q.span - from ? from + (end - x) : q.span;
        const int t0 = from > START ? from - START : 0, t1 = to - START;
        x += to - from;
        if (t1 <= t0) continue;
        const int head = unit / a.groups, row0 = (unit - head * a.groups) * 16 * R;
        const int base = t0 * TILE + wave * 32, stop = t1 * TILE < q.n ? t1 * TILE : q.n;
        typename W::State s;
        typename W::Run run;
        W::begin(a, b, head, base, stop, run);
        const bool own = W::load_q(a, b, head, q, row0, (typename W::T*)lds, size, bits, s);
#pragma unroll
        for (int r = 0; r < R; ++r) {
            s.m[r] = -__builtin_inff(), s.l[r] = 0.f;
#pragma unroll
            for (int j = 0; j < W::NJ; ++j) s.o[r][j] = f4{0.f, 0.f, 0.f, 0.f};
        }
        W::keys(a, b, head, q, base, stop, bits, size, own, run, s, fac[wave]);
        const bool all = t0 == 0 && t1 == q.tiles;
        const i64 slot = 2 * me + (t0 == 0 ? 1 : 0);
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const float l = sum_quarters(s.l[r]);
            __syncthreads();
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < W::NJ; ++j) lo[wave][c][(4 * g + i) * W::NJ + j] = s.o[r][j][i] * W::V_UP;
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
                // a wave without a key that counts: sum and o are 0, or NaN where a NaN was seen
                const float k = lm[w][row] == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(lm[w][row] - m);
                sum = ll[w][row] == 0.f ? sum : fmaf(ll[w][row], k, sum);
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
                    for (int j = 0; j < W::NJ; ++j) o[j] = none ? 0.f : o[j] * inv;
                    put<W::NJ>(a, i * a.dim + d0, a.dim - d0, o);
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
    }
}

// A block per (unit, 16 rows): the shares that hold part of the unit joined.
template <int DP> __global__ __launch_bounds__(256) void tree_join_k(const TreeArgs a, int blocks, int rpb, float bias) {
    constexpr int NJ = DP / 16;
    const int sub = rpb / 16, u = blockIdx.x / sub, r16 = (int)(blockIdx.x - u * sub) * 16;
    const int per = a.H * a.groups, b = u / per, unit = u - b * per;
    const Line line(a, blocks);
    Seq q;
    const int x0 = line.before(a, b, q) + unit * q.span;
    const int i0 = (x0 + START) / line.per, i1 = (x0 + q.span - 1) / line.per;  // the shares of its first and last tile
    if (i0 == i1) return;
    const int head = unit / a.groups, row0 = (unit - head * a.groups) * rpb;
    const int row = threadIdx.x >> 4, d0 = (threadIdx.x & 15) * NJ;
    const int at = row0 + r16 + row, t = at / a.G, h = at - t * a.G;
    if (t >= a.T) return;
    float m = -__builtin_inff(), sum = 0.f, o[NJ];
#pragma unroll
    for (int j = 0; j < NJ; ++j) o[j] = 0.f;
    for (int i = i0; i <= i1; ++i) {
        const i64 prow = (i64)(2 * i + (i == i0 ? 1 : 0)) * rpb + r16 + row;
        const float pm = a.pm[prow], pl = a.pl[prow];
        const float n = fmaxf(m, pm);
        const float ko = m == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(m - n);
        const float kp = pm == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(pm - n);
        sum = (sum == 0.f ? 0.f : sum * ko) + (pl == 0.f ? 0.f : pl * kp);
#pragma unroll
        for (int j = 0; j < NJ; ++j) o[j] = o[j] * ko + a.po[prow * DP + d0 + j] * kp;
        m = n;
    }
    const i64 i = ((i64)b * a.T + t) * a.H * a.G + head * a.G + h;
    const bool none = sum == 0.f || t >= q.w;
    const float inv = none ? 0.f : 1.f / sum;
#pragma unroll
    for (int j = 0; j < NJ; ++j) o[j] = none ? 0.f : o[j] * inv;
    put<NJ>(a, i * a.dim + d0, a.dim - d0, o);
    if (a.lse && (threadIdx.x & 15) == 0) a.lse[i] = none ? -__builtin_inff() : LN2 * (m - bias + __builtin_amdgcn_logf(sum));
}

// ------------------------------------------------------------------------------------------------------- the launches

template <int CODES, int DP, int R> static int tree_run(const TreeArgs& a, const TreePlan& p, hipStream_t st) {
    tree_k<CODES, DP, R><<<p.blocks, 256, 0, st>>>(a, p.blocks);
    int rc = (int)hipGetLastError();
    if (rc || !p.join) return rc;
    tree_join_k<DP><<<a.B * a.H * a.groups * R, 256, 0, st>>>(a, p.blocks, 16 * R, Tree<CODES, DP, R>::BIAS);
    return (int)hipGetLastError();
}

template <int CODES, int DP> static int tree_rows(const TreeArgs& a, const TreePlan& p, hipStream_t st) {
    if (p.rpb == 16) return tree_run<CODES, DP, 1>(a, p, st);
    return p.rpb == 32 ? tree_run<CODES, DP, 2>(a, p, st) : -1;
}

template <int CODES> int tree_codes(const TreeArgs& a, const TreePlan& p, hipStream_t st) {
    switch (p.dp) {
        case 64: return tree_rows<CODES, 64>(a, p, st);
        case 128: return tree_rows<CODES, 128>(a, p, st);
        case 192: return tree_rows<CODES, 192>(a, p, st);
        default: return tree_rows<CODES, 256>(a, p, st);
    }
}
