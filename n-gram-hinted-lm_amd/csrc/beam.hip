// A beam search's step: the K best candidates of a sequence's W beams, and the states of the beams they come from.
//
//   total(w, v) = score[w] + logit[w, v] - log sum_u exp logit[w, u];   a finished beam: (pad, score[w]) and nothing else
//   rank        = total / max(length, 1)^alpha,  length = length[w] + 1 (a finished beam: length[w])
//   the K largest ranks, ties to the lower beam, then the larger logit, then the lower token
//
// A rank that is NaN or -inf is none; where fewer than K are left, the lowest (beam, token) of the others follow, with total
// -inf.
//
// One pass over the logits: a block takes a chunk of a row into registers, sums its exponentials and keeps its K largest
// logits (within a beam candidates order as their logits do). A block a sequence then joins the chunks' sums and compares the
// candidates; where there are many, a block a row first leaves K of them.
//
// Precision. Candidates of different beams lie close to each other, so what decides between them is held in 64 bits: sums
// over more than a thread's 32 elements, the logarithm, totals and ranks (quotients, as they are defined: by the mean of its
// tokens a beam of -n over n of them ranks -1 for every n, where a product with exp(-log n) is an ulp off for some, and beams of
// equal ranks come in their order).
// An exponential is a 32-bit one: its argument's rounding and the instruction's are off by 2^-20 of a term, and average out over
// a row's terms. (Putting each argument's rounding back took 5 more operations an element: 20.5 us a chunk's pass against 17.3
// for 64 x 8 rows of 50257.) One part does not average out: log2(e) as a float is 1.34e-8 of itself low, so a term is (m - v)
// 1.34e-8 of itself large, m the row's largest logit, and a log-sum by 1.34e-8 times the mean of m - v under the softmax's
// weights. That is no more than their entropy, ln V at most: 2^-22 for any V.
//
// Measured (in a trace, us): 64 x 8 rows of 50257 bfloat16 logits, a fifth of the beams finished (41 MB): chunks 17.7 (2.3
// TB/s), joining 8.2; 8 x 32 rows of 100003 float32 ones, a tenth finished, 64 kept (92 MB): chunks 29 (3.2 TB/s), rows 7.2,
// joining 9.3; one sequence of 4 beams: 6.0 and 6.5. The chunks' pass issues vector instructions in 55 and 61 % of its time (some
// 500 and 900 a wave of 32 elements a lane, by counters), and its waves spend 54 and 46 % of theirs waiting, for the loads and at
// the halvings' barriers; the joining is one block's chain of these. Finding a threshold without halvings has not been tried.
#include "choose.h"
#include "vals.h"

#define MOST 128    // beams, and candidates kept
#define ROOM 1024   // candidates that are compared with each other
#define TOKEN_BITS 25

struct BeamArgs {
    const void* logits;  // [B, W, V], strides of sequences and beams in elements
    i64 sb, sw;
    const float* scores;           // [B, W]
    const void* lengths;           // int32 or int64 (lsize 4, 8) [B, W], or NULL
    const unsigned char* finished; // [B, W] or NULL
    float* out_scores;             // [B, K], as are
    i64 *parents, *tokens;
    unsigned char* out_finished;  // NULL: not wanted
    i64* out_lengths;
    u64* part;      // [B * W, chunks, K]: logit's key << 32 | ~token, descending; 0: nothing
    float* top;     // [B * W, chunks]
    double* sum;    // [B * W, chunks]
    int B, W, V, K, chunks, lsize;
    int end, pad;   // -1: none
    i64 row0;       // the rows before this launch's first
    double alpha;
};

__device__ __forceinline__ bool ended(const BeamArgs& a, i64 row) { return a.finished && a.finished[row]; }
__device__ __forceinline__ i64 length_of(const BeamArgs& a, i64 row) {
    return a.lsize == 4 ? (i64)((const int*)a.lengths)[row] : ((const i64*)a.lengths)[row];
}

// Where a threshold that leaves K at least is fine enough: each halving costs as much as ranking some ten keys more.
__device__ __forceinline__ int few(int K) { return K + K / 2 + 12; }

// The n keys of list, all different, in order: the K_ largest to out, 0 behind the last. list has room for 3 more.
__device__ __forceinline__ void write_ranked(u64* list, int n, int K_, u64* out, int threads) {
    if (threadIdx.x < 3) list[n + threadIdx.x] = 0;
    __syncthreads();
    for (int i0 = 0; i0 < n; i0 += threads / 4) {  // four lanes a key
        const int i = i0 + threadIdx.x / 4;
        const u64 mine = i < n ? list[i] : 0;
        int r = 0;
        for (int j = (threadIdx.x & 3) * 4; j < n; j += 16)
            r += (list[j] > mine) + (list[j + 1] > mine) + (list[j + 2] > mine) + (list[j + 3] > mine);
        r += __shfl_xor(r, 1, WAVE);
        r += __shfl_xor(r, 2, WAVE);
        if (i < n && r < K_ && (threadIdx.x & 3) == 0) out[r] = mine;
    }
    for (int i = n + threadIdx.x; i < K_; i += threads) out[i] = 0;
}

// A thread's E logits as they are, 16 bytes in every 256 lanes'; -inf behind the last. whole: the chunk ends before V.
template <typename T, int E> struct Logits {
    static constexpr int N = 16 / (int)sizeof(T), P = E / N;
    Pack<T, N> k[P];
    __device__ __forceinline__ void load(const T* x, int from, int V, bool whole) {
        if (whole) {
#pragma unroll
            for (int p = 0; p < P; ++p) k[p].load(x + from + p * 256 * N);
            return;
        }
#pragma unroll
        for (int p = 0; p < P; ++p) {
            const int i = from + p * 256 * N;
            if (i + N <= V) k[p].load(x + i);
            else
#pragma unroll
                for (int j = 0; j < N; ++j) k[p].v[j] = i + j < V ? x[i + j] : (T)-__builtin_inff();
        }
    }
    __device__ __forceinline__ float at(int p, int j) const { return (float)k[p].v[j]; }
};

// More logits reach the threshold t than are compared with each other: many are equal, or most of them in few threads. The
// threshold that leaves K, and of the logits equal to it the lowest tokens. (The logits are loaded again for each count:
// registers held for this would cost every block a third of its waves.)
template <typename T, int E>
__device__ __forceinline__ void crowded(const T* x, int from, const BeamArgs& a, u32 t, u32 hi, Count<4>& count, u64* list,
                                        int* fill) {
    constexpr int N = 16 / (int)sizeof(T);
    auto each = [&](auto f) {
#pragma unroll 1
        for (int p = 0; p < E / N; ++p)
#pragma unroll 1
            for (int j = 0; j < N; ++j) {
                const int i = from + p * 256 * N + j;
                f(i < a.V ? key_of((float)x[i]) : 0u, (u32)i);
            }
    };
    auto at_least = [&](u32 least, u32 last) {  // keys above `least`, and those equal to it of tokens up to `last`
        int n = 0;
        each([&](u32 k, u32 i) { n += __popcll(__ballot(k > least || (k == least && i <= last))); });
        return count.sum(n);
    };
    u32 up = hi;
    while (t < up) {  // the largest t that K reach
        const u32 mid = t + (up - t) / 2 + 1;
        if (at_least(mid, ~0u) >= a.K) t = mid;
        else up = mid - 1;
    }
    u32 l = 0, h = (u32)a.V - 1;  // the lowest token up to which enough are equal
    while (l < h) {
        const u32 mid = l + (h - l) / 2;
        if (at_least(t, mid) >= a.K) h = mid;
        else l = mid + 1;
    }
    if (threadIdx.x == 0) *fill = 0;
    __syncthreads();
    each([&](u32 k, u32 i) {
        if (k > t || (k == t && i <= l)) list[atomicAdd(fill, 1)] = (u64)k << 32 | (u32)~i;
    });
    __syncthreads();
}

// A block per (row, chunk of 256 E logits): in registers, so that sums, threshold and choice read memory once. (64 registers:
// eight blocks a CU, whose loads and halvings cover each other.)
template <typename T, int E> __global__ __launch_bounds__(256, 8) void beam_part_k(const BeamArgs a) {
    constexpr int N = 16 / (int)sizeof(T), P = E / N;
    __shared__ u64 list[ROOM + 3];
    __shared__ int counts[2][4];
    __shared__ u32 most[4], least[4];
    __shared__ double sums[4];
    __shared__ int fill;
    const u32 row = blockIdx.x / (u32)a.chunks, b = row / (u32)a.W;
    const int chunk = (int)(blockIdx.x - row * a.chunks), tid = threadIdx.x, wave = tid >> 6;
    if (ended(a, row)) return;
    const T* __restrict__ x = (const T*)a.logits + b * a.sb + (i64)(row - b * a.W) * a.sw;
    const int from = chunk * 256 * E + tid * N;
    Logits<T, E> v;
    v.load(x, from, a.V, (i64)(chunk + 1) * 256 * E <= a.V);
    float tops[P], top = -__builtin_inff();  // of each load, and all (NaN passed over)
#pragma unroll
    for (int p = 0; p < P; ++p) {
        tops[p] = v.at(p, 0);
#pragma unroll
        for (int j = 1; j < N; ++j) tops[p] = fmaxf(tops[p], v.at(p, j));
        top = fmaxf(top, tops[p]);
    }
    const u32 mine[1] = {key_of(top)};
    const u32 wm = max_wave(mine[0]), wl = min_wave(mine[0]);
    if (lane_id() == 0) most[wave] = wm, least[wave] = wl;
    if (tid == 0) fill = 0;
    lds_barrier();
    u32 hi = most[0], lo = least[0];
#pragma unroll
    for (int w = 1; w < 4; ++w) hi = most[w] > hi ? most[w] : hi, lo = least[w] < lo ? least[w] : lo;
    const float m = hi ? of_key(hi) : 0.f;  // (nothing above -inf: each term is 0, or NaN)
    // 2^(L v + c) with c = -L m rounded: one operation an argument; how far c is off is put back below, once for all terms.
    // (Where L m is large that is no small correction: the arguments are L (v - m) then.)
    const float L = 1.44269504f, c = -L * m;
    const bool near = __builtin_fabsf(m) < 4096.f;
    float s = 0.f;
    if (near)
#pragma unroll
        for (int e = 0; e < E; ++e) s += __builtin_amdgcn_exp2f(fmaf(v.at(e / N, e % N), L, c));
    else
#pragma unroll
        for (int e = 0; e < E; ++e) s += __builtin_amdgcn_exp2f((v.at(e / N, e % N) - m) * L);
    double sum = s;
#pragma unroll
    for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o, WAVE);
    if (lane_id() == 0) sums[wave] = sum;
    // the threads' largest give a threshold that K logits at least reach
    Count<4> count(counts);
    int n = 256;
    const u32 lowest = 0x00800000u;  // the key of the lowest number: where there are fewer than K, all are taken
    u32 t = count.threshold(mine, lo > lowest ? lo : lowest, hi, a.K, few(a.K), n);
    const float least_v = of_key(t);
#pragma unroll
    for (int p = 0; p < P; ++p)
        if (tops[p] >= least_v)
#pragma unroll
            for (int j = 0; j < N; ++j)
                if (v.at(p, j) >= least_v) {
                    const u32 token = from + p * 256 * N + j;
                    const int at = atomicAdd(&fill, 1);
                    if (at < ROOM) list[at] = (u64)key_of(v.at(p, j)) << 32 | (u32)~token;
                }
    __syncthreads();
    if (fill > ROOM) crowded<T, E>(x, from, a, t, hi, count, list, &fill);
    const i64 at = blockIdx.x;
    write_ranked(list, fill, a.K, a.part + at * a.K, 256);
    if (tid == 0) {
        const double off = near ? 0.69314718055994531 * ((double)L * m + (double)c) : 0.;  // below 2^-11: exp by its series
        a.top[at] = hi ? m : -__builtin_inff();
        a.sum[at] = (sums[0] + sums[1] + sums[2] + sums[3]) * (1. - off * (1. - off * (0.5 - off / 6.)));
    }
}

// The chunks' sums of one row, by LANES lanes of a wave: the row's largest logit and sum of exponentials beside it (NaN or
// infinite, or a sum of 0: the row has no candidates).
template <int LANES> __device__ __forceinline__ void row_sum(const BeamArgs& a, i64 row, float& m, double& s) {
    const int l = lane_id() & (LANES - 1);
    const float* top = a.top + row * a.chunks;
    const double* sum = a.sum + row * a.chunks;
    m = -__builtin_inff(), s = 0;
    for (int c = l; c < a.chunks; c += LANES) {  // (a running maximum: one pass over the loads)
        const float t = top[c];
        const double x = sum[c];
        const float n = fmaxf(m, t);
        if (n == -__builtin_inff()) s += x;
        else if (n == m) s += t == -__builtin_inff() ? x : x * exp((double)t - (double)m);
        else s = (m == -__builtin_inff() ? s : s * exp((double)m - (double)n)) + x, m = n;
    }
    float all = m;
#pragma unroll
    for (int o = LANES / 2; o; o >>= 1) all = fmaxf(all, __shfl_xor(all, o, WAVE));
    if (m != -__builtin_inff() && m != all) s *= exp((double)m - (double)all);
    m = all;
#pragma unroll
    for (int o = LANES / 2; o; o >>= 1) s += __shfl_xor(s, o, WAVE);
}

// The block's largest of x and of y: y the last of a list of K, which as many at least reach (1: no list is full).
template <int NW> __device__ __forceinline__ void ends(u64 x, u64 y, u64 (&lds)[2][NW], u64& hi, u64& lo) {
    x = max_wave(x), y = max_wave(y);
    if (lane_id() == 0) lds[0][threadIdx.x >> 6] = x, lds[1][threadIdx.x >> 6] = y;
    lds_barrier();
    hi = lds[0][0], lo = lds[1][0];
#pragma unroll
    for (int w = 1; w < NW; ++w) hi = lds[0][w] > hi ? lds[0][w] : hi, lo = lds[1][w] > lo ? lds[1][w] : lo;
    if (!lo) lo = 1;
}

// A block a row: its chunks' lists to one of K, and its log sum exp.
template <int NW, int E> __global__ __launch_bounds__(NW * 64) void beam_row_k(const BeamArgs a, u64* part, double* lses) {
    constexpr int NT = NW * 64;
    __shared__ u64 list[ROOM + 3];
    __shared__ int counts[2][NW];
    __shared__ u64 most[2][NW];
    __shared__ int fill;
    const i64 row = blockIdx.x;
    if (ended(a, row)) return;
    const int have = a.chunks * a.K;
    u64 key[E], mine = 0, full = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int i = e * NT + threadIdx.x;
        key[e] = i < have ? a.part[row * have + i] : 0;
        mine = key[e] > mine ? key[e] : mine;
        if ((u32)i % (u32)a.K == (u32)a.K - 1) full = key[e] > full ? key[e] : full;
    }
    u64 lo, hi;
    ends(mine, full, most, hi, lo);
    if (threadIdx.x == 0) fill = 0;
    lds_barrier();
    Count<NW> count(counts);
    int n = count.at_least(key, lo);  // (the keys are all different: a threshold leaves as few as wanted)
    const u64 t = count.threshold(key, lo, hi, a.K, few(a.K), n);
#pragma unroll
    for (int e = 0; e < E; ++e)
        if (key[e] >= t && key[e]) list[atomicAdd(&fill, 1)] = key[e];
    __syncthreads();
    write_ranked(list, fill, a.K, part + row * a.K, NT);
    if (threadIdx.x < 64) {
        float m;
        double s;
        row_sum<64>(a, row, m, s);
        if (threadIdx.x == 0) lses[row] = log(s) + (double)m;
    }
}

// A block a sequence, which holds E candidates a thread. a.top NULL: part holds a list a row and sum its log sum exp.
template <int NW, int E> __global__ __launch_bounds__(NW * 64) void beam_join_k(const BeamArgs a) {
    constexpr int NT = NW * 64;
    __shared__ double lses[MOST], scores[MOST], norms[MOST];
    __shared__ int done[MOST];
    __shared__ u64 most[2][NW];
    __shared__ ulonglong2 list[ROOM + 3];  // a candidate's two words
    __shared__ int counts[2][NW];
    __shared__ int fill;
    const i64 b = blockIdx.x;
    const int tid = threadIdx.x;
    const int per = a.chunks * a.K, have = a.W * per;
    constexpr bool HOLD = E <= 4;  // the candidates are kept beside their ranks, else loaded again where they are chosen
    u64 held[HOLD ? E : 1];
    if constexpr (HOLD)
#pragma unroll
        for (int e = 0; e < E; ++e) held[e] = e * NT + tid < have ? a.part[b * have + e * NT + tid] : 0;
    for (int w = tid / 16; w < a.W; w += NT / 16) {  // 16 lanes a beam
        const i64 row = b * a.W + w;
        const bool end = ended(a, row);
        const i64 len = (a.lengths ? length_of(a, row) : 0) + (end ? 0 : 1);
        const float score = a.scores[row];
        double lse = 0.;
        if (!a.top) lse = end ? 0. : a.sum[row];
        else if (!end) {
            float m;
            row_sum<16>(a, row, m, lse);
            lse = log(lse) + (double)m;
        }
        if ((lane_id() & 15) == 0) {
            lses[w] = lse, scores[w] = score, done[w] = end;
            const double n = len > 1 ? (double)len : 1.;
            norms[w] = a.alpha == 0. ? 1. : a.alpha == 1. ? n : pow(n, a.alpha);  // (pow(n, 1) is an ulp off n for some n)
        }
    }
    if (tid == 0) fill = 0;
    __syncthreads();
    // candidates: the rows' lists, then one of each finished beam. A key's first word is its rank, its second the beam
    // (lower first), the logit and the token (lower first).
    u64 key[E], mine = 0, full = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int i = e * NT + tid;
        key[e] = 0;
        if (i < have) {
            const int w = (int)((u32)i / (u32)per);
            const u64 c = done[w] ? 0ull : HOLD ? held[HOLD ? e : 0] : a.part[b * have + i];
            if (c) key[e] = key_of((scores[w] + ((double)of_key((u32)(c >> 32)) - lses[w])) / norms[w]);
            if (done[w] && i == w * per) key[e] = key_of(scores[w] / norms[w]);
            if ((u32)i % (u32)a.K == (u32)a.K - 1) full = key[e] > full ? key[e] : full;
        }
        mine = key[e] > mine ? key[e] : mine;
    }
    u64 lo, hi;
    ends(mine, full, most, hi, lo);
    Count<NW> count(counts);
    int n = count.at_least(key, lo);
    const u64 t = count.threshold(key, lo, hi, a.K, few(a.K), n);
    auto second = [&](int e) {
        const int i = e * NT + tid, w = (int)((u32)i / (u32)per);
        const u64 c = done[w] ? 0xFFFFFFFFull << 32 | (u32)~a.pad : HOLD ? held[HOLD ? e : 0] : a.part[b * have + i];
        return (u64)(MOST - 1 - w) << 57 | c >> 32 << TOKEN_BITS | ((u32)c & ((1u << TOKEN_BITS) - 1));
    };
    u64 t2 = 0;  // of the keys equal to t, those whose second word is this or more
    if (n > ROOM) {
        const int above = t == hi ? 0 : count.at_least(key, t + 1);
        u64 lo = 0, up = ~0ull;
        while (lo < up) {  // the largest t2 that leaves enough
            const u64 mid = lo + (up - lo) / 2 + 1;
            int k = 0;
#pragma unroll
            for (int e = 0; e < E; ++e) k += __popcll(__ballot(key[e] == t && second(e) >= mid));
            if (above + count.sum(k) >= a.K) lo = mid;
            else up = mid - 1;
        }
        t2 = lo;
    }
#pragma unroll
    for (int e = 0; e < E; ++e)
        if (key[e] >= t && key[e]) {
            const u64 s = second(e);
            if (key[e] > t || s >= t2) {
                const int at = atomicAdd(&fill, 1);
                list[at] = make_ulonglong2(key[e], s);
            }
        }
    __syncthreads();
    n = fill;
    if (tid < 3) list[n + tid] = make_ulonglong2(0, 0);
    __syncthreads();
    auto put = [&](int r, int w, int token, float score) {
        const i64 o = b * a.K + r;
        a.out_scores[o] = score, a.parents[o] = a.row0 + b * a.W + w, a.tokens[o] = token;
        if (a.out_finished) a.out_finished[o] = done[w] || token == a.end;
        if (a.out_lengths) a.out_lengths[o] = length_of(a, b * a.W + w) + (done[w] ? 0 : 1);
    };
    for (int i0 = 0; i0 < n; i0 += NT / 4) {  // four lanes a candidate
        const int i = i0 + tid / 4;
        const u64 k = i < n ? list[i].x : 0, s = i < n ? list[i].y : 0;
        int r = 0;
        for (int j = (tid & 3) * 4; j < n; j += 16)
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const ulonglong2 x = list[j + u];
                r += x.x > k || (x.x == k && x.y > s);
            }
        r += __shfl_xor(r, 1, WAVE);
        r += __shfl_xor(r, 2, WAVE);
        if (i >= n || r >= a.K || (tid & 3)) continue;
        const int w = MOST - 1 - (int)(s >> 57), token = (1 << TOKEN_BITS) - 1 - (int)(s & ((1u << TOKEN_BITS) - 1));
        put(r, w, token, (float)(done[w] ? scores[w] : scores[w] + ((double)of_key((u32)(s >> TOKEN_BITS)) - lses[w])));
    }
    if (n >= a.K) return;
    // too few candidates: of the first 2 K (beam, token) places K - n at least are none of them
    __shared__ unsigned char open[2 * MOST];
    for (int i = tid; i < 2 * a.K; i += NT) {
        const int w = i / a.V, v = i - w * a.V;
        bool o = w < a.W;
        for (int j = 0; j < n; ++j)
            o &= MOST - 1 - (int)(list[j].y >> 57) != w || (1 << TOKEN_BITS) - 1 - (int)(list[j].y & ((1u << TOKEN_BITS) - 1)) != v;
        open[i] = o;
    }
    __syncthreads();
    for (int i = tid; i < 2 * a.K; i += NT) {
        if (!open[i]) continue;
        int r = n;
        for (int j = 0; j < i; ++j) r += open[j];
        if (r < a.K) put(r, i / a.V, i % a.V, -__builtin_inff());
    }
}

// ------------------------------------------------------------------------------------------------------------ the host

struct BeamPlan {
    int E, chunks;
    bool merge;
    i64 nb;                                    // sequences a launch
    i64 part, top, sum, rows, row_sum, bytes;  // offsets in the workspace
};

// A launch has fewer than 2^32 threads: as many sequences at a time as leave blocks of 1024 fewer than that.
#define MOST_BLOCKS (((i64)1 << 22) - 1)

// A chunk is 8192 logits, or fewer where that leaves less than 1024 blocks (4 a CU): 4 rows of 50257 take 5.9 us and 6.5 of
// joining in chunks of 2048, 7.5 and 5.4 in chunks of 8192; 256 rows of 100003 34 us in chunks of 4096, 29 in chunks of 8192.
// Not so few that a row's candidates outgrow the 16384 that the joining blocks hold. More than 4096 candidates a sequence go
// through a block a row first (6656 of 16 rows: 6.0 and 7.0 us against 16.0 at once; 3328: 5.5 and 6.5 against 11.6).
static bool beam_plan(i64 B, i64 W, i64 V, i64 K, BeamPlan& p) {
    if (B < 0 || W < 1 || W > MOST || K < 1 || K > MOST || V < 1 || V > 1 << TOKEN_BITS || K > W * V || B > 1 << 24) return false;
    p.E = 32;
    while (p.E > 8 && B * W * ((V + 256 * p.E - 1) / (256 * p.E)) < 1024 &&
           (V + 128 * p.E - 1) / (128 * p.E) * K <= 16384)
        p.E /= 2;
    const i64 chunks = (V + 256 * p.E - 1) / (256 * p.E);
    if (chunks * K > 16384 || B * W * chunks >= (i64)1 << 31) return false;
    p.chunks = (int)chunks;
    p.merge = W * chunks * K > 4096;
    p.nb = B < MOST_BLOCKS / (W * chunks) ? B : MOST_BLOCKS / (W * chunks);
    const i64 n = p.nb * W * chunks;
    p.part = 0;
    p.sum = p.part + n * K * 8;
    p.rows = p.sum + n * 8;
    p.row_sum = p.rows + (p.merge ? p.nb * W * K * 8 : 0);
    p.top = p.row_sum + (p.merge ? p.nb * W * 8 : 0);
    p.bytes = p.top + n * 4;
    return true;
}

extern "C" i64 ng_beam_work(i64 B, i64 W, i64 V, i64 K) {
    BeamPlan p;
    return beam_plan(B, W, V, K, p) ? p.bytes : -1;
}

template <typename T> static void beam_part(const BeamArgs& a, int E, hipStream_t st) {
    const unsigned grid = (unsigned)(a.B * a.W * a.chunks);
    if (E == 32) beam_part_k<T, 32><<<grid, 256, 0, st>>>(a);
    else if (E == 16) beam_part_k<T, 16><<<grid, 256, 0, st>>>(a);
    else beam_part_k<T, 8><<<grid, 256, 0, st>>>(a);
}

static int beam_launch(BeamArgs a, const BeamPlan& p, int dtype, char* w, hipStream_t st) {
    switch (dtype) {
        case NG_F32: beam_part<float>(a, p.E, st); break;
        case NG_BF16: beam_part<b16>(a, p.E, st); break;
        default: beam_part<f16>(a, p.E, st);
    }
    int rc = (int)hipGetLastError();
    if (rc) return rc;
    if (p.merge) {
        u64* rows = (u64*)(w + p.rows);
        double* lses = (double*)(w + p.row_sum);
        const unsigned grid = (unsigned)(a.B * a.W);
        if (a.chunks * a.K <= 1024) beam_row_k<4, 4><<<grid, 256, 0, st>>>(a, rows, lses);
        else beam_row_k<16, 16><<<grid, 1024, 0, st>>>(a, rows, lses);
        if ((rc = (int)hipGetLastError())) return rc;
        a.part = rows, a.top = nullptr, a.sum = lses, a.chunks = 1;
    }
    const int have = a.W * a.chunks * a.K;
    if (have <= 1024) beam_join_k<4, 4><<<a.B, 256, 0, st>>>(a);
    else if (have <= 2048) beam_join_k<8, 4><<<a.B, 512, 0, st>>>(a);
    else if (have <= 4096) beam_join_k<16, 4><<<a.B, 1024, 0, st>>>(a);
    else beam_join_k<16, 16><<<a.B, 1024, 0, st>>>(a);
    return (int)hipGetLastError();
}

extern "C" int ng_beam_step_alpha64(const void* logits, i64 sb, i64 sw, int dtype, const float* scores, const void* lengths,
                                    int lsize, const void* finished, int B, int W, int V, int K, int end, int pad,
                                    double alpha, float* out_scores, i64* parents, i64* tokens, void* out_finished,
                                    i64* out_lengths, void* work, void* stream) {
    BeamPlan p;
    if (!beam_plan(B, W, V, K, p) || dtype < NG_F32 || dtype > NG_F16 || !(alpha >= 0. && alpha < __builtin_inf()) ||
        (out_lengths && !lengths) || (alpha != 0. && !lengths) || (lengths && lsize != 4 && lsize != 8) ||
        (finished && (pad < 0 || pad >= V)))
        return -1;
    hipStream_t st = (hipStream_t)stream;
    for (i64 b0 = 0; b0 < B; b0 += p.nb) {
        BeamArgs a;
        const i64 r0 = b0 * W, o = b0 * K;
        char* w = (char*)work;
        a.logits = (const char*)logits + b0 * sb * (dtype == NG_F32 ? 4 : 2), a.sb = sb, a.sw = sw, a.scores = scores + r0;
        a.lengths = lengths ? (const char*)lengths + r0 * lsize : nullptr, a.lsize = lsize;
        a.finished = finished ? (const unsigned char*)finished + r0 : nullptr;
        a.out_scores = out_scores + o, a.parents = parents + o, a.tokens = tokens + o;
        a.out_finished = out_finished ? (unsigned char*)out_finished + o : nullptr;
        a.out_lengths = out_lengths ? out_lengths + o : nullptr;
        a.part = (u64*)(w + p.part), a.top = (float*)(w + p.top), a.sum = (double*)(w + p.sum);
        a.B = (int)(B - b0 < p.nb ? B - b0 : p.nb), a.W = W, a.V = V, a.K = K, a.chunks = p.chunks, a.end = end, a.pad = pad;
        a.alpha = alpha, a.row0 = r0;
        const int rc = beam_launch(a, p, dtype, w, st);
        if (rc) return rc;
    }
    return 0;
}

extern "C" int ng_beam_step(const void* logits, i64 sb, i64 sw, int dtype, const float* scores, const void* lengths,
                            int lsize, const void* finished, int B, int W, int V, int K, int end, int pad, float alpha,
                            float* out_scores, i64* parents, i64* tokens, void* out_finished, i64* out_lengths, void* work,
                            void* stream) {
    return ng_beam_step_alpha64(logits, sb, sw, dtype, scores, lengths, lsize, finished, B, W, V, K, end, pad, alpha, out_scores,
                                parents, tokens, out_finished, out_lengths, work, stream);
}

// Rows copied in a given order: out[i] = src[from[i]], zeros where that is no row. U: the unit of a copy; a block takes 256
// units of a row at a time. Memory bounds it: 512 rows of 256 KiB, 134 MB written, 35 us.
template <typename U> __global__ __launch_bounds__(256) void gather_rows_k(const char* __restrict__ src, i64 stride, i64 rows,
                                                                           const i64* __restrict__ from, i64 units, int parts,
                                                                           char* __restrict__ out) {
    const i64 i = blockIdx.x / parts, r = from[i];
    const U* s = (const U*)(src + r * stride);
    U* o = (U*)(out + i * units * (i64)sizeof(U));
    const bool is = (u64)r < (u64)rows;
    for (i64 j = (blockIdx.x % parts) * 256 + threadIdx.x; j < units; j += (i64)parts * 256) {
        U x = {};
        if (is) x = s[j];
        __builtin_nontemporal_store(x, o + j);
    }
}

extern "C" int ng_gather_rows(const void* src, i64 stride, i64 rows, i64 bytes, const i64* from, i64 n, void* out,
                              void* stream) {
    if (n < 0 || rows < 0 || bytes < 0 || n >= (i64)1 << 31) return -1;
    if (n == 0 || bytes == 0) return 0;
    const u64 all = (u64)src | (u64)stride | (u64)bytes | (u64)out;
    const int size = all % 16 == 0 ? 16 : all % 4 == 0 ? 4 : all % 2 == 0 ? 2 : 1;
    const i64 units = bytes / size;
    // enough blocks for the card's 256 CUs 8 times over, each of at least 1024 units
    i64 parts = (units + 1023) / 1024;
    const i64 most = (16384 + n - 1) / n;
    parts = parts < most ? parts : most;
    hipStream_t st = (hipStream_t)stream;
    const i64 step = MOST_BLOCKS / parts;  // (parts is 16384 at most)
    for (i64 i0 = 0; i0 < n; i0 += step, from += step, out = (char*)out + step * bytes) {
        const unsigned grid = (unsigned)(parts * (n - i0 < step ? n - i0 : step));
#define GATHER(U) gather_rows_k<U><<<grid, 256, 0, st>>>((const char*)src, stride, rows, from, units, (int)parts, (char*)out)
        typedef u32 words __attribute__((ext_vector_type(4)));
        if (size == 16) GATHER(words);
        else if (size == 4) GATHER(u32);
        else if (size == 2) GATHER(u16);
        else GATHER(unsigned char);
#undef GATHER
        const int rc = (int)hipGetLastError();
        if (rc) return rc;
    }
    return 0;
}
