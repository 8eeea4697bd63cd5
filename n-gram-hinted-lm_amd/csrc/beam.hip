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
// over more than a thread's 32 elements, the logarithm, totals and ranks. An exponential is a 32-bit one whose argument's
// rounding is put back (its error is the instruction's 2^-23 of itself, and averages out over a row).
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
    double alpha;
};

__device__ __forceinline__ bool ended(const BeamArgs& a, i64 row) { return a.finished && a.finished[row]; }
__device__ __forceinline__ i64 length_of(const BeamArgs& a, i64 row) {
    return a.lsize == 4 ? (i64)((const int*)a.lengths)[row] : ((const i64*)a.lengths)[row];
}

// exp(d) for d <= 0 or NaN
__device__ __forceinline__ float exp_of(float d) {
    d = d < -200.f ? -200.f : d;
    const float t = d * 1.44269504f, r = fmaf(d, 1.44269504f, -t) + d * 1.925963033e-8f;
    const float e = __builtin_amdgcn_exp2f(t);
    return fmaf(e, r * 0.693147181f, e);
}

template <typename K> __device__ __forceinline__ void write_ranked(const u64* list, int n, int K_, u64* out, K threads) {
    for (int i = threadIdx.x; i < n; i += threads) {
        const u64 mine = list[i];
        int r = 0;
        for (int j = 0; j < n; ++j) r += list[j] > mine;
        if (r < K_) out[r] = mine;
    }
    for (int i = n + threadIdx.x; i < K_; i += threads) out[i] = 0;
}

// A block per (row, chunk of 256 E logits).
template <typename T, int E> __global__ __launch_bounds__(256) void beam_part_k(const BeamArgs a) {
    constexpr int N = 16 / (int)sizeof(T), P = E / N;
    __shared__ u64 list[ROOM];
    __shared__ int counts[2][4];
    __shared__ u32 most[4], least[4];
    __shared__ double sums[4];
    __shared__ int fill;
    const i64 row = blockIdx.x / a.chunks;
    const int chunk = (int)(blockIdx.x - row * a.chunks), tid = threadIdx.x, wave = tid >> 6;
    if (ended(a, row)) return;
    const i64 b = row / a.W;
    const T* __restrict__ x = (const T*)a.logits + b * a.sb + (row - b * a.W) * a.sw;
    const int from = chunk * 256 * E + tid * N;
    float v[E];
#pragma unroll
    for (int p = 0; p < P; ++p) {
        const int i = from + p * 256 * N;
        Pack<T, N> k;
        if (i + N <= a.V) k.load(x + i);
        else
#pragma unroll
            for (int j = 0; j < N; ++j) k.v[j] = i + j < a.V ? x[i + j] : (T)-__builtin_inff();
#pragma unroll
        for (int j = 0; j < N; ++j) v[p * N + j] = (float)k.v[j];
    }
    u32 key[E], mine[1] = {0};
#pragma unroll
    for (int e = 0; e < E; ++e) {
        key[e] = key_of(v[e]);
        mine[0] = key[e] > mine[0] ? key[e] : mine[0];
    }
    const u32 wm = max_wave(mine[0]), wl = min_wave(mine[0]);
    if (lane_id() == 0) most[wave] = wm, least[wave] = wl;
    if (tid == 0) fill = 0;
    lds_barrier();
    u32 hi = most[0], lo = least[0];
#pragma unroll
    for (int w = 1; w < 4; ++w) hi = most[w] > hi ? most[w] : hi, lo = least[w] < lo ? least[w] : lo;
    const float m = hi ? of_key(hi) : 0.f;  // (nothing above -inf: each term is 0, or NaN)
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) s += exp_of(v[e] - m);
    double sum = s;
#pragma unroll
    for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o, WAVE);
    if (lane_id() == 0) sums[wave] = sum;
    // the threads' largest give a threshold that K logits at least reach
    Count<4> count(counts);
    int n = 256;
    u32 t = count.threshold(mine, lo ? lo : 1u, hi, a.K, a.K + a.K / 4, n);
    int c = count.at_least(key, t);
    u32 last = ~0u;  // of the keys equal to t, those of tokens up to here
    if (c > ROOM) {  // many equal ones, or most of them in few threads: the threshold that leaves K
        t = count.threshold(key, t, hi, a.K, ROOM, c);
        if (c > ROOM) {
            const int above = t == hi ? 0 : count.at_least(key, t + 1);
            u32 l = 0, h = (u32)a.V - 1;  // the lowest token up to which enough are equal
            while (l < h) {
                const u32 mid = l + (h - l) / 2;
                int k = 0;
#pragma unroll
                for (int e = 0; e < E; ++e) k += __popcll(__ballot(key[e] == t && (u32)(from + e / N * 256 * N + e % N) <= mid));
                if (above + count.sum(k) >= a.K) h = mid;
                else l = mid + 1;
            }
            last = l;
        }
    }
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const u32 token = from + e / N * 256 * N + e % N;
        if (key[e] > t || (key[e] == t && token <= last)) list[atomicAdd(&fill, 1)] = (u64)key[e] << 32 | (u32)~token;
    }
    __syncthreads();
    const i64 at = row * a.chunks + chunk;
    write_ranked(list, fill, a.K, a.part + at * a.K, 256);
    if (tid == 0) a.top[at] = hi ? m : -__builtin_inff(), a.sum[at] = sums[0] + sums[1] + sums[2] + sums[3];
}

// The chunks' sums of one row, by a wave: log sum exp (NaN or infinite: the row has no candidates).
__device__ __forceinline__ double row_lse(const BeamArgs& a, i64 row) {
    float m = -__builtin_inff();
    for (int c = lane_id(); c < a.chunks; c += 64) m = fmaxf(m, a.top[row * a.chunks + c]);
    m = of_key(max_wave(key_of(m)));  // (all -inf: NaN)
    double s = 0;
    for (int c = lane_id(); c < a.chunks; c += 64) {
        const double x = a.sum[row * a.chunks + c];
        const float t = a.top[row * a.chunks + c];
        s += t == -__builtin_inff() ? x : x * exp((double)t - (double)m);
    }
#pragma unroll
    for (int o = 32; o; o >>= 1) s += __shfl_xor(s, o, WAVE);
    return log(s) + (double)m;
}

// A block a row: its chunks' lists to one of K, and its log sum exp.
__global__ __launch_bounds__(1024) void beam_row_k(const BeamArgs a, u64* part, double* lses) {
    constexpr int E = 16;
    __shared__ u64 list[ROOM];
    __shared__ int counts[2][16];
    __shared__ u64 most[16];
    __shared__ int fill;
    const i64 row = blockIdx.x;
    if (ended(a, row)) return;
    const int have = a.chunks * a.K;
    u64 key[E], mine = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int i = e * 1024 + threadIdx.x;
        key[e] = i < have ? a.part[row * have + i] : 0;
        mine = key[e] > mine ? key[e] : mine;
    }
    mine = max_wave(mine);
    if (lane_id() == 0) most[threadIdx.x >> 6] = mine;
    if (threadIdx.x == 0) fill = 0;
    lds_barrier();
    u64 hi = most[0];
#pragma unroll
    for (int w = 1; w < 16; ++w) hi = most[w] > hi ? most[w] : hi;
    Count<16> count(counts);
    int n = count.at_least(key, 1ull);  // (the keys are all different: a threshold leaves as few as wanted)
    const u64 t = count.threshold(key, 1ull, hi, a.K, ROOM / 4, n);
#pragma unroll
    for (int e = 0; e < E; ++e)
        if (key[e] >= t && key[e]) list[atomicAdd(&fill, 1)] = key[e];
    __syncthreads();
    write_ranked(list, fill, a.K, part + row * a.K, 1024);
    if (threadIdx.x < 64) {
        const double lse = row_lse(a, row);
        if (threadIdx.x == 0) lses[row] = lse;
    }
}

// A block a sequence. MERGED: part holds a list a row and sum its log sum exp.
template <int NW, bool MERGED> __global__ __launch_bounds__(NW * 64) void beam_join_k(const BeamArgs a) {
    constexpr int NT = NW * 64, E = 16;
    __shared__ double lses[MOST], scores[MOST], norms[MOST];
    __shared__ int done[MOST];
    __shared__ u64 most[NW], list[ROOM], list2[ROOM];
    __shared__ int counts[2][NW];
    __shared__ int fill;
    const i64 b = blockIdx.x;
    const int tid = threadIdx.x, wave = tid >> 6;
    for (int w = wave; w < a.W; w += NW) {
        const i64 row = b * a.W + w;
        const bool end = ended(a, row);
        const double lse = end ? 0. : MERGED ? a.sum[row] : row_lse(a, row);
        if (lane_id() == 0) {
            const i64 len = (a.lengths ? length_of(a, row) : 0) + (end ? 0 : 1);
            lses[w] = lse, scores[w] = a.scores[row], done[w] = end;
            norms[w] = a.alpha == 0. ? 1. : pow((double)(len < 1 ? 1 : len), a.alpha);
        }
    }
    if (tid == 0) fill = 0;
    __syncthreads();
    // candidates: the rows' lists, then one of each finished beam. A key's first word is its rank, its second the beam
    // (lower first), the logit and the token (lower first).
    const int per = a.chunks * a.K, have = a.W * per;
    u64 key[E], mine = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int i = e * NT + tid;
        key[e] = 0;
        if (i < have) {
            const int w = i / per;
            const u64 c = done[w] ? 0ull : a.part[b * have + i];
            if (c) key[e] = key_of((scores[w] + ((double)of_key((u32)(c >> 32)) - lses[w])) / norms[w]);
            if (done[w] && i == w * per) key[e] = key_of(scores[w] / norms[w]);
        }
        mine = key[e] > mine ? key[e] : mine;
    }
    mine = max_wave(mine);
    if (lane_id() == 0) most[wave] = mine;
    lds_barrier();
    u64 hi = most[0];
#pragma unroll
    for (int w = 1; w < NW; ++w) hi = most[w] > hi ? most[w] : hi;
    Count<NW> count(counts);
    int n = count.at_least(key, 1ull);
    const u64 t = n > a.K ? count.threshold(key, 1ull, hi, a.K, a.K + 64, n) : 1ull;
    auto second = [&](int i) {
        const int w = i / per;
        const u64 c = done[w] ? 0xFFFFFFFFull << 32 | (u32)~a.pad : a.part[b * have + i];
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
            for (int e = 0; e < E; ++e) k += __popcll(__ballot(key[e] == t && second(e * NT + tid) >= mid));
            if (above + count.sum(k) >= a.K) lo = mid;
            else up = mid - 1;
        }
        t2 = lo;
    }
#pragma unroll
    for (int e = 0; e < E; ++e)
        if (key[e] >= t && key[e]) {
            const u64 s = second(e * NT + tid);
            if (key[e] > t || s >= t2) {
                const int at = atomicAdd(&fill, 1);
                list[at] = key[e], list2[at] = s;
            }
        }
    __syncthreads();
    n = fill;
    auto put = [&](int r, int w, int token, float score) {
        const i64 o = b * a.K + r;
        a.out_scores[o] = score, a.parents[o] = b * a.W + w, a.tokens[o] = token;
        if (a.out_finished) a.out_finished[o] = done[w] || token == a.end;
        if (a.out_lengths) a.out_lengths[o] = length_of(a, b * a.W + w) + (done[w] ? 0 : 1);
    };
    for (int i = tid; i < n; i += NT) {
        const u64 k = list[i], s = list2[i];
        int r = 0;
        for (int j = 0; j < n; ++j) r += list[j] > k || (list[j] == k && list2[j] > s);
        if (r >= a.K) continue;
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
            o &= MOST - 1 - (int)(list2[j] >> 57) != w || (1 << TOKEN_BITS) - 1 - (int)(list2[j] & ((1u << TOKEN_BITS) - 1)) != v;
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
    i64 part, top, sum, rows, row_sum, bytes;  // offsets in the workspace
};

// A chunk is 8192 logits, or fewer where that leaves less than 1024 blocks (4 a CU); not so few that a row's candidates
// outgrow the 16384 that the joining blocks hold. More than 4096 candidates a sequence go through a block a row first.
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
    const i64 n = B * W * chunks;
    p.part = 0;
    p.sum = p.part + n * K * 8;
    p.rows = p.sum + n * 8;
    p.row_sum = p.rows + (p.merge ? B * W * K * 8 : 0);
    p.top = p.row_sum + (p.merge ? B * W * 8 : 0);
    p.bytes = p.top + n * 4;
    return true;
}

extern "C" i64 ng_beam_work(i64 B, i64 W, i64 V, i64 K) {
    BeamPlan p;
    return beam_plan(B, W, V, K, p) ? p.bytes : -1;
}

template <typename T> static void beam_part(const BeamArgs& a, int E, hipStream_t st) {
    const unsigned grid = (unsigned)((i64)a.B * a.W * a.chunks);
    if (E == 32) beam_part_k<T, 32><<<grid, 256, 0, st>>>(a);
    else if (E == 16) beam_part_k<T, 16><<<grid, 256, 0, st>>>(a);
    else beam_part_k<T, 8><<<grid, 256, 0, st>>>(a);
}

extern "C" int ng_beam_step(const void* logits, i64 sb, i64 sw, int dtype, const float* scores, const void* lengths,
                            int lsize, const void* finished, int B, int W, int V, int K, int end, int pad, float alpha,
                            float* out_scores, i64* parents, i64* tokens, void* out_finished, i64* out_lengths, void* work,
                            void* stream) {
    BeamPlan p;
    if (!beam_plan(B, W, V, K, p) || dtype < NG_F32 || dtype > NG_F16 || !(alpha >= 0.f) || (out_lengths && !lengths) ||
        (alpha != 0.f && !lengths) || (lengths && lsize != 4 && lsize != 8) || (finished && (pad < 0 || pad >= V)))
        return -1;
    if (B == 0) return 0;
    BeamArgs a;
    char* w = (char*)work;
    a.logits = logits, a.sb = sb, a.sw = sw, a.scores = scores, a.lengths = lengths, a.lsize = lsize;
    a.finished = (const unsigned char*)finished, a.out_scores = out_scores, a.parents = parents, a.tokens = tokens;
    a.out_finished = (unsigned char*)out_finished, a.out_lengths = out_lengths;
    a.part = (u64*)(w + p.part), a.top = (float*)(w + p.top), a.sum = (double*)(w + p.sum);
    a.B = B, a.W = W, a.V = V, a.K = K, a.chunks = p.chunks, a.end = end, a.pad = pad, a.alpha = alpha;
    hipStream_t st = (hipStream_t)stream;
    switch (dtype) {
        case NG_F32: beam_part<float>(a, p.E, st); break;
        case NG_BF16: beam_part<b16>(a, p.E, st); break;
        default: beam_part<f16>(a, p.E, st);
    }
    int rc = (int)hipGetLastError();
    if (rc) return rc;
    if (!p.merge) beam_join_k<4, false><<<B, 256, 0, st>>>(a);
    else {
        u64* rows = (u64*)(w + p.rows);
        double* lses = (double*)(w + p.row_sum);
        beam_row_k<<<(unsigned)(B * W), 1024, 0, st>>>(a, rows, lses);
        a.part = rows, a.sum = lses, a.chunks = 1;
        beam_join_k<16, true><<<B, 1024, 0, st>>>(a);
    }
    return (int)hipGetLastError();
}

// Rows copied in a given order: out[i] = src[from[i]], zeros where that is no row. U: the unit of a copy; a block takes 256
// units of a row at a time.
template <typename U> __global__ __launch_bounds__(256) void gather_rows_k(const char* __restrict__ src, i64 stride, i64 rows,
                                                                           const i64* __restrict__ from, i64 units, int parts,
                                                                           char* __restrict__ out) {
    const i64 i = blockIdx.x / parts, r = from[i];
    const U* s = (const U*)(src + r * stride);
    U* o = (U*)(out + i * units * (i64)sizeof(U));
    const bool is = (u64)r < (u64)rows;
    const U zero = {};
    for (i64 j = (blockIdx.x % parts) * 256 + threadIdx.x; j < units; j += (i64)parts * 256) o[j] = is ? s[j] : zero;
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
    if (parts * n >= (i64)1 << 31) parts = 1;
    hipStream_t st = (hipStream_t)stream;
    const unsigned grid = (unsigned)(parts * n);
#define GATHER(U) gather_rows_k<U><<<grid, 256, 0, st>>>((const char*)src, stride, rows, from, units, (int)parts, (char*)out)
    if (size == 16) GATHER(uint4);
    else if (size == 4) GATHER(u32);
    else if (size == 2) GATHER(u16);
    else GATHER(unsigned char);
#undef GATHER
    return (int)hipGetLastError();
}
