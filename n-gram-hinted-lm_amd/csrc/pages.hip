// The pages of a paged key/value cache: who holds them, room for more tokens, and copies of them.
//
// State: refs[p], the table entries that hold page p; free, a bit a page, set where refs is 0. asks and claim, 0 and INT_MAX
// for each page between calls, are a reservation's own.
//
// Fork: row s of a table becomes what row parents[s] was. refs[p] += children(row) - 1 for each entry of each row, one atomic
// an entry and none where a row has one child; every holder's change is -1 at least and refs counts them all, so a count
// reaches 0 only by its last change, which sets the free bit. Rows read each other: up to 1024 rows' entries go through LDS, a
// strip of columns a block, more through a scratch table (only the rows that move).
//
// Room: positions length .. length + count - 1 of each row, a request per page that holds any of them. A request is met by
// the entry it finds where no other row holds that page, or where all that hold it request it here and this is the longest of
// them, of equal ones the first (an atomic maximum and count: the order of atomics changes nothing); else by the lowest free
// pages in the order of rows. (The longest: where the pages run out, a row that gets none is left with the page it shares, and
// what the keeper writes there must lie behind that row's tokens.)
// One block does this, since each page given depends on all before it: the requests are scanned 1024 at a time and the free
// bits 32768 pages at a time, up to the last one needed. The rows of a shared page that lie before the length are copied by
// a second kernel, a block per row and head, which also writes the slots.
//
// Counts and pages are whole numbers and every choice is by order, so a call gives the same pages on every run.
//
// Measured (in a trace, us): 64 prompts of 8 rows forked (512 x 65 entries) 6.7, room for a token each 8.5, 448 copies of a
// part of a page of 64 x 8 heads x 128 codes with the slots 8.6; a prompt of 4 rows 2.7, 4.9 and 2.9. Where the table lies in the
// caches, a fork of 512 rows takes 3.1 to read strips of four entries of each row, 0.7 more where the rows change places and 1.1
// more where pages' counts change (4 rows: 1.9, 0.4 and 0.5). The room is one block's chain of loads, scans and barriers; what it
// must read is less than a microsecond's. A third of 8192 pages of 256 KiB packed into
// another cache: 4.7, 4.6 and 269 (1.4 GB moved, 5.3 TB/s: memory bounds it).
#include "vals.h"
#include <climits>

struct Pool {
    int* refs;
    u32* free;
    int *asks, *claim;
    int* missing;
    i64 pages;
};

__device__ __forceinline__ int load_agent(const int* p) {  // past the L1: what atomics have made of it
    return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

__global__ __launch_bounds__(256) void pool_clear_k(const Pool p) {
    const i64 words = (p.pages + 31) / 32, step = (i64)gridDim.x * 256;
    for (i64 i = blockIdx.x * 256ll + threadIdx.x; i < p.pages; i += step) {
        p.refs[i] = 0, p.asks[i] = 0, p.claim[i] = INT_MAX;
        if (i < words) p.free[i] = i * 32 + 32 <= p.pages ? ~0u : (1u << (p.pages & 31)) - 1;
        if (i == 0) *p.missing = 0;
    }
}

__device__ __forceinline__ bool is_page(const Pool& p, int e) { return (u32)e < (u64)p.pages; }

__global__ __launch_bounds__(256) void pool_hold_k(const Pool p, const int* __restrict__ table, i64 stride, int S, int width) {
    const i64 n = (i64)S * width;
    for (i64 i = blockIdx.x * 256ll + threadIdx.x; i < n; i += (i64)gridDim.x * 256) {
        const i64 s = i / width;
        const int e = table[s * stride + (i - s * width)];
        if (is_page(p, e) && atomicAdd(&p.refs[e], 1) == 0) atomicAnd(&p.free[e >> 5], ~(1u << (e & 31)));
    }
}

// ---------------------------------------------------------------------------------------------------------------- fork

#define STRIP 2048  // a block's columns

// Each row's children, in the places of the lengths to come.
__global__ __launch_bounds__(256) void pool_zero_k(int* __restrict__ x, int n) {
    const int i = blockIdx.x * 256 + threadIdx.x;
    if (i < n) x[i] = 0;
}
__global__ __launch_bounds__(256) void pool_children_k(const i64* __restrict__ parents, int S, int* __restrict__ children) {
    const int i = blockIdx.x * 256 + threadIdx.x;
    if (i < S && (u64)parents[i] < (u64)S) atomicAdd(&children[parents[i]], 1);
}

// A block a row. COUNTED: its children are counted already (the count is read before the length goes in its place); else it
// finds them among all the parents.
template <bool COUNTED>
__global__ __launch_bounds__(256) void pool_fork_k(const Pool p, const int* __restrict__ table, i64 stride, int S, int width,
                                                   const int* __restrict__ lengths, const i64* __restrict__ parents,
                                                   int* __restrict__ moved, int* moved_len) {
    __shared__ int children;
    const int s = blockIdx.x, tid = threadIdx.x;
    if (tid == 0) children = COUNTED ? moved_len[s] : 0;
    __syncthreads();
    if constexpr (!COUNTED) {
        int n = 0;
        for (int i = tid; i < S; i += 256) n += parents[i] == s;
        if (n) atomicAdd(&children, n);
        __syncthreads();
    }
    const int change = children - 1;
    const i64 from = parents[s];
    const bool is = (u64)from < (u64)S;
    for (int c = tid; c < width; c += 256) {
        if (change) {
            const int e = table[s * stride + c];
            if (is_page(p, e) && atomicAdd(&p.refs[e], change) + change == 0) atomicOr(&p.free[e >> 5], 1u << (e & 31));
        }
        if (from != s) moved[(i64)s * width + c] = is ? table[from * stride + c] : -1;
    }
    if (tid == 0) moved_len[s] = is ? lengths[from] : 0;
}

// Up to MANY rows: a block takes a strip of columns of all rows, which go through its LDS (512 rows of 65 entries: 6.7 us; by
// a scratch table 5.0 and 2.5, and a launch more).
#define MANY 1024
#define HELD 2048  // entries of a strip
__global__ __launch_bounds__(1024) void pool_fork_few_k(const Pool p, int* __restrict__ table, i64 stride, int S, int width,
                                                        int* __restrict__ lengths, const i64* __restrict__ parents, int shift) {
    __shared__ int held[HELD], from[MANY], children[MANY], len[MANY];
    const int tid = threadIdx.x, columns = 1 << shift, c0 = blockIdx.x << shift, n = width - c0;
    if (tid < S) {
        const i64 f = parents[tid];
        from[tid] = (u64)f < (u64)S ? (int)f : -1;
        children[tid] = 0;
        if (blockIdx.x == 0) len[tid] = lengths[tid];
    }
    for (int i = tid; i < S << shift; i += 1024) {
        const int s = i >> shift, c = i & (columns - 1);
        held[i] = c < n ? table[s * stride + c0 + c] : -1;
    }
    __syncthreads();
    if (tid < S && from[tid] >= 0) atomicAdd(&children[from[tid]], 1);
    __syncthreads();
    for (int i = tid; i < S << shift; i += 1024) {
        const int s = i >> shift, c = i & (columns - 1), change = children[s] - 1, e = held[i], f = from[s];
        if (change && is_page(p, e) && atomicAdd(&p.refs[e], change) + change == 0) atomicOr(&p.free[e >> 5], 1u << (e & 31));
        if (f != s && c < n) table[s * stride + c0 + c] = f < 0 ? -1 : held[(f << shift) + c];
    }
    if (blockIdx.x == 0 && tid < S && from[tid] != tid) lengths[tid] = from[tid] < 0 ? 0 : len[from[tid]];
}

__global__ __launch_bounds__(256) void pool_moved_k(int* __restrict__ table, i64 stride, int width, int* __restrict__ lengths,
                                                    const i64* __restrict__ parents, const int* __restrict__ moved,
                                                    const int* __restrict__ moved_len) {
    const int s = blockIdx.x;
    if (parents[s] == s) return;
    const int c1 = (blockIdx.y + 1) * STRIP < width ? (blockIdx.y + 1) * STRIP : width;
    for (int c = blockIdx.y * STRIP + threadIdx.x; c < c1; c += 256) table[s * stride + c] = moved[(i64)s * width + c];
    if (blockIdx.y == 0 && threadIdx.x == 0) lengths[s] = moved_len[s];
}

// ---------------------------------------------------------------------------------------------------------------- room

struct Room {
    int* table;
    i64 stride;
    const int *lengths, *counts;  // counts: NULL, or each row's own
    int S, width, count, shift, per;  // per: requests a row
    int* rank;    // [S * per]: a request's place among those for a free page; KEPT, NONE
    int* page;    // [S * per]: the page a request found, then the one it has got; -1
    int* given;   // [S * per]: the lowest free pages
    int* source;  // [S]: the page whose first rows are copied to page[s * per], -1
};
enum { KEPT = -1, NONE = -2 };

struct Ask {
    int column, entry, refs, len;
    bool is, held;
};

__device__ __forceinline__ int row_count(const Room& r, int s) {
    const int n = r.counts ? r.counts[s] : r.count;
    return n < 0 ? 0 : n < r.count ? n : r.count;
}

__device__ __forceinline__ int row_len(const Room& r, int s) { return r.lengths[s] < 0 ? 0 : r.lengths[s]; }

__device__ __forceinline__ Ask ask_of(const Pool& p, const Room& r, int i) {
    const int s = i / r.per, j = i - s * r.per, len = row_len(r, s);
    Ask q;
    q.len = len, q.column = (len >> r.shift) + j;
    q.is = ((i64)q.column << r.shift) < (i64)len + row_count(r, s) && q.column < r.width && row_count(r, s) > 0;
    q.entry = q.is ? r.table[s * r.stride + q.column] : -1;
    q.refs = q.is && is_page(p, q.entry) ? p.refs[q.entry] : 0;
    q.held = q.refs > 0;  // (an entry that was never counted is none)
    return q;
}

// The sum over a block of 1024 of the threads before this one, and the whole.
__device__ __forceinline__ int scan_block(int x, int* lds, int& total) {
    int inc = x;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int up = __shfl_up(inc, o, 64);
        if (lane_id() >= o) inc += up;
    }
    __syncthreads();  // (lds was read by the call before)
    if (lane_id() == 63) lds[threadIdx.x >> 6] = inc;
    __syncthreads();
    int before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < 16; ++w) {
        before += w < (int)(threadIdx.x >> 6) ? lds[w] : 0;
        total += lds[w];
    }
    return before + inc - x;
}

// The requests for a shared page, in LDS where there are no more than 1024: a place for each page, found by probing from its
// number's.
#define PLACES 2048
struct Askers {
    int page[PLACES], count[PLACES];
    u64 best[PLACES];  // the largest of longest()
    __device__ __forceinline__ int place(int p) {
        for (u32 i = (u32)p * 2654435761u >> 21;; i = (i + 1) % PLACES) {  // (twice as many places as requests: one is empty)
            const int at = atomicCAS(&page[i], -1, p);
            if (at == p || at == -1) return (int)i;
        }
    }
};

// A request as a number that is larger for longer rows, of equal ones for the first.
__device__ __forceinline__ u64 longest(int len, int i) { return (u64)len << 32 | (u32)~i; }

// The request that page e goes to so far, in its claim, against request i. Each exchange puts a larger one there: it ends.
__device__ __forceinline__ void claim_page(const Pool& p, const Room& r, int e, int len, int i) {
    int cur = load_agent(&p.claim[e]);
    while (cur == INT_MAX || longest(len, i) > longest(row_len(r, cur / r.per), cur)) {
        const int was = atomicCAS(&p.claim[e], cur, i);
        if (was == cur) break;
        cur = was;
    }
}

// ONE: no more than 1024 requests, each in its thread's registers throughout; else they are read again in each phase (1024
// requests so: 11.0 us against 8.2).
template <bool ONE> __global__ __launch_bounds__(1024) void pool_room_k(const Pool p, const Room r) {
    __shared__ int sums[16];
    __shared__ int lowest[ONE ? 1024 : 1];
    __shared__ Askers askers[1];
    const int n = r.S * r.per, tid = threadIdx.x;
    int* given = ONE ? lowest : r.given;
    Ask one;
    int refs = 0;
    one.is = one.held = false;
    const i64 words = (p.pages + 31) / 32;
    const u32 first = tid < words ? p.free[tid] : 0u;
    int place = 0;
    // who else asks for a shared page
    if constexpr (ONE) {
        for (int i = tid; i < PLACES; i += 1024) askers->page[i] = -1, askers->count[i] = 0, askers->best[i] = 0;
        if (tid < n) one = ask_of(p, r, tid), refs = one.refs;
        lds_barrier();
        if (one.held && refs != 1) {
            place = askers->place(one.entry);
            atomicAdd(&askers->count[place], 1);
            atomicMax(&askers->best[place], longest(one.len, tid));
        }
        lds_barrier();
    } else {
        for (int i = tid; i < n; i += 1024) {
            const Ask q = ask_of(p, r, i);
            if (q.held && q.refs != 1) {
                atomicAdd(&p.asks[q.entry], 1);
                claim_page(p, r, q.entry, q.len, i);
            }
        }
        __syncthreads();
    }
    int wanted = 0, rank = NONE;
    for (int i0 = 0; i0 < n; i0 += 1024) {
        const int i = i0 + tid;
        Ask q = one;
        if (!ONE && i < n) q = ask_of(p, r, i);
        bool want = i < n && q.is;
        if (want && q.held) {
            const int refs = q.refs;
            if (ONE) want = refs != 1 && !(refs == askers->count[place] && askers->best[place] == longest(q.len, i));
            else want = refs != 1 && !(refs == load_agent(&p.asks[q.entry]) && load_agent(&p.claim[q.entry]) == i);
        }
        int total;
        const int at = scan_block(want, sums, total);
        if (i < n) {
            rank = want ? wanted + at : q.is ? KEPT : NONE;
            if (!ONE) r.rank[i] = rank, r.page[i] = q.held ? q.entry : -1;
        }
        wanted += total;
    }
    // the lowest free pages
    int found = 0;
    for (i64 w0 = 0; w0 < words && found < wanted; w0 += 1024) {
        u32 bits = w0 == 0 ? first : w0 + tid < words ? p.free[w0 + tid] : 0u;
        int total, at = found + scan_block(__popc(bits), sums, total);
        for (; bits && at < wanted; ++at, bits &= bits - 1) given[at] = (int)((w0 + tid) * 32 + __builtin_ctz(bits));
        found += total;
    }
    if (found > wanted) found = wanted;
    if (tid == 0 && wanted > found) *p.missing += wanted - found;
    __syncthreads();
    for (int i = tid; i < n; i += 1024) {
        const int k = ONE ? rank : r.rank[i], held = !ONE ? r.page[i] : one.held ? one.entry : -1, s = i / r.per, j = i - s * r.per;
        int page = k == KEPT ? held : -1, source = -1;
        if (k >= 0 && k < found) {
            page = given[k];
            r.table[s * r.stride + (ONE ? one.column : (row_len(r, s) >> r.shift) + j)] = page;
            p.refs[page] = 1;
            atomicAnd(&p.free[page >> 5], ~(1u << (page & 31)));
            if (held >= 0) {
                atomicSub(&p.refs[held], 1);
                source = held;
            }
        }
        if (!ONE && held >= 0) p.asks[held] = 0, p.claim[held] = INT_MAX;
        r.page[i] = page;
        if (j == 0) r.source[s] = source;
    }
}

// ------------------------------------------------------------------------------------------------------------- copies

// What a page is made of: parts of `bytes` a row and head. (The bounds have one row a page and head.)
struct Part {
    const char* src;
    char* dst;
    i64 bytes;  // a row
};
struct Parts {
    Part part[5];
    int n, H, shift;
    i64 src_pages, dst_pages;
};

// A store of lines that nothing reads soon: they leave the L2 while the kernel runs, not at its end.
__device__ __forceinline__ void stream16(char* p, uint4 x) {
    typedef u32 words __attribute__((ext_vector_type(4)));
    __builtin_nontemporal_store(__builtin_bit_cast(words, x), (words*)p);
}

__device__ __forceinline__ void copy_bytes(const char* s, char* d, i64 bytes) {  // both at multiples of 16 bytes
    const i64 n = bytes / 16;
    i64 i = threadIdx.x;
    for (; i + 768 < n; i += 1024) {
        uint4 x[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) x[k] = ((const uint4*)s)[i + k * 256];
#pragma unroll
        for (int k = 0; k < 4; ++k) stream16(d + (i + k * 256) * 16, x[k]);
    }
    for (; i < n; i += 256) ((uint4*)d)[i] = ((const uint4*)s)[i];
    for (i = n * 4 + threadIdx.x; i < bytes / 4; i += 256) ((u32*)d)[i] = ((const u32*)s)[i];
}

// A block per (row, head): the slots of the row's positions (head 0), and the rows of a copied page. (128 threads: the blocks
// of 512 rows and 8 heads are on the card at once, and what they wait for one after the other they wait for together.)
__global__ __launch_bounds__(128) void pool_slots_k(const Pool p, const Room r, const Parts c, i64* __restrict__ slots,
                                                    int s0) {
    const int at = blockIdx.x / c.H, h = blockIdx.x - at * c.H, s = s0 + at;
    const int len = row_len(r, s), from = r.source[s], to = r.page[s * r.per], own = row_count(r, s);
    const int in = (1 << r.shift) - 1;
    if (h == 0)
        for (int i = threadIdx.x; i < r.count; i += 128) {
            const i64 pos = (i64)len + i;
            const int page = i < own ? r.page[s * r.per + (int)((pos >> r.shift) - (len >> r.shift))] : -1;
            slots[(i64)s * r.count + i] = page < 0 ? -1 : ((i64)page << r.shift) + (pos & in);
        }
    const int rows = len & in;
    if (!rows || from < 0) return;
    const i64 a = ((i64)from * c.H + h) << c.shift, b = ((i64)to * c.H + h) << c.shift;
    // keys and values together, so that a row's loads are all under way before its stores
    const i64 row = c.part[0].bytes;
    const int units = (int)(rows * row / 16), t = threadIdx.x;
    const bool q8 = c.n > 2;
    u32 ks = 0, vs = 0;
    if (q8 && t < rows) ks = ((const u32*)c.part[2].src)[a + t], vs = ((const u32*)c.part[3].src)[a + t];
    for (int i = t; i < units; i += 512) {
        uint4 x[2][4];
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (i + u * 128 < units) x[k][u] = ((const uint4*)(c.part[k].src + a * row))[i + u * 128];
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (i + u * 128 < units) stream16(c.part[k].dst + b * row + (i + u * 128) * 16ll, x[k][u]);
    }
    if (!q8) return;
    if (t < rows) ((u32*)c.part[2].dst)[b + t] = ks, ((u32*)c.part[3].dst)[b + t] = vs;
    for (int i = t + 128; i < rows; i += 128) {
        ((u32*)c.part[2].dst)[b + i] = ((const u32*)c.part[2].src)[a + i];
        ((u32*)c.part[3].dst)[b + i] = ((const u32*)c.part[3].src)[a + i];
    }
}

// Page dst[i] of one cache := page src[i] of another, in pieces of PIECE bytes, from i0 on; entries that are no pages are passed
// over. (dst NULL: page i, for a move's list of live pages.)
#define PIECE 65536
template <typename I>
__global__ __launch_bounds__(256) void copy_pages_k(const Parts c, const I* __restrict__ src, const I* __restrict__ dst,
                                                    i64 i0, int pieces) {
    const u32 at = blockIdx.x / (u32)pieces;
    const i64 i = i0 + at;
    const int piece = (int)(blockIdx.x - at * pieces);
    const i64 a = src[i], b = dst ? (i64)dst[i] : i;
    if ((u64)a >= (u64)c.src_pages || (u64)b >= (u64)c.dst_pages) return;
    i64 from = (i64)piece * PIECE, end = from + PIECE;
    for (int k = 0; k < c.n; ++k) {  // the parts laid end to end
        const Part& t = c.part[k];
        const i64 size = t.bytes * c.H << (k < 4 ? c.shift : 0);
        const i64 x = from < 0 ? 0 : from, y = end < size ? end : size;
        if (x < y) copy_bytes(t.src + a * size + x, t.dst + b * size + x, y - x);
        from -= size, end -= size;
        if (end <= 0) break;
    }
}

// The live pages in order: list[i] = the i-th, map[p] = its place (-1), and the other pool's state. A thread a page; a block
// counts the free bits before its own by itself.
__global__ __launch_bounds__(1024) void pool_pack_k(const Pool p, const Pool to, int* __restrict__ list, int* __restrict__ map) {
    __shared__ int sums[16];
    const i64 page = (i64)blockIdx.x * 1024 + threadIdx.x;
    const bool is = page < p.pages && !(p.free[page >> 5] >> (page & 31) & 1);
    const int refs = is ? p.refs[page] : 0;
    int n = 0, before, total;
    for (i64 w = threadIdx.x; w < (i64)blockIdx.x * 32; w += 1024) n += __popc(~p.free[w]);  // (whole words)
    scan_block(n, sums, before);
    const int at = before + scan_block(is, sums, total);
    if (page < p.pages) map[page] = is && at < to.pages ? at : -1;
    if (is && at < to.pages) list[at] = (int)page, to.refs[at] = refs;
    if (blockIdx.x + 1 < gridDim.x) return;
    const int all = before + total, tid = threadIdx.x;  // the last block: what is behind the live pages
    if (tid == 0) *to.missing += all > to.pages ? (int)(all - to.pages) : 0;
    for (i64 i = all + tid; i < to.pages; i += 1024) list[i] = -1, to.refs[i] = 0;
    for (i64 v = tid; v < (to.pages + 31) / 32; v += 1024) {
        const i64 from = all - v * 32;  // the word's first free page
        const u32 in = v * 32 + 32 <= to.pages ? ~0u : (1u << (to.pages & 31)) - 1;
        to.free[v] = from >= 32 ? 0u : from <= 0 ? in : in & ~0u << from;
    }
}

__global__ __launch_bounds__(256) void pool_map_k(const Pool p, const int* __restrict__ table, i64 stride, int S, int width,
                                                  const int* __restrict__ map, int* __restrict__ out) {
    const i64 n = (i64)S * width;
    for (i64 i = blockIdx.x * 256ll + threadIdx.x; i < n; i += (i64)gridDim.x * 256) {
        const i64 s = i / width;
        const int e = table[s * stride + (i - s * width)];
        out[i] = is_page(p, e) ? map[e] : -1;
    }
}

// ------------------------------------------------------------------------------------------------------------ the host

// refs, asks, claim int32 [pages], free u32 [(pages + 31) / 32], missing int32 [1], end to end
static i64 pool_words(i64 pages) { return 3 * pages + (pages + 31) / 32 + 1; }
static bool pool_of(void* state, i64 pages, Pool& p) {
    if (pages < 1 || pages >= (i64)1 << 31) return false;
    p.refs = (int*)state, p.asks = p.refs + pages, p.claim = p.asks + pages, p.free = (u32*)(p.claim + pages);
    p.missing = (int*)(p.free + (pages + 31) / 32), p.pages = pages;
    return true;
}

#define MOST_BLOCKS (((i64)1 << 24) - 1)  // of a launch, of up to 256 threads: fewer than 2^32 in all

static int some_blocks(i64 n) {
    const int g = grid_for(n, 256);
    return g < 2048 ? g : 2048;
}

extern "C" i64 ng_pool_state(i64 pages) { return pages < 1 || pages >= (i64)1 << 31 ? -1 : pool_words(pages) * 4; }

extern "C" int ng_pool_clear(void* state, i64 pages, void* stream) {
    Pool p;
    if (!pool_of(state, pages, p)) return -1;
    pool_clear_k<<<some_blocks(pages), 256, 0, (hipStream_t)stream>>>(p);
    return (int)hipGetLastError();
}

extern "C" int ng_pool_hold(void* state, i64 pages, const int* table, i64 stride, int S, int width, void* stream) {
    Pool p;
    if (!pool_of(state, pages, p) || S < 0 || width < 0) return -1;
    if ((i64)S * width == 0) return 0;
    pool_hold_k<<<some_blocks((i64)S * width), 256, 0, (hipStream_t)stream>>>(p, table, stride, S, width);
    return (int)hipGetLastError();
}

extern "C" i64 ng_pool_fork_work(i64 S, i64 width) {
    if (S < 0 || width < 1 || S > MOST_BLOCKS || width > 1 << 26 || S * width >= (i64)1 << 40) return -1;
    return S <= MANY ? 0 : (S * width + S) * 4;
}

extern "C" int ng_pool_fork(void* state, i64 pages, int* table, i64 stride, int S, int width, int* lengths,
                            const i64* parents, void* work, void* stream) {
    Pool p;
    if (!pool_of(state, pages, p) || ng_pool_fork_work(S, width) < 0) return -1;
    if (S == 0) return 0;
    if (S <= MANY) {
        int shift = 5;  // 32 columns, 2 for 1024 rows
        while (S << shift > HELD) --shift;
        pool_fork_few_k<<<(unsigned)(((i64)width + (1 << shift) - 1) >> shift), 1024, 0, (hipStream_t)stream>>>(
            p, table, stride, S, width, lengths, parents, shift);
        return (int)hipGetLastError();
    }
    int* moved = (int*)work;
    int* moved_len = moved + (i64)S * width;
    const dim3 grid(S, (width + STRIP - 1) / STRIP);
    hipStream_t st = (hipStream_t)stream;
    // Looking for the children costs rows squared, counting them two launches: 2048 rows of 65 entries 18.7 and 21.9 us, 4096
    // 28.5 and 27.4, 16384 160 and 59, 65536 of 17 1880 and 78, 262144 of 2 28600 and 245.
    if (S <= 4096) pool_fork_k<false><<<S, 256, 0, st>>>(p, table, stride, S, width, lengths, parents, moved, moved_len);
    else {
        const unsigned blocks = (S + 255) / 256;
        pool_zero_k<<<blocks, 256, 0, st>>>(moved_len, S);
        pool_children_k<<<blocks, 256, 0, st>>>(parents, S, moved_len);
        pool_fork_k<true><<<S, 256, 0, st>>>(p, table, stride, S, width, lengths, parents, moved, moved_len);
    }
    const int rc = (int)hipGetLastError();
    if (rc) return rc;
    pool_moved_k<<<grid, 256, 0, st>>>(table, stride, width, lengths, parents, moved, moved_len);
    return (int)hipGetLastError();
}

static int room_per(int count, int shift) { return ((count - 1) >> shift) + 2; }

extern "C" i64 ng_pool_room_work(i64 S, i64 count, i64 page) {
    if (S < 0 || count < 1 || count >= (i64)1 << 30 || page < 16 || page > 4096 || (page & (page - 1))) return -1;
    const i64 n = S * room_per((int)count, __builtin_ctz((unsigned)page));
    return n >= (i64)1 << 28 ? -1 : (3 * n + S) * 4;
}

// A cache's parts side by side with another's (the same one: a page's rows copied within it). Without scales, or bounds: NULL.
static bool parts_of(const void* const (&src)[5], void* const (&dst)[5], i64 src_pages, i64 dst_pages, int page, int heads,
                     int dim, int codes, Parts& c) {
    if (page < 16 || page > 4096 || (page & (page - 1)) || heads < 1 || dim < 1 || dim > 256 || codes < KV_INT8 ||
        codes > KV_F16 || src_pages < 1 || dst_pages < 1 || src_pages >= (i64)1 << 31 || dst_pages >= (i64)1 << 31)
        return false;
    const i64 dp = (dim + 63) / 64 * 64;
    const bool q8 = codes == KV_INT8 || codes == KV_FP8;
    c.n = 0, c.H = heads, c.shift = __builtin_ctz((unsigned)page), c.src_pages = src_pages, c.dst_pages = dst_pages;
    for (int i = 0; i < 5; ++i) {
        c.part[i].src = (const char*)src[i], c.part[i].dst = (char*)dst[i];
        c.part[i].bytes = i < 2 ? dp * (q8 ? 1 : 2) : i < 4 ? (q8 ? 4 : 0) : 4 * dp;
    }
    c.n = q8 ? 4 : 2;
    return true;
}

extern "C" int ng_pool_room(void* state, i64 pages, int* table, i64 stride, int S, int width, const int* lengths,
                            const int* counts, int count, void* k, void* v, void* ks, void* vs, int page, int heads,
                            int dim, int codes, i64* slots, void* work, void* stream) {
    Pool p;
    Parts c;
    const void* const src[5] = {k, v, ks, vs, nullptr};
    void* const dst[5] = {k, v, ks, vs, nullptr};
    if (!pool_of(state, pages, p) || S < 0 || width < 1 || ng_pool_room_work(S, count, page) < 0 ||
        !parts_of(src, dst, pages, pages, page, heads, dim, codes, c) || heads > MOST_BLOCKS)
        return -1;
    if (S == 0) return 0;
    Room r;
    r.table = table, r.stride = stride, r.lengths = lengths, r.counts = counts, r.S = S, r.width = width, r.count = count;
    r.shift = c.shift, r.per = room_per(count, c.shift);
    const i64 n = (i64)S * r.per;
    r.rank = (int*)work, r.page = r.rank + n, r.given = r.page + n, r.source = r.given + n;
    hipStream_t st = (hipStream_t)stream;
    if (n <= 1024) pool_room_k<true><<<1, 1024, 0, st>>>(p, r);
    else pool_room_k<false><<<1, 1024, 0, st>>>(p, r);
    const int rc = (int)hipGetLastError();
    if (rc) return rc;
    const i64 most = MOST_BLOCKS / heads;  // rows a launch
    for (i64 s0 = 0; s0 < S; s0 += most) {
        const i64 rows = S - s0 < most ? S - s0 : most;
        pool_slots_k<<<(unsigned)(rows * heads), 128, 0, st>>>(p, r, c, slots, (int)s0);
        const int rc = (int)hipGetLastError();
        if (rc) return rc;
    }
    return 0;
}

static i64 page_pieces(const Parts& c, bool bounds) {
    i64 size = 0;
    for (int i = 0; i < 5; ++i)
        if (i < c.n || (i == 4 && bounds)) size += c.part[i].bytes * c.H << (i < 4 ? c.shift : 0);
    return (size + PIECE - 1) / PIECE;
}

template <typename I> static int copy_list(Parts c, bool bounds, const I* src, const I* dst, i64 n, hipStream_t st) {
    const i64 pieces = page_pieces(c, bounds);
    if (bounds) c.n = 5;  // (a 16-bit cache's scales have rows of no bytes)
    if (pieces > MOST_BLOCKS) return -1;
    const i64 most = MOST_BLOCKS / pieces;  // pages a launch
    for (i64 i0 = 0; i0 < n; i0 += most) {
        const i64 pages = n - i0 < most ? n - i0 : most;
        copy_pages_k<I><<<(unsigned)(pages * pieces), 256, 0, st>>>(c, src, dst, i0, (int)pieces);
        const int rc = (int)hipGetLastError();
        if (rc) return rc;
    }
    return 0;
}

extern "C" int ng_copy_pages(const void* k, const void* v, const void* ks, const void* vs, const void* bounds, i64 pages,
                             void* to_k, void* to_v, void* to_ks, void* to_vs, void* to_bounds, i64 to_pages, int page,
                             int heads, int dim, int codes, const i64* src, const i64* dst, i64 n, void* stream) {
    Parts c;
    const void* const from[5] = {k, v, ks, vs, bounds};
    void* const to[5] = {to_k, to_v, to_ks, to_vs, to_bounds};
    if (n < 0 || (bounds == nullptr) != (to_bounds == nullptr) ||
        !parts_of(from, to, pages, to_pages, page, heads, dim, codes, c))
        return -1;
    return n == 0 ? 0 : copy_list(c, bounds != nullptr, src, dst, n, (hipStream_t)stream);
}

extern "C" i64 ng_pool_move_work(i64 pages, i64 to_pages) {
    return pages < 1 || to_pages < 1 || pages >= (i64)1 << 31 || to_pages >= (i64)1 << 31 ? -1 : (pages + to_pages) * 4;
}

extern "C" int ng_pool_move(void* state, i64 pages, const void* k, const void* v, const void* ks, const void* vs,
                            const void* bounds, void* to_state, i64 to_pages, void* to_k, void* to_v, void* to_ks, void* to_vs,
                            void* to_bounds, int page, int heads, int dim, int codes, const int* table, i64 stride, int S,
                            int width, int* out, void* work, void* stream) {
    Pool p, to;
    Parts c;
    const void* const from[5] = {k, v, ks, vs, bounds};
    void* const into[5] = {to_k, to_v, to_ks, to_vs, to_bounds};
    if (!pool_of(state, pages, p) || !pool_of(to_state, to_pages, to) || S < 0 || width < 0 ||
        (bounds == nullptr) != (to_bounds == nullptr) ||
        !parts_of(from, into, pages, to_pages, page, heads, dim, codes, c))
        return -1;
    int* list = (int*)work;
    int* map = list + to_pages;
    hipStream_t st = (hipStream_t)stream;
    pool_pack_k<<<(unsigned)((pages + 1023) / 1024), 1024, 0, st>>>(p, to, list, map);
    int rc = (int)hipGetLastError();
    if (rc) return rc;
    if ((i64)S * width) {
        pool_map_k<<<some_blocks((i64)S * width), 256, 0, st>>>(p, table, stride, S, width, map, out);
        if ((rc = (int)hipGetLastError())) return rc;
    }
    return copy_list<int>(c, bounds != nullptr, list, nullptr, pages < to_pages ? pages : to_pages, st);
}
