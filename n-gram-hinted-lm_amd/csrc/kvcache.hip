// A key/value cache in pages, held in 8 bits (int8 or fp8 e4m3) with a float32 scale per token and head, or in 16 bits:
// codes [pages, heads, page size, DP] (DP: the head's size to a multiple of 64, zeros behind it), scales [pages, heads,
// page size]. A token's slot is page * page size + row.
//
// Quantising, per row x of one head: a = max |x|, inv = M / a, code = x * inv rounded half to even (M = 127 for int8, 448
// for e4m3), scale = a / M; all in 32 bits, the two divisions once a row. a = 0, or so small that inv overflows: code and
// scale 0. A row that holds a NaN or an infinity: codes 0 and scale NaN, so that it reads back as NaN wherever it is seen
// and nothing of it reaches a row that masks it.
//
// Both directions move every byte once and compute little: memory bounds them. A row is 8 elements a lane (8, 16 or 32
// lanes by DP), so that the 16-bit side moves 16 bytes a lane and a row's lanes cover whole 128-byte lines. Measured, 8
// heads of 128, bfloat16 to and from int8: 4096 tokens written 11.2 us (2.3 TB/s; one filling of the card, its start and
// end count), 32768 read 45 us (4.5 TB/s); 8 tokens written 3.3 us, a launch.
#include "vals.h"

template <typename T> __device__ __forceinline__ void load8(const T* p, int d0, int dim, bool vec, float (&x)[8]) {
    if (vec && d0 + 8 <= dim) {
        constexpr int N = 16 / (int)sizeof(T);
#pragma unroll
        for (int j = 0; j < 8; j += N) {
            Pack<T, N> k;
            k.load(p + d0 + j);
#pragma unroll
            for (int i = 0; i < N; ++i) x[j + i] = (float)k.v[i];
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = d0 + j < dim ? (float)p[d0 + j] : 0.f;
    }
}

struct WriteArgs {
    const void *x[2];       // keys, values [n, heads, dim]
    void* codes[2];
    float* scale[2];
    i64 tok_stride[2], head_stride[2];
    const i64* slots;
    i64 n, total_slots;
    int heads, dim, shift;  // page size = 1 << shift
    int vec;
};

// One group of GS lanes writes one (token, head) row; blockIdx.y: 0 keys, 1 values.
template <typename T, int CODES, int DP, int GS>
__global__ __launch_bounds__(256) void kv_write_k(const WriteArgs a) {
    const int side = blockIdx.y, sub = threadIdx.x % GS, d0 = sub * 8;
    const T* __restrict__ x = (const T*)a.x[side];
    const i64 rows = a.n * a.heads, step = (i64)gridDim.x * (256 / GS);
    for (i64 r = (i64)blockIdx.x * (256 / GS) + threadIdx.x / GS; r < rows; r += step) {
        const i64 tok = r / a.heads;
        const int head = (int)(r - tok * a.heads);
        const i64 slot = a.slots[tok];
        if ((u64)slot >= (u64)a.total_slots) continue;  // -1 or out of range: not written (uniform in the group)
        const i64 row = (((slot >> a.shift) * a.heads + head) << a.shift) + (slot & ((1 << a.shift) - 1));
        float v[8];
        load8(x + tok * a.tok_stride[side] + head * a.head_stride[side], d0, a.dim, a.vec, v);
        if constexpr (CODES == KV_BF16 || CODES == KV_F16) {
            if (d0 < DP) {
                Pack<T, 8> k;
#pragma unroll
                for (int j = 0; j < 8; ++j) k.v[j] = (T)v[j];  // the cache's own type: exact
                k.store((T*)a.codes[side] + row * DP + d0);
            }
        } else {
            float m = 0.f;
            bool fine = true;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                m = fmaxf(m, __builtin_fabsf(v[j]));
                fine &= finite_f(v[j]);
            }
            if (!fine) m = __builtin_inff();
#pragma unroll
            for (int o = GS / 2; o; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, GS));
            constexpr float top = CODES == KV_INT8 ? 127.f : 448.f;
            float inv = top / m, scale = m / top;
            if (!finite_f(inv)) inv = 0.f, scale = 0.f;  // m = 0, or too small for its inverse
            const bool bad = !finite_f(m);
            if (bad) scale = __builtin_nanf("");
            u32 w[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float y[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) y[j] = bad ? 0.f : v[4 * h + j] * inv;
                if constexpr (CODES == KV_INT8) {
                    w[h] = 0;
#pragma unroll
                    for (int j = 0; j < 4; ++j) w[h] |= ((u32)(int)__builtin_rintf(y[j]) & 0xFFu) << (8 * j);
                } else {
                    int p = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
                    w[h] = (u32)__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], p, true);
                }
            }
            if (d0 < DP) *(uint2*)((char*)a.codes[side] + row * DP + d0) = make_uint2(w[0], w[1]);
            if (sub == 0) a.scale[side][row] = scale;
        }
    }
}

struct ReadArgs {
    const void* codes[2];
    const float* scale[2];
    void* out[2];  // [n, heads, dim]
    const i64* slots;
    i64 n, total_slots;
    int heads, dim, shift, vec;
};

template <int CODES> struct code_t { typedef unsigned char type; };
template <> struct code_t<KV_BF16> { typedef b16 type; };
template <> struct code_t<KV_F16> { typedef f16 type; };

template <typename T, int CODES, int DP, int GS>
__global__ __launch_bounds__(256) void kv_read_k(const ReadArgs a) {
    typedef typename code_t<CODES>::type C;
    const int side = blockIdx.y, sub = threadIdx.x % GS, d0 = sub * 8;
    const C* __restrict__ codes = (const C*)a.codes[side];
    T* __restrict__ out = (T*)a.out[side];
    const i64 rows = a.n * a.heads, step = (i64)gridDim.x * (256 / GS);
    for (i64 r = (i64)blockIdx.x * (256 / GS) + threadIdx.x / GS; r < rows; r += step) {
        const i64 tok = r / a.heads;
        const int head = (int)(r - tok * a.heads);
        const i64 slot = a.slots[tok];
        float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if ((u64)slot < (u64)a.total_slots && d0 < DP) {
            const i64 row = (((slot >> a.shift) * a.heads + head) << a.shift) + (slot & ((1 << a.shift) - 1));
            Pack<C, 8> k;
            k.load(codes + row * DP + d0);
            if constexpr (CODES == KV_INT8 || CODES == KV_FP8) {
                const float s = a.scale[side][row];
                if constexpr (CODES == KV_INT8) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) v[j] = (float)(signed char)k.v[j] * s;
                } else {
                    u32 w[2];
                    __builtin_memcpy(w, k.v, 8);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[h], false);
                        const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[h], true);
                        v[4 * h] = lo[0] * s, v[4 * h + 1] = lo[1] * s, v[4 * h + 2] = hi[0] * s, v[4 * h + 3] = hi[1] * s;
                    }
                }
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = (float)k.v[j];
            }
        }
        T* o = out + r * a.dim + d0;
        if (a.vec && d0 + 8 <= a.dim) {
            constexpr int N = 16 / (int)sizeof(T);
#pragma unroll
            for (int j = 0; j < 8; j += N) {
                Pack<T, N> p;
#pragma unroll
                for (int i = 0; i < N; ++i) p.v[i] = (T)v[j + i];
                p.store(o + j);
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (d0 + j < a.dim) o[j] = (T)v[j];
        }
    }
}

// The row's lanes and the grid: enough groups for every row, at most 4096 blocks a side (16 waves of blocks of the
// whole card), each taking rows in turns.
template <int DP> constexpr int group_lanes() { return DP <= 64 ? 8 : DP <= 128 ? 16 : 32; }

static inline int kv_grid(i64 rows, int gs) {
    const i64 g = (rows + 256 / gs - 1) / (256 / gs);
    return (int)(g < 4096 ? g : 4096);
}

template <typename T, int CODES> static int kv_write_dp(int dp, const WriteArgs& a, hipStream_t st) {
    switch (dp) {
#define DP_CASE(DP)                                                                                                     \
    case DP:                                                                                                            \
        kv_write_k<T, CODES, DP, group_lanes<DP>()>                                                                     \
            <<<dim3(kv_grid(a.n * a.heads, group_lanes<DP>()), 2), 256, 0, st>>>(a);                                    \
        break;
        DP_CASE(64) DP_CASE(128) DP_CASE(192) DP_CASE(256)
#undef DP_CASE
        default: return -1;
    }
    return (int)hipGetLastError();
}

template <typename T, int CODES> static int kv_read_dp(int dp, const ReadArgs& a, hipStream_t st) {
    switch (dp) {
#define DP_CASE(DP)                                                                                                     \
    case DP:                                                                                                            \
        kv_read_k<T, CODES, DP, group_lanes<DP>()>                                                                      \
            <<<dim3(kv_grid(a.n * a.heads, group_lanes<DP>()), 2), 256, 0, st>>>(a);                                    \
        break;
        DP_CASE(64) DP_CASE(128) DP_CASE(192) DP_CASE(256)
#undef DP_CASE
        default: return -1;
    }
    return (int)hipGetLastError();
}

static bool kv_shape_ok(i64 n, i64 pages, int page, int heads, int dim, int codes) {
    return n >= 0 && pages >= 0 && page >= 16 && (page & (page - 1)) == 0 && page <= 4096 && heads >= 1 && dim >= 1 &&
           dim <= 256 && codes >= KV_INT8 && codes <= KV_F16 && pages <= (i64)1 << 40 && n <= ((i64)1 << 50) / heads;
}

extern "C" int ng_kv_write(const void* k, const void* v, i64 k_tok, i64 k_head, i64 v_tok, i64 v_head, int dtype,
                           const i64* slots, i64 n, void* kc, void* vc, float* ks, float* vs, i64 pages, int page,
                           int heads, int dim, int codes, void* stream) {
    if (!kv_shape_ok(n, pages, page, heads, dim, codes)) return -1;
    if (n == 0) return 0;
    WriteArgs a;
    a.x[0] = k, a.x[1] = v, a.codes[0] = kc, a.codes[1] = vc, a.scale[0] = ks, a.scale[1] = vs;
    a.tok_stride[0] = k_tok, a.tok_stride[1] = v_tok, a.head_stride[0] = k_head, a.head_stride[1] = v_head;
    a.slots = slots, a.n = n, a.total_slots = pages * page, a.heads = heads, a.dim = dim;
    a.shift = __builtin_ctz((unsigned)page);
    const i64 size = dtype == NG_F32 ? 4 : 2;
    a.vec = ((((u64)k | (u64)v) & 15) == 0) && (((k_tok | k_head | v_tok | v_head) * size) & 15) == 0;
    const int dp = (dim + 63) / 64 * 64;
    hipStream_t st = (hipStream_t)stream;
    if (codes == KV_BF16) return dtype == NG_BF16 ? kv_write_dp<b16, KV_BF16>(dp, a, st) : -1;
    if (codes == KV_F16) return dtype == NG_F16 ? kv_write_dp<f16, KV_F16>(dp, a, st) : -1;
    if (codes == KV_INT8) switch (dtype) {
        case NG_F32: return kv_write_dp<float, KV_INT8>(dp, a, st);
        case NG_BF16: return kv_write_dp<b16, KV_INT8>(dp, a, st);
        case NG_F16: return kv_write_dp<f16, KV_INT8>(dp, a, st);
        default: return -1;
    }
    switch (dtype) {
        case NG_F32: return kv_write_dp<float, KV_FP8>(dp, a, st);
        case NG_BF16: return kv_write_dp<b16, KV_FP8>(dp, a, st);
        case NG_F16: return kv_write_dp<f16, KV_FP8>(dp, a, st);
        default: return -1;
    }
}

template <typename T> static int kv_read_codes(int codes, int dp, const ReadArgs& a, hipStream_t st) {
    switch (codes) {
        case KV_INT8: return kv_read_dp<T, KV_INT8>(dp, a, st);
        case KV_FP8: return kv_read_dp<T, KV_FP8>(dp, a, st);
        case KV_BF16: return kv_read_dp<T, KV_BF16>(dp, a, st);
        default: return kv_read_dp<T, KV_F16>(dp, a, st);
    }
}

extern "C" int ng_kv_read(const void* kc, const void* vc, const float* ks, const float* vs, i64 pages, int page, int heads,
                          int dim, int codes, const i64* slots, i64 n, void* k, void* v, int dtype, void* stream) {
    if (!kv_shape_ok(n, pages, page, heads, dim, codes)) return -1;
    if (n == 0) return 0;
    ReadArgs a;
    a.codes[0] = kc, a.codes[1] = vc, a.scale[0] = ks, a.scale[1] = vs, a.out[0] = k, a.out[1] = v;
    a.slots = slots, a.n = n, a.total_slots = pages * page, a.heads = heads, a.dim = dim;
    a.shift = __builtin_ctz((unsigned)page);
    a.vec = ((((u64)k | (u64)v) & 15) == 0) && dim % 8 == 0;
    const int dp = (dim + 63) / 64 * 64;
    hipStream_t st = (hipStream_t)stream;
    switch (dtype) {
        case NG_F32: return kv_read_codes<float>(codes, dp, a, st);
        case NG_BF16: return kv_read_codes<b16>(codes, dp, a, st);
        case NG_F16: return kv_read_codes<f16>(codes, dp, a, st);
        default: return -1;
    }
}

// The slots of positions start[b] .. start[b] + count - 1 of B sequences: [B, count], -1 past the table or where its page
// is none of the cache's.
__global__ void kv_slots_k(const int* __restrict__ table, i64 stride, int width, const int* __restrict__ start, int B,
                           int count, i64 pages, int shift, i64* __restrict__ out) {
    const i64 n = (i64)B * count;
    for (i64 i = blockIdx.x * (i64)blockDim.x + threadIdx.x; i < n; i += (i64)gridDim.x * blockDim.x) {
        const int b = (int)(i / count);
        const i64 p = (i64)start[b] + (i - (i64)b * count);
        i64 s = -1;
        if (p >= 0 && (p >> shift) < width) {
            const int g = table[b * stride + (p >> shift)];
            if (g >= 0 && g < pages) s = ((i64)g << shift) + (p & ((1 << shift) - 1));
        }
        out[i] = s;
    }
}

extern "C" int ng_kv_slots(const int* table, i64 stride, int width, const int* start, int B, int count, i64 pages, int page,
                           i64* out, void* stream) {
    if (B < 0 || count < 0 || width < 0 || page < 16 || (page & (page - 1))) return -1;
    const i64 n = (i64)B * count;
    if (n == 0) return 0;
    const int g = grid_for(n, 256);
    kv_slots_k<<<g > 4096 ? 4096 : g, 256, 0, (hipStream_t)stream>>>(table, stride, width, start, B, count, pages,
                                                                     __builtin_ctz((unsigned)page), out);
    return (int)hipGetLastError();
}
