// Attention for a tree of drafted tokens over a paged key/value cache.
//
//   o[i] = sum_p softmax_p(scale * q[i] . k[p]) v[p]   over the positions p that tree token i sees: the sequence's cached
//          tokens, and the tree token j (position length + j) where bit j of mask[i] is set; a row that sees nothing: 0
//
// Mathematics. One pass over the keys with a running maximum M and sum l per row, in base 2 and 32 bits. A cache held in
// 8 bits is not dequantised: the key's scale multiplies the finished score, and the value's scale joins the exponent,
// P = exp2(score + log2(vscale) - M), so that P keeps its bits whatever the scales are to each other and the product P V
// runs on the codes; the sum of the softmax takes P / vscale. (Value scales of 2^-64 to 2^40: a smaller one is split in
// two factors, and beside a larger one weights below 2^-30 of the row's largest can be missing in the sum.) M follows the
// maximum in steps of 2^4 at least, and over 8-bit caches P is raised by 2^8: it is at most 2^12. Codes of 8 bits are exact
// in 16-bit floats. The 8-bit caches run on f16 products (queries scaled by a power of two to f16's range), 16-bit caches
// on their own type.
//
// Rounding. Scores, M, l and the outputs' sums are held in 32 bits. P is rounded to 16 bits for its product with the
// values (f16; bf16 over a bf16 cache), because the matrix instructions take no 32-bit operand at this rate: each key's
// weight is off by up to 2^-11 (2^-8) of itself, as much as an output of that type is rounded in any case, and over 8-bit
// caches by up to 2^-33 of the largest weighted value. l sums P before that rounding.
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
//
// Measured (8 kv heads of 128, groups of 4, int8 unless said). 64 sequences x 8 tokens over up to 8192 cached: 145 us and
// 6.5 of joining, 4.7 TB/s of the cache, near a copy's 5.2: memory bounds it. 2 x 64 tokens over 131072, fp8: 425 us, 640
// TFLOP/s against a large product's 1294: vector instructions bound it (8.8 a matrix instruction with the matrix ones: each
// of the head's eight groups of rows turns the same codes into operands again, and the softmax's). 8 x 16 tokens over up to
// 4096: 25 + 5 us against 8 of bytes: a share is few tiles long, so its beginning and end and the joining are most of it.
// One token over 300 keys: 7.7 + 3.3 us, launches. Heads of 192 and 256 hold one wave a SIMD: 16 x 8 tokens over 8192
// 100 us (4.2 TB/s) and 143 (3.9; fp8 130), bf16 caches 163 (5.0) and 220 (4.9).
#include "tree.h"

// (One wave a sequence; a launch bounds it.)
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

static bool tree_plan(int B, int T, int H, int G, int dim, int codes, i64 cap, TreePlan& p) {
    if (B < 0 || T < 1 || T > 64 || H < 1 || G < 1 || dim < 1 || dim > 256 || codes < KV_INT8 || codes > KV_F16 || cap < 1 ||
        cap > (i64)1 << 30 || (i64)T * G > 1 << 20)
        return false;
    p.dp = (dim + 63) / 64 * 64;
    const int rows = T * G;
    p.rpb = rows <= 16 ? 16 : 32;
    p.groups = (rows + p.rpb - 1) / p.rpb;
    const i64 units = (i64)B * H * p.groups, most = units * ((cap + TILE - 1) / TILE + START);
    if (units > 1 << 24 || most > (i64)1 << 30) return false;
    p.blocks = most < MAX_BLOCKS ? (int)(most + 7) / 8 * 8 : MAX_BLOCKS;
    p.join = cap > TILE;
    const i64 slots = p.join ? 2ll * p.blocks * p.rpb : 0;
    p.po = 0, p.pm = slots * p.dp * 4, p.bytes = p.pm + 2 * slots * 4;
    return true;
}

extern "C" i64 ng_tree_attention_work(i64 B, i64 T, i64 H, i64 G, i64 dim, i64 codes, i64 cap) {
    TreePlan p;
    const i64 lim = 1 << 30;
    if (B > lim || T > lim || H > lim || G > lim || dim > lim) return -1;
    return tree_plan((int)B, (int)T, (int)H, (int)G, (int)dim, (int)codes, cap, p) ? p.bytes : -1;
}

extern template int tree_codes<KV_INT8>(const TreeArgs&, const TreePlan&, hipStream_t);
extern template int tree_codes<KV_FP8>(const TreeArgs&, const TreePlan&, hipStream_t);
extern template int tree_codes<KV_BF16>(const TreeArgs&, const TreePlan&, hipStream_t);
extern template int tree_codes<KV_F16>(const TreeArgs&, const TreePlan&, hipStream_t);

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
    a.pl = a.pm + (p.join ? 2ll * p.blocks * p.rpb : 0);
    a.pages = pages, a.B = B, a.T = T, a.H = H, a.G = G, a.dim = dim, a.shift = __builtin_ctz((unsigned)page);
    a.width = width, a.groups = p.groups, a.qtype = qtype, a.scale = scale;
    a.vec = ((u64)q & 15) == 0 && (((qb | qt | qh) * 2) & 15) == 0;
    hipStream_t st = (hipStream_t)stream;
    switch (codes) {
        case KV_INT8: return tree_codes<KV_INT8>(a, p, st);
        case KV_FP8: return tree_codes<KV_FP8>(a, p, st);
        case KV_BF16: return tree_codes<KV_BF16>(a, p, st);
        default: return tree_codes<KV_F16>(a, p, st);
    }
}

extern "C" int ng_tree_mask(const int* parents, int B, int T, u64* bits, void* stream) {
    if (B < 0 || T < 1 || T > 64) return -1;
    if (B == 0) return 0;
    tree_mask_k<<<B, 64, 0, (hipStream_t)stream>>>(parents, T, bits);
    return (int)hipGetLastError();
}
