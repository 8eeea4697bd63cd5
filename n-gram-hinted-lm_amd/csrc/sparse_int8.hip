// Attention over chosen pages of a int8 cache, and their bounds (sparse.hip).
#include "sparse.h"

template int sparse_codes<KV_INT8>(const SparseArgs&, int, hipStream_t);
template int bounds_codes<KV_INT8>(const void*, const float*, i64, int, int, int, const int*, i64, int, const int*, int, int, b16*,
                              hipStream_t);
