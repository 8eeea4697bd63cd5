// Tree attention over fp8 (e4m3) caches.
#include "tree.h"

template int tree_codes<KV_FP8>(const TreeArgs&, const TreePlan&, hipStream_t);
