// Tree attention over bfloat16 caches.
#include "tree.h"

template int tree_codes<KV_BF16>(const TreeArgs&, const TreePlan&, hipStream_t);
