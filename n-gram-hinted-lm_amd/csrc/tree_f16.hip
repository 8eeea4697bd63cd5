// Tree attention over float16 caches.
#include "tree.h"

template int tree_codes<KV_F16>(const TreeArgs&, const TreePlan&, hipStream_t);
