// Tree attention over int8 caches.
#include "tree.h"

template int tree_codes<KV_INT8>(const TreeArgs&, const TreePlan&, hipStream_t);
