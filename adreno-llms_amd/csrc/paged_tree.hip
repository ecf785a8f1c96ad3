// Attention of a tree of drafted tokens over a cache in pages (mi_attention_tree): paged_kernels.h for trees, in a file of its own
// so that both compile at the same time.
#include "paged_kernels.h"

namespace mi {

bool launch_paged_tree(hipStream_t s, const TreeArgs& a, const StreamRoom& room) { return launch_attention("mi_attention_tree", s, a, room); }

}  // namespace mi
