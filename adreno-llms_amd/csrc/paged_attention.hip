// Attention of many sequences' new tokens over a cache in pages (mi_attention): paged_kernels.h for plain batches.
#include "paged_kernels.h"

namespace mi {

bool launch_paged_attention(hipStream_t s, const AttentionArgs& a, const StreamRoom& room) { return launch_attention("mi_attention", s, a, room); }

}  // namespace mi
