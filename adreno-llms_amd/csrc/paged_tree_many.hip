// Attention of trees of many rows over a cache in pages (mi_attention_tree): the kernel for many rows, in a file of its own so that
// both compile at the same time.  8 trees of 64 drafts behind 16384, 32 heads over 8 of width 128: fp16 108 us, int8 103, Q4 106.  What bounds it is the chain
// of a tile, as in plain batches; counters of the fp16 ones: matrix cores busy 29 % of the SIMD-cycles, vector units 33 %, LDS 30 % of the CU-cycles (half of it
// conflicts); of the wavefronts' time 40 % are instructions, 37 % waits for memory, LDS and barriers, 23 % for their turn.  int8 and Q4, whose
// tiles are converted on the way to LDS: 26 and 26 %, 40 and 45 %, 42 and 42 %; 39, 46 and 15 %, 39, 48 and 13 %.
#include "paged_chunk.h"

namespace mi {

bool launch_paged_tree_many(hipStream_t s, const TreeArgs& a, float* sums, uint32_t* counters, const PagedLaunch& l) {
    const PartRoom room = {sums, counters};
    const bool wide = a.head_dim == 128;
    return a.kind == MI_KV_F16    ? wide ? launch_chunk<MI_KV_F16, 128, 4, 1>(s, a, room, l) : launch_chunk<MI_KV_F16, 64, 4, 1>(s, a, room, l)
           : a.kind == MI_KV_INT8 ? wide ? launch_chunk<MI_KV_INT8, 128, 4, 1>(s, a, room, l) : launch_chunk<MI_KV_INT8, 64, 4, 1>(s, a, room, l)
                                  : wide ? launch_chunk<MI_KV_Q4, 128, 4, 1>(s, a, room, l) : launch_chunk<MI_KV_Q4, 64, 4, 1>(s, a, room, l);
}

}  // namespace mi
