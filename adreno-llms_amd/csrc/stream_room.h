// The device memory that a stream of the library's owns: how much of it, for what, and what becomes of a stream where there is not
// enough.  Plain C++.
#pragma once
#include <cstddef>
#include <cstdint>

namespace mi {

// A stream's workspace holds kWorkspaceBytes for whatever a launch puts there and, behind them, kSliceCounters
// counters that are 0 between launches (slices of K that meet inside a launch, parts of a sequence's keys).
constexpr size_t kWorkspaceBytes = 16u << 20;
constexpr int kSliceCounters = 16384;
inline uint32_t* slice_counters(void* workspace) {
    return reinterpret_cast<uint32_t*>(static_cast<char*>(workspace) + kWorkspaceBytes);
}
// An allocation of its own: room for the sums of attention's rows whose keys several blocks share (paged_attention.hip).
constexpr size_t kPartialBytes = 32u << 20;

struct StreamRoom {
    void* workspace = nullptr;     // null: GEMMs do not slice K, attention does not split keys
    void* sums = nullptr;          // null: attention does not split keys
};

// allocate(bytes): device memory or null; clear(workspace): its counters, false if that failed; release(p).  Where the memory is not
// enough for both, the GEMMs' share stays.
template <class Allocate, class Clear, class Release>
StreamRoom make_stream_room(Allocate allocate, Clear clear, Release release) {
    StreamRoom r;
    r.workspace = allocate(kWorkspaceBytes + kSliceCounters * sizeof(uint32_t));
    if (r.workspace && !clear(r.workspace)) {
        release(r.workspace);
        r.workspace = nullptr;
    }
    if (r.workspace) r.sums = allocate(kPartialBytes);
    return r;
}

}  // namespace mi
