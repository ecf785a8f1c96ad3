// Rows of a paged cache that move, as they are stored, in all layers' caches at once: the accepted ones of a sequence's drafts to where they
// belong (mi_kv_keep), a beam's last page to one of its own (mi_kv_reorder).
#include "../../include/mi_attention.h"
#include "common.h"
#include "paged.h"

namespace mi {
namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kMostCaches = 32;                    // of a launch: 1 KB of arguments
struct Pools {
    uint8_t *k, *v;
    uint16_t *k_scale, *v_scale;
};
struct Layers {
    Pools of[kMostCaches];
};

// ---- accepted drafts --------------------------------------------------------------------------------------
//
// Numbers ascend, so row keep[i] >= i moves down or stays, and rows done in order never overwrite one that is still to be read.  A wavefront
// has some 16-byte columns of a sequence's rows in one pool and looks up where 64 of its kept rows come from and go to, one to a lane;
// then it moves as many at a time as its lanes and kAhead registers take: these are all read before the first of them is written.
//
// What bounds it: five trips to memory one after the other, to lengths, numbers, page table, rows and back, and the launch: 16 paths in 24 layers of
// 2 x 64 3.8 to 4.2 us on the GPU, 7.6 with the host's call; 48 paths of up to 11 rows in 16 layers of 8 x 128, 17 MB, 8.1 to 8.9 (each row's
// place looked up where it moves, four rows at a time: 10).  In int8 and Q4 all of these are the host's call, 7.4 to 8.2.
constexpr int kAhead = 8;

struct KeepArgs {
    PagedArgs p;
    const int *keep, *kept;
    int* new_len;
    int column_blocks;
};

template <int KIND, int D>
__global__ __launch_bounds__(64) void kv_keep_kernel(const KeepArgs a, const Layers layers) {
    constexpr int kPieces = row_bytes(KIND, D) / 16, kScales = row_scales(KIND, D);
    const int lane = threadIdx.x;
    const int b = blockIdx.x / a.column_blocks, block = blockIdx.x - b * a.column_blocks;
    const Span s = span_of(a.p.q_start[b], a.p.q_start[b + 1], a.p.kv_len[b], a.p.n_tokens);
    int kept = a.kept[b];
    kept = kept < 0 ? 0 : kept > s.n ? s.n : kept;
    if (a.new_len && blockIdx.y == 0 && block == 0 && lane == 0) a.new_len[b] = s.pos + kept;
    // the lane's column, and which of the rows of a load it has
    const int columns = a.p.n_kv_heads * kPieces, width = columns < 64 ? columns : 64, together = 64 / width;
    const int mine = lane / width, column = block * 64 + (lane - mine * width), head = column / kPieces, piece = column % kPieces;
    const bool busy = mine < together && column < columns;
    const Pools& pools = layers.of[blockIdx.y / 2];
    uint8_t* const pool = blockIdx.y % 2 ? pools.v : pools.k;
    uint16_t* const scales = blockIdx.y % 2 ? pools.v_scale : pools.k_scale;
    const int* const table = a.p.pages + static_cast<int64_t>(b) * a.p.max_pages;
    const auto place = [&](int pos) {              // of head 0's row
        if (pos < 0 || pos >= a.p.cap) return static_cast<int64_t>(-1);
        const int page = divide(pos, a.p.page), number = table[page];
        if (static_cast<uint32_t>(number) >= static_cast<uint32_t>(a.p.n_pages)) return static_cast<int64_t>(-1);
        return row_number(a.p, number, 0, pos - page * a.p.page.d);
    };
    const auto of_lane = [](int64_t x, int from) {
        return static_cast<int64_t>(static_cast<uint32_t>(__shfl(static_cast<int>(x), from))) | static_cast<int64_t>(__shfl(static_cast<int>(x >> 32), from)) << 32;
    };
    for (int first = 0; first < kept; first += 64) {
        int64_t from = -1, to = -1;                // of kept row first + lane; -1: it does not move
        if (first + lane < kept) {
            const int i = first + lane, number = a.keep[s.first + i];
            if (number != i && number >= 0 && number < s.n) {
                from = place(s.pos + number);
                to = place(s.pos + i);
            }
            if (from < 0) to = -1;
        }
        const int last = kept - first < 64 ? kept - first : 64;
        for (int i0 = 0; i0 < last; i0 += kAhead * together) {
            int64_t src[kAhead], dst[kAhead];
            u32x4 x[kAhead];
            uint16_t sc[kAhead][kScales > 0 ? kScales : 1];
            #pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                const int i = i0 + u * together + mine;
                src[u] = of_lane(from, i & 63) + head * a.p.page.d;
                dst[u] = of_lane(to, i & 63);
                dst[u] = busy && i < last && dst[u] >= 0 ? dst[u] + head * a.p.page.d : -1;
            }
            #pragma unroll
            for (int u = 0; u < kAhead; ++u)
                if (dst[u] >= 0) {
                    x[u] = *reinterpret_cast<const u32x4*>(pool + src[u] * row_bytes(KIND, D) + 16 * piece);
                    if constexpr (kScales > 0)
                        if (piece == 0)
                            for (int z = 0; z < kScales; ++z) sc[u][z] = scales[src[u] * kScales + z];
                }
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");       // (a row of this load may be where another goes)
            #pragma unroll
            for (int u = 0; u < kAhead; ++u)
                if (dst[u] >= 0) {
                    *reinterpret_cast<u32x4*>(pool + dst[u] * row_bytes(KIND, D) + 16 * piece) = x[u];
                    if constexpr (kScales > 0)
                        if (piece == 0)
                            for (int z = 0; z < kScales; ++z) scales[dst[u] * kScales + z] = sc[u][z];
                }
        }
    }
}

// ---- copies of sequences ----------------------------------------------------------------------------------
//
// The rows of a last page lie together for each head, and go in pieces of 16 bytes; the tables go in the same launch.  What bounds it: bytes where
// there are many, 48 beams' pages of up to 99 rows of 8 x 128 in 16 layers, 180 MB written, 67 to 70 us (copies of one page read it from the caches), of int8
// and Q4 33 and 21, as many bytes a second (their scales go by two bytes a thread);
// else the launch and three trips, 2.7 to 3.1 us on the GPU for 16 beams in 24 layers, 7.3 with the host's call.

struct ReorderArgs {
    PagedArgs p;                                   // (kv_len, pages; no rows)
    const int *source, *fresh;
    int *new_len, *new_pages;
    int parts;
    int pools;                                     // of this launch; blockIdx.y = pools: the tables
};
constexpr int kCopyThreads = 256, kCopyAhead = 4;

template <int KIND, int D>
__global__ __launch_bounds__(kCopyThreads) void kv_reorder_kernel(const ReorderArgs a, const Layers layers) {
    constexpr int kPieces = row_bytes(KIND, D) / 16, kScales = row_scales(KIND, D);
    const int b = blockIdx.x / a.parts, part = blockIdx.x - b * a.parts, tid = threadIdx.x;
    const int f = a.source[b];
    const bool valid = static_cast<uint32_t>(f) < static_cast<uint32_t>(a.p.n_seqs);
    const int given = valid ? a.p.kv_len[f] : 0, len = given < 0 ? 0 : given;
    const int full = divide(len, a.p.page), tail = len - full * a.p.page.d;
    const bool own = valid && f != b && tail > 0;  // a page of its own
    const int64_t row = static_cast<int64_t>(a.p.max_pages);
    if (static_cast<int>(blockIdx.y) == a.pools) {
        const int used = full + (tail > 0);
        for (int j = part * kCopyThreads + tid; j < a.p.max_pages; j += a.parts * kCopyThreads)
            a.new_pages[b * row + j] = j >= used ? -1 : own && j == full ? a.fresh[b] : a.p.pages[f * row + j];
        if (part == 0 && tid == 0) a.new_len[b] = given;
        return;
    }
    if (!own || full >= a.p.max_pages) return;
    const int src = a.p.pages[f * row + full], dst = a.fresh[b];
    if (static_cast<uint32_t>(src) >= static_cast<uint32_t>(a.p.n_pages) || static_cast<uint32_t>(dst) >= static_cast<uint32_t>(a.p.n_pages)) return;
    const Pools& pools = layers.of[blockIdx.y / 2];
    uint8_t* const pool = blockIdx.y % 2 ? pools.v : pools.k;
    const int64_t from = row_number(a.p, src, 0, 0), to = row_number(a.p, dst, 0, 0);
    // a head's rows lie together: pieces of 16 bytes, the heads' one after the other
    const uint32_t each = static_cast<uint32_t>(tail) * kPieces, all = each * a.p.n_kv_heads;
    const auto* const in = reinterpret_cast<const u32x4*>(pool + from * row_bytes(KIND, D));
    auto* const out = reinterpret_cast<u32x4*>(pool + to * row_bytes(KIND, D));
    for (uint32_t z0 = part * (kCopyThreads * kCopyAhead) + tid; z0 < all; z0 += a.parts * (kCopyThreads * kCopyAhead)) {
        u32x4 x[kCopyAhead];
        uint32_t at[kCopyAhead];
        #pragma unroll
        for (int u = 0; u < kCopyAhead; ++u) {
            const uint32_t z = z0 + u * kCopyThreads, head = z / each;
            at[u] = head * (a.p.page.d * kPieces) + (z - head * each);
            if (z < all) x[u] = in[at[u]];
        }
        #pragma unroll
        for (int u = 0; u < kCopyAhead; ++u)
            if (z0 + u * kCopyThreads < all) out[at[u]] = x[u];
    }
    if constexpr (kScales > 0) {
        uint16_t* const scales = blockIdx.y % 2 ? pools.v_scale : pools.k_scale;
        const uint32_t few = static_cast<uint32_t>(tail) * kScales, total = few * a.p.n_kv_heads;
        for (uint32_t z = part * kCopyThreads + tid; z < total; z += a.parts * kCopyThreads) {
            const uint32_t head = z / few, place = head * (a.p.page.d * kScales) + (z - head * few);
            scales[to * kScales + place] = scales[from * kScales + place];
        }
    }
}

// ---- the host's side ----------------------------------------------------------------------------------------

bool off(const void* p, uintptr_t align) { return !p || reinterpret_cast<uintptr_t>(p) % align; }

// Whether x or y is one of a and b.
bool among(const void* x, const void* y, const void* a, const void* b) { return (x == a) | (x == b) | (y == a) | (y == b); }

// Checks the caches of a call, which are alike but for their pools, and its batch.  (A pool that is there twice would have its rows moved twice,
// by two wavefronts at once, one of scales its scales.  Every pool is compared with all before it, in loops
// of their own: of 24 caches the call's host time with all its checks is 1.0 us in fp16, 1.4 in int8; in one loop 1.5 and 1.4.)
bool layers_args(const char* who, const mi_kv_cache* caches, int n, const mi_kv_batch& batch, PagedArgs* out) {
    if (!caches || n < 1) {
        MI_ERROR_FMT("%s: no caches (caches=%p n_caches=%d)", who, static_cast<const void*>(caches), n);
        return false;
    }
    for (int i = 0; i < n; ++i) {
        const mi_kv_cache &c = caches[i], &d = caches[0];
        if (!paged_args(who, &c, &batch, out)) return false;
        if (c.kind != d.kind || c.n_pages != d.n_pages || c.page_size != d.page_size || c.n_kv_heads != d.n_kv_heads || c.head_dim != d.head_dim) {
            MI_ERROR_FMT("%s: cache %d differs from the first in more than its pools", who, i);
            return false;
        }
    }
    const bool quantised = caches->kind != MI_KV_F16;
    for (int i = 0; i < n; ++i) {
        const mi_kv_cache& c = caches[i];
        bool pools = c.k == c.v, scales = quantised && c.k_scale == c.v_scale;
        for (int j = 0; j < i; ++j) pools |= among(c.k, c.v, caches[j].k, caches[j].v);
        for (int j = 0; j < i && quantised; ++j) scales |= among(c.k_scale, c.v_scale, caches[j].k_scale, caches[j].v_scale);
        if (pools) {
            MI_ERROR_FMT("%s: a pool of cache %d is there twice", who, i);
            return false;
        }
        if (scales) {
            MI_ERROR_FMT("%s: scales of cache %d are there twice", who, i);
            return false;
        }
    }
    return true;
}

Layers layers_of(const mi_kv_cache* caches, int n) {
    Layers l{};
    for (int i = 0; i < n; ++i)
        l.of[i] = {static_cast<uint8_t*>(caches[i].k), static_cast<uint8_t*>(caches[i].v), static_cast<uint16_t*>(caches[i].k_scale),
                   static_cast<uint16_t*>(caches[i].v_scale)};
    return l;
}

// `go` with the kernel for a cache's kind and width.
#define MI_KV_KERNEL(KERNEL, CACHE, GO)                                                                                              \
    [&] {                                                                                                                            \
        const bool wide = (CACHE).head_dim == 128;                                                                                   \
        if ((CACHE).kind == MI_KV_F16) wide ? GO(KERNEL<MI_KV_F16, 128>) : GO(KERNEL<MI_KV_F16, 64>);                                \
        else if ((CACHE).kind == MI_KV_INT8) wide ? GO(KERNEL<MI_KV_INT8, 128>) : GO(KERNEL<MI_KV_INT8, 64>);                        \
        else wide ? GO(KERNEL<MI_KV_Q4, 128>) : GO(KERNEL<MI_KV_Q4, 64>);                                                            \
        return MI_HIP_OK(hipGetLastError());                                                                                         \
    }()

}  // namespace
}  // namespace mi

using namespace mi;

extern "C" int mi_kv_keep(void* stream, const mi_kv_cache* caches, int n_caches, const mi_kv_batch* batch, const int* keep, const int* kept,
                          int* new_len) {
    if (!batch) {
        MI_ERROR_FMT("mi_kv_keep: null batch");
        return 0;
    }
    KeepArgs a{};
    if (!layers_args("mi_kv_keep", caches, n_caches, *batch, &a.p)) return 0;
    if (a.p.n_seqs == 0) return 1;
    if ((a.p.n_tokens > 0 && off(keep, 4)) || off(kept, 4) || (new_len && (off(new_len, 4) || new_len == keep || new_len == kept || new_len == a.p.q_start || new_len == a.p.kv_len || new_len == a.p.pages))) {
        MI_ERROR_FMT("mi_kv_keep: bad argument (keep=%p kept=%p new_len=%p)", static_cast<const void*>(keep), static_cast<const void*>(kept),
                     static_cast<void*>(new_len));
        return 0;
    }
    const int64_t columns = static_cast<int64_t>(a.p.n_kv_heads) * (row_bytes(caches->kind, caches->head_dim) / 16);
    const int64_t column_blocks = (columns + 63) / 64, blocks = column_blocks * a.p.n_seqs;
    if (blocks > 0x7fffffff / 64 || columns > 0x3fffffff) {
        MI_ERROR_FMT("mi_kv_keep: %d sequences of %d heads are more than a launch counts", a.p.n_seqs, a.p.n_kv_heads);
        return 0;
    }
    if (!ensure_init()) return 0;
    a.keep = keep;
    a.kept = kept;
    a.new_len = new_len;
    a.column_blocks = static_cast<int>(column_blocks);
    for (int at = 0; at < n_caches; at += kMostCaches) {
        const int n = n_caches - at < kMostCaches ? n_caches - at : kMostCaches;
        const Layers layers = layers_of(caches + at, n);
        const auto go = [&](auto kern) {
            hipLaunchKernelGGL(kern, dim3(static_cast<unsigned>(blocks), 2 * n), dim3(64), 0, static_cast<hipStream_t>(stream), a, layers);
        };
        if (!MI_KV_KERNEL(kv_keep_kernel, *caches, go)) return 0;
        a.new_len = nullptr;
    }
    return 1;
}

extern "C" int mi_kv_reorder(void* stream, const mi_kv_cache* caches, int n_caches, const mi_kv_reorder_call* call) {
    if (!call) {
        MI_ERROR_FMT("mi_kv_reorder: null call");
        return 0;
    }
    const mi_kv_reorder_call& c = *call;
    // (q_start is not read: a sequence has no rows in this call)
    const mi_kv_batch batch = {c.kv_len, c.kv_len, c.pages, c.n_seqs, 0, 0, c.max_pages};
    ReorderArgs a{};
    if (!layers_args("mi_kv_reorder", caches, n_caches, batch, &a.p)) return 0;
    if (a.p.n_seqs == 0) return 1;
    const void* const read[] = {c.kv_len, c.pages, c.source, c.fresh};
    bool bad = off(c.source, 4) || off(c.fresh, 4) || off(c.new_len, 4) || off(c.new_pages, 4) || c.new_len == c.new_pages;
    for (const void* p : read) bad |= p == c.new_len || p == c.new_pages;
    if (bad) {
        MI_ERROR_FMT("mi_kv_reorder: bad argument (source=%p fresh=%p new_len=%p new_pages=%p)", static_cast<const void*>(c.source),
                     static_cast<const void*>(c.fresh), static_cast<void*>(c.new_len), static_cast<void*>(c.new_pages));
        return 0;
    }
    // Blocks per sequence and pool: for a page that is full but for a row.  (A page is less than 2 GiB: fewer than 2^27 pieces.)
    const int64_t pieces = static_cast<int64_t>(a.p.n_kv_heads) * a.p.page.d * (row_bytes(caches->kind, caches->head_dim) / 16);
    const int64_t parts = (pieces + kCopyThreads * kCopyAhead - 1) / (kCopyThreads * kCopyAhead);
    a.parts = static_cast<int>(parts < 64 ? parts : 64);
    if (static_cast<int64_t>(a.parts) * a.p.n_seqs > 0x7fffffff / kCopyThreads) {
        MI_ERROR_FMT("mi_kv_reorder: %d sequences are more than a launch counts", a.p.n_seqs);
        return 0;
    }
    if (!ensure_init()) return 0;
    a.source = c.source;
    a.fresh = c.fresh;
    a.new_len = c.new_len;
    a.new_pages = c.new_pages;
    for (int at = 0; at < n_caches; at += kMostCaches) {
        const int n = n_caches - at < kMostCaches ? n_caches - at : kMostCaches;
        const Layers layers = layers_of(caches + at, n);
        a.pools = 2 * n;
        const auto go = [&](auto kern) {
            hipLaunchKernelGGL(kern, dim3(static_cast<unsigned>(a.parts * a.p.n_seqs), 2 * n + (at == 0)), dim3(kCopyThreads), 0,
                               static_cast<hipStream_t>(stream), a, layers);
        };
        if (!MI_KV_KERNEL(kv_reorder_kernel, *caches, go)) return 0;
    }
    return 1;
}
