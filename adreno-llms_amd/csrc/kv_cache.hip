// Rows of keys and values into the pages of a cache and back out (mi_kv_write, mi_kv_read), and the checks that the entry
// points over such a cache share.  The reference appends one row at the sequence's position, fp16 (KV cache
// QW/src/layers/attention.cpp:111-131).
//
// scale = fp16(greatest |x| / top) with top = 127 or 7, code = x / scale to the nearest integer, ties to even.  Both are
// exact: an fp16 number over 127 or 7 is never within 2^-9 of an fp16 step of the middle between two fp16 numbers, and a quotient of
// two fp16 numbers that is not a half-integer is at least 2^-12 away from one, more than an fp32 quotient's error at 127.
#include "../../include/mi_linear.h"
#include "device_math.h"
#include "paged.h"

#include <cmath>
#include <type_traits>

namespace mi {
namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

constexpr int kThreads = 256;
constexpr int kPiece = 8;                          // values per thread: 16 bytes of an fp16 row

// Where row `row` of the batch lies in the cache: the number of its row of head 0 in the pools (the next head's is a page further), -1
// where it has no place.  `mine`: it belongs to a sequence.  The same for a wavefront; its lanes look for the sequence together, as
// a search by halves would wait for a load at every step.
struct Place {
    int64_t cache;
    bool mine;
};
__device__ __forceinline__ Place place_of(const PagedArgs& a, int row) {
    Place p{-1, false};
    const int lane = threadIdx.x & 63;
    int b = -1;
    for (int b0 = 0; b0 < a.n_seqs; b0 += 64) {
        const int s = b0 + lane < a.n_seqs ? b0 + lane : a.n_seqs - 1;
        const int here = __popcll(__ballot(b0 + lane < a.n_seqs && a.q_start[s] <= row));
        b += here;
        if (here < 64) break;
    }
    b = __builtin_amdgcn_readfirstlane(b);
    if (b < 0) return p;
    const Span s = span_of(a.q_start[b], a.q_start[b + 1], a.kv_len[b], a.n_tokens);
    if (row < s.first || row - s.first >= s.n) return p;
    p.mine = true;
    const int pos = s.pos + (row - s.first);
    if (pos < 0 || pos >= a.cap) return p;
    const int page = divide(pos, a.page);
    const int number = __builtin_amdgcn_readfirstlane(a.pages[static_cast<int64_t>(b) * a.max_pages + page]);
    if (static_cast<uint32_t>(number) >= static_cast<uint32_t>(a.n_pages)) return p;
    p.cache = row_number(a, number, 0, pos - page * a.page.d);
    return p;
}

// The greatest of the values of N neighbouring lanes (N = 4, 8, 16: a piece of a DPP row), in each of them.
template <int N>
__device__ __forceinline__ uint32_t max_of(uint32_t m) {
    auto with = [&](auto ctrl) {
        const uint32_t o = __builtin_amdgcn_update_dpp(0, m, decltype(ctrl)::value, 0xf, 0xf, true);
        m = o > m ? o : m;
    };
    with(std::integral_constant<int, 0xb1>{});                                 // lane ^ 1
    with(std::integral_constant<int, 0x4e>{});                                 // lane ^ 2
    if constexpr (N >= 8) with(std::integral_constant<int, 0x141>{});          // half rows mirrored
    if constexpr (N >= 16) with(std::integral_constant<int, 0x140>{});         // rows mirrored
    return m;
}

// A wavefront has one row of keys or values (blockIdx.y), 512 of its elements at a time, 8 to a lane.  Bound by bytes where there
// are many rows, by the chain of loads to a row's place (q_start, kv_len, pages) where there are few.  A thread for every 8
// elements that looked its place up by itself took 42 us to read 6 Q4 conversations of up to 8000 (102 MB); so it is 26.5, 3.85 TB/s.
// 2048 rows of 8 x 128 written as int8 and read back, 25 MB: 10.0 us for the two launches, 2.5 TB/s; in fp16 / int8 / Q4 written 5.2 / 5.5 / 4.9,
// read 5.7 / 4.9 / 5.1; 31800 such rows read back 53 / 45 / 45 us, 4.9 / 4.4 / 3.7 TB/s; 7 rows written: 2.5 us.
template <int KIND, int D>
__global__ __launch_bounds__(kThreads) void kv_write_kernel(const PagedArgs a, const uint16_t* __restrict__ k, const uint16_t* __restrict__ v,
                                                            const int64_t ld_k, const int64_t ld_v) {
    const int row = __builtin_amdgcn_readfirstlane(blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6)), lane = threadIdx.x & 63;
    if (row >= a.n_tokens) return;
    const uint16_t* const src = blockIdx.y ? v + row * ld_v : k + row * ld_k;
    const bool wide = reinterpret_cast<uintptr_t>(src) % 16 == 0;
    const int width = a.n_kv_heads * D;
    // (the first elements are on their way while the row's place is looked up)
    auto load = [&](int e0) {
        half8 x = {};
        const int e = e0 + kPiece * lane;
        if (e >= width) return x;
        if (wide) return *reinterpret_cast<const half8*>(src + e);
        #pragma unroll
        for (int z = 0; z < 8; ++z) x[z] = __builtin_bit_cast(_Float16, src[e + z]);
        return x;
    };
    half8 x = load(0);
    const Place p = place_of(a, row);
    if (p.cache < 0) return;
    uint8_t* const pool = const_cast<uint8_t*>(blockIdx.y ? a.v : a.k);
    uint16_t* const scales = const_cast<uint16_t*>(blockIdx.y ? a.v_scale : a.k_scale);
    for (int e0 = 0; e0 < width; e0 += 64 * kPiece) {
        const half8 next = load(e0 + 64 * kPiece);
        const int e = e0 + kPiece * lane, at = e % D;
        const int64_t cache = p.cache + static_cast<int64_t>(e / D) * a.page.d;
        if (e < width) {
            if constexpr (KIND == MI_KV_F16) {
                *reinterpret_cast<half8*>(pool + (cache * D + at) * 2) = x;
            } else {
                constexpr bool kInt8 = KIND == MI_KV_INT8;
                constexpr float kTop = kInt8 ? 127.0f : 7.0f, kMost = kInt8 ? 515.5f : 9352.0f;     // (code * scale stays below 65520)
                // The greatest |x| as fp16 bits, which ascend with the value, an infinity's and NaNs' behind all finite ones.
                const u32x4 bits = __builtin_bit_cast(u32x4, x) & 0x7fff7fffu;
                uint32_t most = 0;
                #pragma unroll
                for (int z = 0; z < 4; ++z) {
                    most = bits[z] >> 16 > most ? bits[z] >> 16 : most;
                    most = (bits[z] & 0xffffu) > most ? bits[z] & 0xffffu : most;
                }
                most = max_of<kInt8 ? D / kPiece : 32 / kPiece>(most);
                const bool finite = most < 0x7c00u;
                const float big = h_f(static_cast<uint16_t>(most));
                const _Float16 h = static_cast<_Float16>(finite ? fminf(__fdiv_rn(big, kTop), kMost) : __builtin_nanf(""));
                const float scale = static_cast<float>(h);
                // x / scale from the reciprocal and what is left of x behind it (exact in fma): a half-integer comes out as such.
                // (scale 0: reciprocal 0, all codes 0.)  Added to 1.5 * 2^23 the quotient is rounded to an integer, which is then in
                // the low bits (Q4: plus 8).
                const float inverse = finite && scale > 0.0f ? __builtin_amdgcn_rcpf(scale) : 0.0f, by = finite ? scale : 0.0f;
                constexpr float kBase = 12582912.0f + (kInt8 ? 0.0f : 8.0f);
                uint32_t code[8];
                #pragma unroll
                for (int z = 0; z < 8; ++z) {
                    const float f = finite ? static_cast<float>(x[z]) : 0.0f, q = f * inverse;
                    const float c = __builtin_amdgcn_fmed3f(fmaf(fmaf(-q, by, f), inverse, q), kInt8 ? -127.0f : -8.0f, kTop);
                    code[z] = __float_as_uint(c + kBase);
                }
                // the low bytes of four
                auto bytes = [&](int z, int step) {
                    return __builtin_amdgcn_perm(__builtin_amdgcn_perm(code[z + 3 * step], code[z + 2 * step], 0x0c0c0400u),
                                                 __builtin_amdgcn_perm(code[z + step], code[z], 0x0c0c0400u), 0x05040100u);
                };
                if constexpr (kInt8) {
                    *reinterpret_cast<u32x2*>(pool + cache * D + at) = u32x2{bytes(0, 1), bytes(4, 1)};
                    if (at == 0) scales[cache] = __builtin_bit_cast(uint16_t, h);
                } else {
                    *reinterpret_cast<uint32_t*>(pool + (cache * D + at) / 2) = bytes(0, 2) | bytes(1, 2) << 4;
                    if (at % 32 == 0) scales[cache * (D / 32) + at / 32] = __builtin_bit_cast(uint16_t, h);
                }
            }
        }
        x = next;
    }
}

template <int KIND, int D>
__global__ __launch_bounds__(kThreads) void kv_read_kernel(const PagedArgs a, uint16_t* __restrict__ k, uint16_t* __restrict__ v,
                                                           const int64_t ld_k, const int64_t ld_v) {
    const int row = __builtin_amdgcn_readfirstlane(blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6)), lane = threadIdx.x & 63;
    if (row >= a.n_tokens) return;
    const Place p = place_of(a, row);
    if (!p.mine) return;
    uint16_t* const dst = blockIdx.y ? v + row * ld_v : k + row * ld_k;
    const bool wide = reinterpret_cast<uintptr_t>(dst) % 16 == 0;
    const uint8_t* const pool = blockIdx.y ? a.v : a.k;
    const uint16_t* const scales = blockIdx.y ? a.v_scale : a.k_scale;
    const int width = a.n_kv_heads * D;
    #pragma unroll 2
    for (int e = kPiece * lane; e < width; e += 64 * kPiece) {
        const int at = e % D;
        const int64_t cache = p.cache + static_cast<int64_t>(e / D) * a.page.d;
        half8 x = {};
        if (p.cache >= 0) {
            if constexpr (KIND == MI_KV_F16) {
                x = *reinterpret_cast<const half8*>(pool + (cache * D + at) * 2);
            } else if constexpr (KIND == MI_KV_INT8) {
                const float scale = h_f(scales[cache]);
                const u32x2 w = *reinterpret_cast<const u32x2*>(pool + cache * D + at);
                #pragma unroll
                for (int z = 0; z < 8; ++z)
                    x[z] = static_cast<_Float16>(static_cast<float>(static_cast<int8_t>(w[z / 4] >> (8 * (z % 4)))) * scale);
            } else {
                const float scale = h_f(scales[cache * (D / 32) + at / 32]);
                const uint32_t w = *reinterpret_cast<const uint32_t*>(pool + (cache * D + at) / 2);
                #pragma unroll
                for (int z = 0; z < 8; ++z) x[z] = static_cast<_Float16>(static_cast<float>(static_cast<int>(w >> (4 * z) & 15) - 8) * scale);
            }
        }
        if (wide) *reinterpret_cast<half8*>(dst + e) = x;
        else
            #pragma unroll
            for (int z = 0; z < 8; ++z) dst[e + z] = __builtin_bit_cast(uint16_t, static_cast<_Float16>(x[z]));
    }
}

// Blocks for one wavefront per row of keys; 0 (and said): more than a grid counts.
unsigned blocks_for(const char* who, const PagedArgs& a) {
    const int64_t blocks = (a.n_tokens + static_cast<int64_t>(kThreads / 64) - 1) / (kThreads / 64);
    if (blocks <= 0x7fffffff / kThreads) return static_cast<unsigned>(blocks);
    MI_ERROR_FMT("%s: %d rows are more than a launch counts", who, a.n_tokens);
    return 0;
}

bool bad_rows(const char* who, const void* k, int ld_k, const void* v, int ld_v, const PagedArgs& a, int D) {
    const int64_t width = static_cast<int64_t>(a.n_kv_heads) * D;
    if (width > 0x7fffffff - 64 * kPiece) {            // (the kernels count elements of a row in ints, a wavefront's past the last)
        MI_ERROR_FMT("%s: rows of %lld elements are more than a launch counts", who, static_cast<long long>(width));
        return true;
    }
    if (k && v && ld_k >= width && ld_v >= width && reinterpret_cast<uintptr_t>(k) % 2 == 0 && reinterpret_cast<uintptr_t>(v) % 2 == 0)
        return false;
    MI_ERROR_FMT("%s: bad rows (k=%p ld_k=%d v=%p ld_v=%d, %lld elements each)", who, k, ld_k, v, ld_v, static_cast<long long>(width));
    return true;
}

}  // namespace

bool paged_args(const char* who, const mi_kv_cache* c, const mi_kv_batch* b, PagedArgs* out) {
    if (!c || !b) {
        MI_ERROR_FMT("%s: null cache or batch", who);
        return false;
    }
    const bool quantised = c->kind == MI_KV_INT8 || c->kind == MI_KV_Q4;
    if ((c->kind != MI_KV_F16 && !quantised) || (c->head_dim != 64 && c->head_dim != 128) || c->n_pages < 1 || c->page_size < 1 ||
        c->n_kv_heads < 1) {
        MI_ERROR_FMT("%s: bad cache (kind=%d n_pages=%d page_size=%d n_kv_heads=%d head_dim=%d)", who, c->kind, c->n_pages,
                     c->page_size, c->n_kv_heads, c->head_dim);
        return false;
    }
    const auto off = [](const void* p, uintptr_t align) { return !p || reinterpret_cast<uintptr_t>(p) % align; };
    if (off(c->k, 16) || off(c->v, 16) || (quantised && (off(c->k_scale, 8) || off(c->v_scale, 8)))) {
        MI_ERROR_FMT("%s: pools must be 16-byte aligned, scales 8-byte (k=%p v=%p k_scale=%p v_scale=%p)", who, c->k, c->v, c->k_scale,
                     c->v_scale);
        return false;
    }
    const double page_bytes = static_cast<double>(c->n_kv_heads) * c->page_size * row_bytes(c->kind, c->head_dim);
    if (page_bytes >= 2147483648.0) {
        MI_ERROR_FMT("%s: a page of %.0f bytes (less than 2 GiB are taken)", who, page_bytes);
        return false;
    }
    if (b->n_seqs < 0 || b->n_tokens < 0 || b->max_pages < 1 ||
        (b->n_seqs > 0 && (off(b->q_start, 4) || off(b->kv_len, 4) || off(b->pages, 4)))) {
        MI_ERROR_FMT("%s: bad batch (n_seqs=%d n_tokens=%d max_pages=%d q_start=%p kv_len=%p pages=%p)", who, b->n_seqs, b->n_tokens,
                     b->max_pages, static_cast<const void*>(b->q_start), static_cast<const void*>(b->kv_len),
                     static_cast<const void*>(b->pages));
        return false;
    }
    PagedArgs a{};
    a.k = static_cast<const uint8_t*>(c->k);
    a.v = static_cast<const uint8_t*>(c->v);
    a.k_scale = static_cast<const uint16_t*>(c->k_scale);
    a.v_scale = static_cast<const uint16_t*>(c->v_scale);
    a.q_start = b->q_start;
    a.kv_len = b->kv_len;
    a.pages = b->pages;
    a.n_seqs = b->n_seqs;
    a.n_tokens = b->n_tokens;
    a.max_pages = b->max_pages;
    a.n_pages = c->n_pages;
    a.n_kv_heads = c->n_kv_heads;
    a.cap = capacity(b->max_pages, c->page_size);
    a.page = make_divider(c->page_size);
    *out = a;
    return true;
}

#define MI_KV_LAUNCH(KERNEL, K, V)                                                                                                   \
    [&] {                                                                                                                            \
        const dim3 grid(blocks, 2), block(kThreads);                                                                                 \
        const auto s = static_cast<hipStream_t>(stream);                                                                             \
        auto go = [&](auto kern) { hipLaunchKernelGGL(kern, grid, block, 0, s, a, K, V, ld_k, ld_v); };                              \
        const bool wide = cache->head_dim == 128;                                                                                    \
        if (cache->kind == MI_KV_F16) wide ? go(KERNEL<MI_KV_F16, 128>) : go(KERNEL<MI_KV_F16, 64>);                                 \
        else if (cache->kind == MI_KV_INT8) wide ? go(KERNEL<MI_KV_INT8, 128>) : go(KERNEL<MI_KV_INT8, 64>);                         \
        else wide ? go(KERNEL<MI_KV_Q4, 128>) : go(KERNEL<MI_KV_Q4, 64>);                                                            \
        return MI_HIP_OK(hipGetLastError()) ? 1 : 0;                                                                                 \
    }()

}  // namespace mi

using namespace mi;

extern "C" int mi_kv_write(void* stream, const mi_kv_cache* cache, const mi_kv_batch* batch, const void* k, int ld_k, const void* v, int ld_v) {
    PagedArgs a;
    if (!paged_args("mi_kv_write", cache, batch, &a) || bad_rows("mi_kv_write", k, ld_k, v, ld_v, a, cache->head_dim)) return 0;
    if (a.n_seqs == 0 || a.n_tokens == 0) return 1;
    const unsigned blocks = blocks_for("mi_kv_write", a);
    if (!blocks) return 0;
    if (!ensure_init()) return 0;
    return MI_KV_LAUNCH(kv_write_kernel, static_cast<const uint16_t*>(k), static_cast<const uint16_t*>(v));
}

extern "C" int mi_kv_read(void* stream, const mi_kv_cache* cache, const mi_kv_batch* batch, void* k, int ld_k, void* v, int ld_v) {
    PagedArgs a;
    if (!paged_args("mi_kv_read", cache, batch, &a) || bad_rows("mi_kv_read", k, ld_k, v, ld_v, a, cache->head_dim)) return 0;
    if (a.n_seqs == 0 || a.n_tokens == 0) return 1;
    const unsigned blocks = blocks_for("mi_kv_read", a);
    if (!blocks) return 0;
    if (!ensure_init()) return 0;
    return MI_KV_LAUNCH(kv_read_kernel, static_cast<uint16_t*>(k), static_cast<uint16_t*>(v));
}

namespace {

// Checks a call of mi_attention, or of `who` which goes by the same, and makes the kernels' form.  1: to be launched, 0: nothing to do, -1:
// refused.
int attention_args(const char* who, const mi_attention_call& c, AttentionArgs& a) {
    PagedArgs p;
    if (!paged_args(who, c.cache, c.batch, &p)) return -1;
    const int64_t width = static_cast<int64_t>(c.n_heads) * c.cache->head_dim;
    if (c.n_heads < 1 || c.n_heads % p.n_kv_heads || !c.q || !c.out || c.ld_q < width || c.ld_out < width ||
        reinterpret_cast<uintptr_t>(c.q) % 2 || reinterpret_cast<uintptr_t>(c.out) % 2) {
        MI_ERROR_FMT("%s: bad argument (n_heads=%d over %d q=%p ld_q=%d out=%p ld_out=%d)", who, c.n_heads, p.n_kv_heads, c.q, c.ld_q,
                     c.out, c.ld_out);
        return -1;
    }
    if (!(c.scale > 0.0f && c.scale <= 65504.0f) || c.sinks < 0) {
        MI_ERROR_FMT("%s: bad argument (scale=%g, window=%d, sinks=%d)", who, static_cast<double>(c.scale), c.window, c.sinks);
        return -1;
    }
    if (p.n_seqs == 0 || p.n_tokens == 0) return 0;
    if (static_cast<int64_t>(p.n_tokens) * c.n_heads > 0x3fffffff) {
        MI_ERROR_FMT("%s: %d rows of %d heads are more than a launch counts", who, p.n_tokens, c.n_heads);
        return -1;
    }
    a.p = p;
    a.q = static_cast<const uint16_t*>(c.q);
    a.out = static_cast<uint16_t*>(c.out);
    a.ld_q = c.ld_q;
    a.ld_out = c.ld_out;
    a.n_heads = c.n_heads;
    a.kind = c.cache->kind;
    a.head_dim = c.cache->head_dim;
    a.max_tokens = c.batch->max_tokens;
    a.window = c.window;
    a.sinks = c.sinks;
    a.scale = c.scale;
    return 1;
}

}  // namespace

extern "C" int mi_attention(void* stream, const mi_attention_call* call) {
    if (!call) {
        MI_ERROR_FMT("mi_attention: null call");
        return 0;
    }
    AttentionArgs a{};
    const int todo = attention_args("mi_attention", *call, a);
    if (todo <= 0) return todo == 0;
    if (!ensure_init()) return 0;
    const auto s = static_cast<hipStream_t>(stream);
    return launch_paged_attention(s, a, stream_room(s)) ? 1 : 0;
}

extern "C" int mi_attention_tree(void* stream, const mi_attention_call* call, const mi_tree_mask* tree) {
    if (!call || !tree) {
        MI_ERROR_FMT("mi_attention_tree: null call or tree");
        return 0;
    }
    TreeArgs a{};
    const int todo = attention_args("mi_attention_tree", *call, a);
    if (todo < 0) return 0;
    if (tree->words < 1 || tree->words > 65536) {
        MI_ERROR_FMT("mi_attention_tree: bad argument (words=%d)", tree->words);
        return 0;
    }
    if (todo == 0) return 1;
    const bool windowed = call->window > 0;
    if (!tree->seen || reinterpret_cast<uintptr_t>(tree->seen) % 4 || (windowed && !tree->position) ||
        reinterpret_cast<uintptr_t>(tree->position) % 4) {
        MI_ERROR_FMT("mi_attention_tree: bad argument (seen=%p position=%p window=%d)", static_cast<const void*>(tree->seen),
                     static_cast<const void*>(tree->position), call->window);
        return 0;
    }
    if (!ensure_init()) return 0;
    a.seen = tree->seen;
    a.position = tree->position;
    a.words = tree->words;
    const auto s = static_cast<hipStream_t>(stream);
    return launch_paged_tree(s, a, stream_room(s)) ? 1 : 0;
}
