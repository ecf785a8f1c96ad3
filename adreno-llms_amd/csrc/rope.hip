// Rotary positions of new rows (mi_rope): a pair (x, y) of a head becomes (x cos a - y sin a, y cos a + x sin a), a = position * inv_freq of the
// pair, between a batch's projections and its cache.  (The decoders' own rotary embedding, with its tables of rounded cosines, is
// in decode.hip.)
//
// An angle of position 10^6 is known to 2^-4 in fp32, so it is taken in 64 bits and what their roundings leave, in turns (rope_rule.h), and its cosine
// and sine are fp32's.  All heads of a row turn by the same angles, which a wavefront works out once, a pair per lane, and hands round in LDS.
//
// What bounds it: bytes where there are many rows, 84 MB of 4096 rows of 32 + 8 heads of 128 in 14.3 us (16.4 with rows that no cache holds, a
// large copy's rate); below about 2000 rows the host's call (6.5 us; on the GPU 16 rows 3.3: the launch, the positions, the angles).  An
// output is rounded once, from the fp32 sum.
#include "../../include/mi_attention.h"
#include "common.h"
#include "device_math.h"
#include "rope_rule.h"

namespace mi {
namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef float floatx4 __attribute__((ext_vector_type(4)));

constexpr int kWaves = 4, kMostPairs = 128;

struct RopeArgs {
    const uint16_t *q, *k;
    uint16_t *q_out, *k_out;
    const float* inv_freq;
    const int* position;
    int64_t ld_q, ld_k, ld_q_out, ld_k_out;
    int n_tokens, n_heads, heads, head_dim, pairs;     // heads: of q and k
    uint32_t axis[kMostPairs / 16];                    // of a pair, 2 bits each
};

// Cosines and sines of a row's pairs, to `turn` [2][kMostPairs].
__device__ __forceinline__ void angles(const RopeArgs& a, int row, int lane, float* turn) {
    for (int i = lane; i < a.pairs; i += 64) {
        const int axis = a.axis[i / 16] >> (i % 16 * 2) & 3;
        const float f = 2.0f * static_cast<float>(turns_of<>(a.position[static_cast<int64_t>(axis) * a.n_tokens + row], a.inv_freq[i]));
        turn[i] = cospif(f);
        turn[kMostPairs + i] = sinpif(f);
    }
}
__device__ __forceinline__ float turned_x(float x, float y, float c, float s) { return fmaf(x, c, -(y * s)); }
__device__ __forceinline__ float turned_y(float x, float y, float c, float s) { return fmaf(y, c, x * s); }

__device__ __forceinline__ const uint16_t* from(const RopeArgs& a, int row, int head) {
    return head < a.n_heads ? a.q + row * a.ld_q + head * a.head_dim : a.k + row * a.ld_k + (head - a.n_heads) * a.head_dim;
}
__device__ __forceinline__ uint16_t* to(const RopeArgs& a, int row, int head) {
    return head < a.n_heads ? a.q_out + row * a.ld_q_out + head * a.head_dim : a.k_out + row * a.ld_k_out + (head - a.n_heads) * a.head_dim;
}

// A wavefront has a row, a lane 16 elements of a head at a time: 8 pairs, or 16 of those behind them.  Where all rows and halves are whole
// pieces of 16 bytes (4096 rows of 32 + 8 heads of 128: 14.3 us, a pair at a time as below 27.6).
template <bool SPLIT>
__global__ __launch_bounds__(64 * kWaves) void rope_wide_kernel(const RopeArgs a) {
    __shared__ __attribute__((aligned(16))) float turn[kWaves][2 * kMostPairs];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int row = blockIdx.x * kWaves + wave;
    if (row >= a.n_tokens) return;
    const int each = a.head_dim / 16, turning = a.pairs / 8, n = a.heads * each;
    struct Piece {
        half8 x, y;
        int at_x, at_y, i;                         // elements of the head; first pair, -1: none
        uint16_t* dst;
    };
    auto load = [&](int z) {
        Piece p;
        const int head = z / each, c = z - head * each;
        const uint16_t* const src = from(a, row, head);
        p.dst = to(a, row, head);
        p.i = c < turning ? 8 * c : -1;
        p.at_x = SPLIT && c < turning ? 8 * c : 16 * c;
        p.at_y = SPLIT && c < turning ? 8 * c + a.pairs : 16 * c + 8;
        p.x = *reinterpret_cast<const half8*>(src + p.at_x);
        p.y = *reinterpret_cast<const half8*>(src + p.at_y);
        return p;
    };
    auto finish = [&](Piece p) {
        if (p.i >= 0) {
            float c[8], s[8];
            #pragma unroll
            for (int e = 0; e < 8; e += 4) {
                const floatx4 cs = *reinterpret_cast<const floatx4*>(&turn[wave][p.i + e]);
                const floatx4 sn = *reinterpret_cast<const floatx4*>(&turn[wave][kMostPairs + p.i + e]);
                #pragma unroll
                for (int z = 0; z < 4; ++z) c[e + z] = cs[z], s[e + z] = sn[z];
            }
            #pragma unroll
            for (int e = 0; e < 8; ++e) {
                _Float16 &x = SPLIT ? reinterpret_cast<_Float16*>(&p.x)[e] : e < 4 ? reinterpret_cast<_Float16*>(&p.x)[2 * e] : reinterpret_cast<_Float16*>(&p.y)[2 * e - 8];
                _Float16 &y = SPLIT ? reinterpret_cast<_Float16*>(&p.y)[e] : e < 4 ? reinterpret_cast<_Float16*>(&p.x)[2 * e + 1] : reinterpret_cast<_Float16*>(&p.y)[2 * e - 7];
                const float fx = static_cast<float>(x), fy = static_cast<float>(y);
                x = static_cast<_Float16>(turned_x(fx, fy, c[e], s[e]));
                y = static_cast<_Float16>(turned_y(fx, fy, c[e], s[e]));
            }
        }
        *reinterpret_cast<half8*>(p.dst + p.at_x) = p.x;
        *reinterpret_cast<half8*>(p.dst + p.at_y) = p.y;
    };
    // (the first two pieces are on their way while the angles are worked out)
    Piece now{}, next{};
    if (lane < n) now = load(lane);
    if (lane + 64 < n) next = load(lane + 64);
    angles(a, row, lane, turn[wave]);
    __builtin_amdgcn_wave_barrier();
    for (int z = lane; z < n; z += 64) {
        Piece after{};
        if (z + 128 < n) after = load(z + 128);
        finish(now);
        now = next;
        next = after;
    }
}

// The same for any rows, a lane one pair after the other, two bytes a load: rows that begin, or lie apart, at other than multiples of 16 bytes,
// heads or turned parts of them that are no multiple of 16 elements (4096 rows of 9 + 3 heads of 72 7.0 us, the host's call and little more).
template <bool SPLIT>
__global__ __launch_bounds__(64 * kWaves) void rope_kernel(const RopeArgs a) {
    __shared__ float turn[kWaves][2 * kMostPairs];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int row = blockIdx.x * kWaves + wave;
    if (row >= a.n_tokens) return;
    angles(a, row, lane, turn[wave]);
    __builtin_amdgcn_wave_barrier();
    const int rest = a.head_dim - 2 * a.pairs, each = a.pairs + rest, n = a.heads * each;
    for (int z = lane; z < n; z += 64) {
        const int head = z / each, i = z - head * each;
        const uint16_t* const src = from(a, row, head);
        uint16_t* const dst = to(a, row, head);
        if (i >= a.pairs) {
            dst[a.pairs + i] = src[a.pairs + i];
            continue;
        }
        const int at_x = SPLIT ? i : 2 * i, at_y = SPLIT ? i + a.pairs : 2 * i + 1;
        const float x = h_f(src[at_x]), y = h_f(src[at_y]), c = turn[wave][i], s = turn[wave][kMostPairs + i];
        dst[at_x] = f_h(turned_x(x, y, c, s));
        dst[at_y] = f_h(turned_y(x, y, c, s));
    }
}

}  // namespace
}  // namespace mi

using namespace mi;

extern "C" int mi_rope(void* stream, const mi_rope_call* call) {
    if (!call) {
        MI_ERROR_FMT("mi_rope: null call");
        return 0;
    }
    const mi_rope_call& c = *call;
    if (c.n_tokens < 0 || c.n_heads < 0 || c.n_kv_heads < 0 || c.head_dim < 2 || c.head_dim > 2 * kMostPairs || c.head_dim % 2 ||
        c.rot_dim < 0 || c.rot_dim > c.head_dim || c.rot_dim % 2 || c.n_axes < 1 || c.n_axes > 4) {
        MI_ERROR_FMT("mi_rope: bad argument (n_tokens=%d n_heads=%d n_kv_heads=%d head_dim=%d rot_dim=%d n_axes=%d)", c.n_tokens, c.n_heads,
                     c.n_kv_heads, c.head_dim, c.rot_dim, c.n_axes);
        return 0;
    }
    const auto off = [](const void* p, uintptr_t align) { return !p || reinterpret_cast<uintptr_t>(p) % align; };
    const auto bad = [&](const char* name, int heads, const void* in, int ld_in, const void* out, int ld_out) {
        const int64_t width = static_cast<int64_t>(heads) * c.head_dim;
        if (heads == 0 || (!off(in, 2) && !off(out, 2) && ld_in >= width && ld_out >= width && (in != out || ld_in == ld_out))) return false;
        MI_ERROR_FMT("mi_rope: bad rows (%s=%p ld=%d out=%p ld=%d, %lld elements each)", name, in, ld_in, out, ld_out,
                     static_cast<long long>(width));
        return true;
    };
    if (bad("q", c.n_heads, c.q, c.ld_q, c.q_out, c.ld_q_out) || bad("k", c.n_kv_heads, c.k, c.ld_k, c.k_out, c.ld_k_out)) return 0;
    RopeArgs a{};
    a.pairs = c.rot_dim / 2;
    for (int i = 0; c.axis && i < a.pairs; ++i) {
        if (c.axis[i] >= c.n_axes) {
            MI_ERROR_FMT("mi_rope: bad argument (axis[%d]=%d of %d)", i, c.axis[i], c.n_axes);
            return 0;
        }
        a.axis[i / 16] |= static_cast<uint32_t>(c.axis[i]) << (i % 16 * 2);
    }
    const int64_t heads = static_cast<int64_t>(c.n_heads) + c.n_kv_heads;
    if (heads * c.head_dim > 0x3fffffff || static_cast<int64_t>(c.n_tokens) > 0x3fffffff) {
        MI_ERROR_FMT("mi_rope: %d rows of %lld heads are more than a launch counts", c.n_tokens, static_cast<long long>(heads));
        return 0;
    }
    if (c.n_tokens == 0 || heads == 0) return 1;
    if (a.pairs > 0 && (off(c.inv_freq, 4) || off(c.position, 4))) {
        MI_ERROR_FMT("mi_rope: bad argument (inv_freq=%p position=%p)", static_cast<const void*>(c.inv_freq), static_cast<const void*>(c.position));
        return 0;
    }
    a.q = static_cast<const uint16_t*>(c.q);
    a.k = static_cast<const uint16_t*>(c.k);
    a.q_out = static_cast<uint16_t*>(c.q_out);
    a.k_out = static_cast<uint16_t*>(c.k_out);
    a.inv_freq = c.inv_freq;
    a.position = c.position;
    a.ld_q = c.ld_q;
    a.ld_k = c.ld_k;
    a.ld_q_out = c.ld_q_out;
    a.ld_k_out = c.ld_k_out;
    a.n_tokens = c.n_tokens;
    a.n_heads = c.n_heads;
    a.heads = static_cast<int>(heads);
    a.head_dim = c.head_dim;
    const int64_t blocks = (static_cast<int64_t>(a.n_tokens) + kWaves - 1) / kWaves;
    if (blocks > 0x7fffffff / (64 * kWaves)) {
        MI_ERROR_FMT("mi_rope: %d rows are more than a launch counts", c.n_tokens);
        return 0;
    }
    if (!ensure_init()) return 0;
    const auto go = [&](auto kern) {
        hipLaunchKernelGGL(kern, dim3(static_cast<unsigned>(blocks)), dim3(64 * kWaves), 0, static_cast<hipStream_t>(stream), a);
    };
    const auto whole = [&](const void* p, int ld, int of) { return of == 0 || (reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld % 8 == 0); };
    const bool wide = c.head_dim % 16 == 0 && c.rot_dim % 16 == 0 && whole(c.q, c.ld_q, c.n_heads) && whole(c.q_out, c.ld_q_out, c.n_heads) &&
                      whole(c.k, c.ld_k, c.n_kv_heads) && whole(c.k_out, c.ld_k_out, c.n_kv_heads);
    if (wide) c.interleaved ? go(rope_wide_kernel<false>) : go(rope_wide_kernel<true>);
    else c.interleaved ? go(rope_kernel<false>) : go(rope_kernel<true>);
    return MI_HIP_OK(hipGetLastError()) ? 1 : 0;
}
