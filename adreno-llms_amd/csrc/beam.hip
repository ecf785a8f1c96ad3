// Beam search's choice (mi_beam_select): of a group's rows of logits the n_out greatest of score[r] + x[r][t] - log sum exp x[r][.].
//
// One pass over the logits: a wavefront has a tile of 4096 in registers, takes the sum of their exponentials relative to the tile's
// greatest and the greatest of each lane's 64 (a bin), a 64th of what it read.  A row's best n_out then lie in bins that reach the
// n_out-th greatest of a wavefront's maxima over all bins, some 20 of 2400, which are read again.  Within a row the order is that of the
// fp16 logits themselves, ties by token; rows of a group are merged by sums in 64 bits, which a near tie of two beams turns on.
#include "../../include/mi_linear.h"
#include "beam_rule.h"
#include "common.h"
#include "device_math.h"

namespace mi {
namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef uint16_t ushort8 __attribute__((ext_vector_type(8)));

constexpr float kLog2e = 1.44269504088896341f;
constexpr int kScanWaves = 4, kPickWaves = 8;
constexpr int kList = 256, kBinList = 1024;        // of a wavefront that picks: candidates, bins

struct BeamArgs {
    const uint16_t* logits;
    const float* score;
    float* out_score;
    int *out_token, *out_row;
    int64_t ld;
    int beams, vocab, n_out, tiles;
    int first;                                     // group of the launch's first
    int64_t rows;                                  // of the launch
};

template <class T>
__device__ __forceinline__ T sum_of_wave(T x) {
    #pragma unroll
    for (int s = 32; s > 0; s /= 2) x += __shfl_xor(x, s);
    return x;
}

// Tile `tile` of a row: its sum and reference, and the lane's bin.
struct Scanned {
    float top, sum;            // its greatest logit (-65504 of -infinities), the sum of 2^scaled(x, top)
    uint32_t bin;
};
// x log2 e less the rounded top log2 e, in one rounding: the second's own, up to 2^-8 where logits are in the tens of thousands, is the same in
// all of a tile, and correction() takes it out of their sum.
__device__ __forceinline__ float scaled(float x, float top_log2) { return fmaf(x, kLog2e, -top_log2); }
__device__ __forceinline__ float correction(float top) {
    return static_cast<float>(static_cast<double>(top * kLog2e) - static_cast<double>(top) * static_cast<double>(kLog2e));
}
__device__ __forceinline__ Scanned scan_tile(const uint16_t* row, int vocab, int tile) {
    const int lane = threadIdx.x & 63;
    half8 x[8];
    #pragma unroll
    for (int j = 0; j < 8; ++j) {
        const int t = token_of(tile, lane, 8 * j);
        if (t + 8 <= vocab) {
            __builtin_memcpy(&x[j], row + t, 16);
        } else {
            #pragma unroll
            for (int e = 0; e < 8; ++e) x[j][e] = t + e < vocab ? __builtin_bit_cast(_Float16, row[t + e]) : -__builtin_huge_valf();
        }
    }
    half8 top = x[0];
    #pragma unroll
    for (int j = 1; j < 8; ++j) top = __builtin_elementwise_max(top, x[j]);
    _Float16 most = top[0];
    #pragma unroll
    for (int e = 1; e < 8; ++e) most = __builtin_elementwise_max(most, top[e]);
    Scanned s;
    s.bin = ascending(__builtin_bit_cast(uint16_t, most));
    s.top = fmaxf(wave_max(static_cast<float>(most)), -65504.0f);
    const float top_log2 = s.top * kLog2e;
    float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    #pragma unroll
    for (int j = 0; j < 8; ++j)
        #pragma unroll
        for (int e = 0; e < 8; ++e) sum[e % 4] += __builtin_amdgcn_exp2f(scaled(static_cast<float>(x[j][e]), top_log2));
    s.sum = sum_of_wave((sum[0] + sum[1]) + (sum[2] + sum[3]));
    return s;
}

__global__ __launch_bounds__(64 * kScanWaves) void beam_scan_kernel(const BeamArgs a, float2* __restrict__ sums, uint16_t* __restrict__ bins) {
    const int64_t item = static_cast<int64_t>(blockIdx.x) * kScanWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t row = item / a.tiles;
    if (row >= a.rows) return;
    const int lane = threadIdx.x & 63;
    const Scanned s = scan_tile(a.logits + (static_cast<int64_t>(a.first) * a.beams + row) * a.ld, a.vocab, static_cast<int>(item - row * a.tiles));
    bins[item * kBins + lane] = static_cast<uint16_t>(s.bin);
    if (lane == 0) sums[item] = float2{s.top, s.sum};
}

// A candidate: the logit above, the complement of its token below, so that the greater is the better one, ties to the lower token.
__device__ __forceinline__ uint64_t candidate(uint32_t value, int token) { return static_cast<uint64_t>(value) << 32 | ~static_cast<uint32_t>(token); }

struct PickRoom {
    uint64_t list[kList];
    uint16_t bins[kBinList];
};

// The best n of a wavefront's `count` candidates in order, in place; how many there are.
__device__ __forceinline__ int best_of(uint64_t* list, int count, int n) {
    const int lane = threadIdx.x & 63;
    constexpr int kEach = kList / 64;
    uint64_t mine[kEach];
    int rank[kEach];
    #pragma unroll
    for (int u = 0; u < kEach; ++u) {
        mine[u] = u * 64 + lane < count ? list[u * 64 + lane] : 0;
        rank[u] = 0;
    }
    for (int z = 0; z < count; ++z) {
        const uint64_t other = list[z];
        #pragma unroll
        for (int u = 0; u < kEach; ++u) rank[u] += other > mine[u];
    }
    __builtin_amdgcn_wave_barrier();
    #pragma unroll
    for (int u = 0; u < kEach; ++u)
        if (u * 64 + lane < count && rank[u] < n) list[rank[u]] = mine[u];
    __builtin_amdgcn_wave_barrier();
    return count < n ? count : n;
}

// What a row's candidates count beside their logits (NaN or infinite: the row has none), from its tiles' sums.
__device__ __forceinline__ double offset_of(const float2* sums, int tiles, float score) {
    const int lane = threadIdx.x & 63;
    float top = -__builtin_huge_valf();
    for (int t = lane; t < tiles; t += 64) top = fmaxf(top, sums[t].x);
    top = wave_max(top);
    double sum = 0.0;
    for (int t = lane; t < tiles; t += 64) {
        const float2 s = sums[t];
        sum += static_cast<double>(s.y) * static_cast<double>(__builtin_amdgcn_exp2f(fmaf(s.x - top, kLog2e, correction(s.x))));
    }
    sum = sum_of_wave(sum);
    return static_cast<double>(score) - (static_cast<double>(top) + log(sum));
}

// The best n of a row's logits to room.list, in order; how many there are.
__device__ __forceinline__ int pick(const uint16_t* row, int vocab, int tiles, const uint16_t* bins, int n, PickRoom& room) {
    const int lane = threadIdx.x & 63, all = tiles * kBins;
    // n lanes have a bin that reaches `least`, so the best n candidates do
    uint32_t most = 0;
    for (int f = 8 * lane; f < all; f += 8 * 64) {
        const ushort8 b = *reinterpret_cast<const ushort8*>(bins + f);
        #pragma unroll
        for (int e = 0; e < 8; ++e) most = b[e] > most ? b[e] : most;
    }
    uint32_t least = 0;
    #pragma unroll
    for (int bit = 0x8000; bit > 0; bit /= 2)
        if (__popcll(__ballot(most >= (least | bit))) >= n) least |= bit;
    if (least < kLeast) least = kLeast;
    uint64_t above = static_cast<uint64_t>(least) << 32;         // (a token's complement is never 0)
    int count = 0, listed = 0;
    auto take = [&] {                                            // the listed bins' logits
        for (int z0 = 0; z0 < listed; z0 += 4) {
            uint32_t value[4];
            int token[4];
            #pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int f = room.bins[z0 + u < listed ? z0 + u : listed - 1];
                token[u] = token_of(f / kBins, f % kBins, lane);
                value[u] = token[u] < vocab ? ascending(row[token[u]]) : 0;
            }
            #pragma unroll
            for (int u = 0; u < 4; ++u) {
                if (z0 + u >= listed) break;
                if (count > kList - 64) {
                    count = best_of(room.list, count, n);
                    if (count == n) above = room.list[n - 1];
                }
                const uint64_t c = candidate(value[u], token[u]);
                const uint64_t in = __ballot(c > above);
                if (c > above) room.list[count + __popcll(in & ((1ull << lane) - 1))] = c;
                count += __popcll(in);
                __builtin_amdgcn_wave_barrier();
            }
        }
        listed = 0;
    };
    for (int f0 = 0; f0 < all; f0 += 8 * 64) {
        const int f = f0 + 8 * lane;
        ushort8 b = {};
        if (f < all) b = *reinterpret_cast<const ushort8*>(bins + f);
        #pragma unroll
        for (int e = 0; e < 8; ++e) {
            const uint64_t in = __ballot(b[e] >= least);
            if (b[e] >= least) room.bins[listed + __popcll(in & ((1ull << lane) - 1))] = static_cast<uint16_t>(f + e);
            listed += __popcll(in);
        }
        __builtin_amdgcn_wave_barrier();
        if (listed > kBinList - 512) take();
    }
    take();
    return best_of(room.list, count, n);
}

// The rows' best, merged by one wavefront: lane r has row r's, the best first.
__device__ __forceinline__ void merge(const BeamArgs& a, int64_t group, const uint64_t* lists, const int* counts, const double* offsets) {
    const int lane = threadIdx.x & 63;
    const int count = lane < a.beams ? counts[lane] : 0;
    const double offset = lane < a.beams ? offsets[lane] : 0.0;
    const uint64_t* const list = lists + (lane < a.beams ? lane : 0) * a.n_out;
    int at = 0;
    const double none = -__builtin_huge_val();
    auto value_at = [&](int i, uint64_t c) {
        return i < count ? offset + static_cast<double>(h_f(static_cast<uint16_t>(half_bits(static_cast<uint32_t>(c >> 32))))) : none;
    };
    uint64_t here = list[0];
    double value = value_at(0, here);
    for (int i = 0; i < a.n_out; ++i) {
        double best = value;
        #pragma unroll
        for (int s = 32; s > 0; s /= 2) best = fmax(best, __shfl_xor(best, s));
        const uint64_t who = __ballot(value == best && best > none);
        const int winner = who ? __builtin_ctzll(who) : 0;
        if (lane == winner) {
            const int64_t to = group * a.n_out + i;
            a.out_score[to] = static_cast<float>(best);
            a.out_token[to] = who ? static_cast<int>(~static_cast<uint32_t>(here)) : -1;
            a.out_row[to] = who ? static_cast<int>(group * a.beams) + lane : -1;
            ++at;
            here = list[at < a.n_out ? at : 0];
            value = value_at(at, here);
        }
    }
}

// LDS of a block that picks: the rows' lists, then what is said of each.
struct Picked {
    uint64_t* lists;
    double* offsets;
    int* counts;
    __device__ Picked(uint8_t* lds, const BeamArgs& a)
        : lists(reinterpret_cast<uint64_t*>(lds)), offsets(reinterpret_cast<double*>(lds) + a.beams * a.n_out),
          counts(reinterpret_cast<int*>(offsets + a.beams)) {}
};
constexpr size_t picked_bytes(int beams, int n_out) { return static_cast<size_t>(beams) * (8 * n_out + 8 + 4) + 4 * (beams % 2); }

// Row r of a group: its list, by one wavefront.
__device__ __forceinline__ void pick_row(const BeamArgs& a, int64_t group, int r, const float2* sums, const uint16_t* bins, PickRoom& room, const Picked& to) {
    const int lane = threadIdx.x & 63;
    const int64_t row = group * a.beams + r;
    const double offset = offset_of(sums, a.tiles, a.score[row]);
    int n = 0;
    if (fabs(offset) < __builtin_huge_val()) n = pick(a.logits + row * a.ld, a.vocab, a.tiles, bins, a.n_out, room);
    if (lane < n) to.lists[r * a.n_out + lane] = room.list[lane];
    if (lane == 0) {
        to.offsets[r] = offset;
        to.counts[r] = n;
    }
}

__global__ __launch_bounds__(64 * kPickWaves) void beam_pick_kernel(const BeamArgs a, const float2* __restrict__ sums, const uint16_t* __restrict__ bins) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    __shared__ PickRoom rooms[kPickWaves];
    const Picked picked(lds, a);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    for (int r = wave; r < a.beams; r += kPickWaves) {
        const int64_t item = (static_cast<int64_t>(blockIdx.x) * a.beams + r) * a.tiles;
        pick_row(a, static_cast<int64_t>(a.first) + blockIdx.x, r, sums + item, bins + item * kBins, rooms[wave], picked);
    }
    __syncthreads();
    if (wave == 0) merge(a, static_cast<int64_t>(a.first) + blockIdx.x, picked.lists, picked.counts, picked.offsets);
}

// Everything in one block per group, for streams that have no workspace: row by row, sums and bins in LDS.
__global__ __launch_bounds__(64 * kPickWaves) void beam_alone_kernel(const BeamArgs a) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    __shared__ PickRoom room;
    auto* const sums = reinterpret_cast<float2*>(lds);
    auto* const bins = reinterpret_cast<uint16_t*>(sums + (a.tiles + 1) / 2 * 2);
    const Picked picked(reinterpret_cast<uint8_t*>(bins + a.tiles * kBins), a);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    for (int r = 0; r < a.beams; ++r) {
        const uint16_t* const row = a.logits + (static_cast<int64_t>(blockIdx.x) * a.beams + r) * a.ld;
        for (int t = wave; t < a.tiles; t += kPickWaves) {
            const Scanned s = scan_tile(row, a.vocab, t);
            bins[t * kBins + lane] = static_cast<uint16_t>(s.bin);
            if (lane == 0) sums[t] = float2{s.top, s.sum};
        }
        __syncthreads();
        if (wave == 0) pick_row(a, blockIdx.x, r, sums, bins, room, picked);
        __syncthreads();
    }
    if (wave == 0) merge(a, blockIdx.x, picked.lists, picked.counts, picked.offsets);
}
constexpr size_t alone_bytes(int tiles) { return static_cast<size_t>((tiles + 1) / 2 * 2) * 8 + static_cast<size_t>(tiles) * kBins * 2; }
static_assert(alone_bytes(tiles_of_row(MI_BEAM_MAX_VOCAB)) + picked_bytes(kMostBeams, kMostOut) + sizeof(PickRoom) <= 160 * 1024, "fits LDS");
static_assert(picked_bytes(kMostBeams, kMostOut) + kPickWaves * sizeof(PickRoom) <= 160 * 1024, "fits LDS");
static_assert(groups_that_fit(kWorkspaceBytes, kMostBeams, MI_BEAM_MAX_VOCAB) >= 1, "a group fits the workspace");
static_assert(tiles_of_row(MI_BEAM_MAX_VOCAB) * kBins <= 65536, "a bin's number has 16 bits");
static_assert(kMostOut <= 64 && kMostOut + 64 <= kList && kMostBeams <= 64, "a lane each");

bool raise_lds(const void* kern, int bytes) {
    return MI_HIP_OK(hipFuncSetAttribute(kern, hipFuncAttributeMaxDynamicSharedMemorySize, bytes));
}

}  // namespace
}  // namespace mi

using namespace mi;

extern "C" int mi_beam_select(void* stream, const mi_beam_call* call) {
    if (!call) {
        MI_ERROR_FMT("mi_beam_select: null call");
        return 0;
    }
    const mi_beam_call& c = *call;
    if (c.n_groups < 0 || c.beams < 1 || c.beams > kMostBeams || c.n_out < 1 || c.n_out > kMostOut || c.vocab < 1 ||
        c.vocab > MI_BEAM_MAX_VOCAB || c.ld < c.vocab) {
        MI_ERROR_FMT("mi_beam_select: bad argument (n_groups=%d beams=%d n_out=%d vocab=%d ld=%d)", c.n_groups, c.beams, c.n_out, c.vocab, c.ld);
        return 0;
    }
    if (c.n_groups == 0) return 1;
    const auto off = [](const void* p, uintptr_t align) { return !p || reinterpret_cast<uintptr_t>(p) % align; };
    if (off(c.logits, 2) || off(c.score, 4) || off(c.out_score, 4) || off(c.out_token, 4) || off(c.out_row, 4)) {
        MI_ERROR_FMT("mi_beam_select: bad argument (logits=%p score=%p out_score=%p out_token=%p out_row=%p)", c.logits,
                     static_cast<const void*>(c.score), static_cast<void*>(c.out_score), static_cast<void*>(c.out_token), static_cast<void*>(c.out_row));
        return 0;
    }
    if (static_cast<int64_t>(c.n_groups) * c.beams > 0x7fffffff || c.n_groups > 0x7fffffff / (64 * kPickWaves)) {
        MI_ERROR_FMT("mi_beam_select: %d groups of %d beams are more than a launch counts", c.n_groups, c.beams);
        return 0;
    }
    if (!ensure_init()) return 0;
    BeamArgs a{};
    a.logits = static_cast<const uint16_t*>(c.logits);
    a.score = c.score;
    a.out_score = c.out_score;
    a.out_token = c.out_token;
    a.out_row = c.out_row;
    a.ld = c.ld;
    a.beams = c.beams;
    a.vocab = c.vocab;
    a.n_out = c.n_out;
    a.tiles = tiles_of_row(c.vocab);
    const auto s = static_cast<hipStream_t>(stream);
    const size_t picked = picked_bytes(c.beams, c.n_out);
    void* const workspace = stream_room(s).workspace;
    if (!workspace) {
        if (!MI_ONCE_OK(raise_lds(reinterpret_cast<const void*>(beam_alone_kernel),
                                  static_cast<int>(alone_bytes(tiles_of_row(MI_BEAM_MAX_VOCAB)) + picked_bytes(kMostBeams, kMostOut)))))
            return 0;
        hipLaunchKernelGGL(beam_alone_kernel, dim3(c.n_groups), dim3(64 * kPickWaves), alone_bytes(a.tiles) + picked, s, a);
        return MI_HIP_OK(hipGetLastError()) ? 1 : 0;
    }
    if (!MI_ONCE_OK(raise_lds(reinterpret_cast<const void*>(beam_pick_kernel), static_cast<int>(picked_bytes(kMostBeams, kMostOut))))) return 0;
    const int64_t fit = groups_that_fit(kWorkspaceBytes, c.beams, c.vocab);
    for (int64_t first = 0; first < c.n_groups; first += fit) {
        const int64_t n = c.n_groups - first < fit ? c.n_groups - first : fit, items = n * c.beams * a.tiles;
        a.first = static_cast<int>(first);
        a.rows = n * c.beams;
        auto* const bins = static_cast<uint16_t*>(workspace);
        auto* const sums = reinterpret_cast<float2*>(bins + items * kBins);
        hipLaunchKernelGGL(beam_scan_kernel, dim3(static_cast<unsigned>((items + kScanWaves - 1) / kScanWaves)), dim3(64 * kScanWaves), 0, s, a, sums,
                           bins);
        if (!MI_HIP_OK(hipGetLastError())) return 0;
        hipLaunchKernelGGL(beam_pick_kernel, dim3(static_cast<unsigned>(n)), dim3(64 * kPickWaves), picked, s, a, sums, bins);
        if (!MI_HIP_OK(hipGetLastError())) return 0;
    }
    return 1;
}
