// Beam search's choice (mi_beam_select): of a group's rows of logits the n_out greatest of score[r] + x[r][t] - log sum exp x[r][.].
//
// One pass over the logits: a wavefront has a tile of 4096 in registers, takes the sum of their exponentials relative to the tile's
// greatest and the greatest of each lane's 64 (a bin), a 64th of what it read.  A row's best n_out then lie in bins that reach the
// n_out-th greatest of a wavefront's maxima over all bins, some 20 of 2400, which are read again.  Within a row the order is that of the
// fp16 logits themselves, ties by token; rows of a group are merged by sums in 64 bits, of which a row's logarithm has the
// error of fp32's exponentials.
//
// What bounds it: the pass over many logits by memory, 78 MB of 256 rows of 151 936 in 14.2 us, 5.4 TB/s (an exponential takes 16 cycles of a
// SIMD, a logit 26 in all: 7 us of the vector units); behind it, and for few rows, a chain that a group's block goes through once: 5 us for 4 rows, 7.5
// for 8 rows by 32 groups, of which two answers of memory (bins, logits) are 1.5 and 2.9 and the rest instructions of one
// wavefront, eight cycles each; rows of one or two tiles: see pick_crowded.  Before offers that share a place were told apart among themselves it was 11 for 8 rows; with candidates in
// order and merged one list after the other 7 and 14; with calls of functions, which need scratch memory, 9 and 24.  Error of the sum: 3e-8 of a score near -20.
#include "../../include/mi_linear.h"
#include "beam_rule.h"
#include "common.h"
#include "device_math.h"

#include <type_traits>

namespace mi {
namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef uint16_t ushort8 __attribute__((ext_vector_type(8)));
typedef int16_t short8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

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
    int first, rows;                               // group of the launch's first; rows of the launch
};

// Sum of all lanes, in each of them.
__device__ __forceinline__ double sum_of_wave(double x) {
    const auto add = [&](auto ctrl, auto rows) {
        const uint64_t u = __builtin_bit_cast(uint64_t, x);
        const uint32_t lo = __builtin_amdgcn_update_dpp(0, static_cast<uint32_t>(u), decltype(ctrl)::value, decltype(rows)::value, 0xf, false);
        const uint32_t hi = __builtin_amdgcn_update_dpp(0, static_cast<uint32_t>(u >> 32), decltype(ctrl)::value, decltype(rows)::value, 0xf, false);
        x += __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
    };
    using std::integral_constant;
    add(integral_constant<int, 0x111>{}, integral_constant<int, 0xf>{});       // from 1, 2, 4, 8 lanes below, in rows of 16
    add(integral_constant<int, 0x112>{}, integral_constant<int, 0xf>{});
    add(integral_constant<int, 0x114>{}, integral_constant<int, 0xf>{});
    add(integral_constant<int, 0x118>{}, integral_constant<int, 0xf>{});
    add(integral_constant<int, 0x142>{}, integral_constant<int, 0xa>{});       // row 0's last lane to row 1, 2's to 3
    add(integral_constant<int, 0x143>{}, integral_constant<int, 0xc>{});       // lane 31 to rows 2 and 3
    const uint64_t u = __builtin_bit_cast(uint64_t, x);
    const uint32_t lo = __builtin_amdgcn_readlane(static_cast<uint32_t>(u), 63), hi = __builtin_amdgcn_readlane(static_cast<uint32_t>(u >> 32), 63);
    return __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
}
// Sum of the lanes up to a lane's own.
__device__ __forceinline__ int scan(int x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);
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
    s.sum = wave_tree_sum((sum[0] + sum[1]) + (sum[2] + sum[3]));
    return s;
}

__global__ __launch_bounds__(64 * kScanWaves) void beam_scan_kernel(const BeamArgs a, float2* __restrict__ sums, uint16_t* __restrict__ bins) {
    const int item = blockIdx.x * kScanWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), row = item / a.tiles;      // (few: they fit the workspace)
    if (row >= a.rows) return;
    const int lane = threadIdx.x & 63;
    const Scanned s = scan_tile(a.logits + (static_cast<int64_t>(a.first) * a.beams + row) * a.ld, a.vocab, item - row * a.tiles);
    bins[item * kBins + lane] = static_cast<uint16_t>(s.bin);
    if (lane == 0) sums[item] = float2{s.top, s.sum};
}

// ---- what a row offers ---------------------------------------------------------------------------------------

// A candidate: the logit above, the complement of its token below, so that the greater is the better one, ties to the lower token.
__device__ __forceinline__ uint64_t candidate(uint32_t value, int token) { return static_cast<uint64_t>(value) << 32 | ~static_cast<uint32_t>(token); }

constexpr int kAhead = 3;                          // times eight bins whose logits are asked for together
struct PickRoom {
    uint64_t list[kList + 4];
    uint16_t bins[kBinList];
    ushort8 pieces[kAhead][64];
};

// The best n of a wavefront's `count` candidates in order, in place; how many there are.  (A candidate's place is how many are better: no
// two are alike.)
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
    if (lane < 4) list[count + lane] = 0;
    __builtin_amdgcn_wave_barrier();
    #pragma unroll 1
    for (int z = 0; z < count; z += 4) {
        uint64_t other[4];
        #pragma unroll
        for (int w = 0; w < 4; ++w) other[w] = list[z + w];
        #pragma unroll
        for (int w = 0; w < 4; ++w)
            #pragma unroll
            for (int u = 0; u < kEach; ++u) rank[u] += other[w] > mine[u];
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
    const float2 first = lane < tiles ? sums[lane] : float2{-__builtin_huge_valf(), 0.0f};
    float top = first.x;
    #pragma unroll 1
    for (int t = 64 + lane; t < tiles; t += 64) top = fmaxf(top, sums[t].x);
    top = wave_max(top);
    double sum = 0.0;
    #pragma unroll 1
    for (int t = lane; t < tiles; t += 64) {
        const float2 s = t < 64 ? first : sums[t];
        sum += static_cast<double>(s.y) * static_cast<double>(__builtin_amdgcn_exp2f(fmaf(s.x - top, kLog2e, correction(s.x))));
    }
    sum = sum_of_wave(sum);
    return static_cast<double>(score) - (static_cast<double>(top) + log(sum));
}

// ascending() of eight.  (-0 + 0 is 0.)
__device__ __forceinline__ ushort8 ascending8(ushort8 x) {
    constexpr int16_t k = -0x8000;
    const short8 s = __builtin_bit_cast(short8, __builtin_bit_cast(half8, x) + half8{}), top = {k, k, k, k, k, k, k, k};
    return __builtin_bit_cast(ushort8, s ^ (s >> 15 | top));
}

// 1 in the elements greater than `below`'s two halves, as bits: element 2 w + h at bit w + 16 h.  (asm: the compiler makes a comparison, a
// selection and half a permute of each element out of these two instructions for two.)
__device__ __forceinline__ uint32_t reach(ushort8 x, uint32_t below) {
    const auto u = __builtin_bit_cast(u32x4, x);
    uint32_t w[4];
    #pragma unroll
    for (int e = 0; e < 4; ++e)
        asm("v_pk_sub_u16 %0, %1, %2 clamp\n\tv_pk_min_u16 %0, %0, %3" : "=&v"(w[e]) : "v"(u[e]), "v"(below), "v"(0x00010001u));
    return (w[0] | w[1] << 1) | (w[2] | w[3] << 1) << 2;
}

// The best n of a row's logits, in order, where so many reach `least` that the fast way has no room for them: bin after bin, each an answer of
// memory, the best kept whenever the list is full; bins that cannot hold a better one are passed over.  So it is where many values tie, and where
// few lanes have bins: a lane holds eight neighbouring ones, so a tile has them in eight lanes, and `least` is below all logits for more outputs
// than that (up to 24; beyond, than four times as many).  4 beams of 4096 tokens: 8 outputs 9.4 us, 9 36.8, 25 10.7, 64 52; 10 beams, 20 outputs: 1000 tokens 57,
// 8000 84, 12000 17.
__device__ __forceinline__ int pick_crowded(const uint16_t* row, int vocab, int all, const uint16_t* bins, int n, uint32_t least, PickRoom& room) {
    const int lane = threadIdx.x & 63;
    uint64_t above = static_cast<uint64_t>(least) << 32;
    int count = 0;
    #pragma unroll 1
    for (int f0 = 0; f0 < all; f0 += kBins) {
        const uint64_t best = candidate(bins[f0 + lane], token_of(f0 / kBins, lane, 0));
        #pragma unroll 1
        for (uint64_t some = __ballot(best > above); some; ) {
            const int token = token_of(f0 / kBins, __builtin_ctzll(some), lane);
            if (count > kList - 64) {
                count = best_of(room.list, count, n);
                if (count == n) above = room.list[n - 1];
            }
            const uint64_t c = token < vocab ? candidate(ascending(row[token]), token) : 0, in = __ballot(c > above);
            if (c > above) room.list[count + __popcll(in & ((1ull << lane) - 1))] = c;
            count += __popcll(in);
            __builtin_amdgcn_wave_barrier();
            some &= some - 1;
            some &= __ballot(best > above);
        }
    }
    return best_of(room.list, count, n);
}

// The best of a row's logits to room.list, at least n if the row has them; how many there are.  (A wavefront goes through this once, an
// instruction every eight cycles, beside two answers of memory: the bins, and the logits of those that matter.)
__device__ __forceinline__ int pick(const uint16_t* row, int vocab, int tiles, const uint16_t* bins, int n, PickRoom& room) {
    const int lane = threadIdx.x & 63, all = tiles * kBins;
    constexpr int kHeld = 8, kAtOnce = kHeld * 512;              // bins in a wavefront's registers (262144 tokens)
    ushort8 held[kHeld];
    auto load = [&](int from) {
        #pragma unroll
        for (int v = 0; v < kHeld; ++v) {
            held[v] = ushort8{};
            if (from + v * 512 < all) {
                const int f = from + v * 512 + 8 * lane;
                if (f < all) held[v] = *reinterpret_cast<const ushort8*>(bins + f);
            }
        }
    };
    // n of the lanes' maxima, over all of their bins or (many wanted) over a quarter of them each, reach `least`, so the best n candidates do (no n lanes
    // with bins: all do)
    ushort8 top = {};
    #pragma unroll 1
    for (int from = (all - 1) / kAtOnce * kAtOnce; from >= 0; from -= kAtOnce) {
        load(from);
        #pragma unroll
        for (int v = 0; v < kHeld; ++v) top = __builtin_elementwise_max(top, held[v]);
    }
    uint32_t quarter[4], least = 0;
    #pragma unroll
    for (int e = 0; e < 4; ++e) quarter[e] = top[e] > top[e + 4] ? top[e] : top[e + 4];
    if (n <= 24) {
        const uint32_t a = quarter[0] > quarter[1] ? quarter[0] : quarter[1], b = quarter[2] > quarter[3] ? quarter[2] : quarter[3];
        const uint32_t most = a > b ? a : b;
        #pragma unroll 1
        for (uint32_t bit = 0x4000; bit > 0; bit /= 4) {         // two bits at a time
            const int one = __popcll(__ballot(most >= least + bit)), two = __popcll(__ballot(most >= least + 2 * bit)),
                      three = __popcll(__ballot(most >= least + 3 * bit));
            least += bit * ((one >= n) + (two >= n) + (three >= n));
        }
    } else {
        #pragma unroll 1
        for (int bit = 0x8000; bit > 0; bit /= 2) {
            int enough = 0;
            #pragma unroll
            for (int e = 0; e < 4; ++e) enough += __popcll(__ballot(quarter[e] >= (least | bit)));
            if (enough >= n) least |= bit;
        }
    }
    if (least < kLeast) least = kLeast;
    const uint32_t below = (least - 1) * 0x00010001u;
    int count = 0;
    #pragma unroll 1
    for (int from = 0; from < all; from += kAtOnce) {
        if (from > 0) load(from);
        // the lanes' bins that reach it, as bits, then as a list
        uint32_t half[2] = {0, 0};
        #pragma unroll
        for (int v = 0; v < kHeld; ++v) half[v / 4] |= reach(held[v], below) << (4 * (v % 4));
        uint64_t bits = static_cast<uint64_t>(half[1]) << 32 | half[0];
        const int mine = __popcll(bits), upto = scan(mine), listed = __builtin_amdgcn_readlane(upto, 63);
        if (__builtin_expect(listed > kBinList, 0)) return pick_crowded(row, vocab, all, bins, n, least, room);
        #pragma unroll 1
        for (int at = upto - mine; bits; ++at, bits &= bits - 1) {
            const int bit = __builtin_ctzll(bits);
            room.bins[at] = static_cast<uint16_t>(from + (bit / 32 * 4 + bit % 16 / 4) * 512 + 8 * lane + bit % 4 * 2 + bit / 16 % 2);
        }
        __builtin_amdgcn_wave_barrier();
        // eight lanes to a bin, a piece of eight logits each
        #pragma unroll 1
        for (int z0 = 0; z0 < listed; z0 += 8 * kAhead) {
            ushort8 x[kAhead];
            int token[kAhead];
            #pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                const int z = z0 + 8 * u + lane / 8, f = room.bins[z < listed ? z : listed - 1];
                token[u] = token_of(f / kBins, f % kBins, lane % 8 * 8);
                if (z >= listed) token[u] = vocab;
                constexpr uint16_t none = 0xfc00;
                x[u] = ushort8{none, none, none, none, none, none, none, none};
                if (token[u] + 8 <= vocab) __builtin_memcpy(&x[u], row + token[u], 16);
            }
            if (__builtin_expect(__any((token[0] + 8 > vocab && token[0] < vocab) || (token[1] + 8 > vocab && token[1] < vocab) ||
                                       (token[2] + 8 > vocab && token[2] < vocab)), 0)) {       // a piece with the row's end in it
                #pragma unroll
                for (int u = 0; u < kAhead; ++u)
                    #pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (token[u] + 8 > vocab && token[u] + e < vocab) x[u][e] = row[token[u] + e];
            }
            uint32_t in = 0;                       // bit 8 u + 4 h + w: element 2 w + h of piece u
            #pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                x[u] = ascending8(x[u]);
                room.pieces[u][lane] = x[u];
                const uint32_t r = reach(x[u], below);
                in |= ((r | r >> 12) & 0xffu) << (8 * u);
            }
            const int own = __popc(in), behind = scan(own), new_ones = __builtin_amdgcn_readlane(behind, 63);
            if (__builtin_expect(count + new_ones > kList, 0)) return pick_crowded(row, vocab, all, bins, n, least, room);
            #pragma unroll 1
            for (int at = count + behind - own; in; ++at, in &= in - 1) {
                const int bit = __builtin_ctz(in), u = bit / 8, e = bit % 4 * 2 + bit / 4 % 2;
                static_assert(kAhead == 3, "one of three");
                const int t = (u == 0 ? token[0] : u == 1 ? token[1] : token[2]) + e;
                room.list[at] = candidate(reinterpret_cast<const uint16_t*>(&room.pieces[u][lane])[e], t);
            }
            count += new_ones;
            __builtin_amdgcn_wave_barrier();
        }
    }
    return count;
}

// ---- what a group chooses -------------------------------------------------------------------------------------
//
// A block has a group: kPickWaves wavefronts that pick, row by row, and as many that take the rows' sums meanwhile.

constexpr int kGroupWaves = 2 * kPickWaves, kGroupThreads = 64 * kGroupWaves;
constexpr int kOffer = 64;                         // offers of a row at most
constexpr int kIdBits = 21;                        // of the token
constexpr int kSame = 8;
struct Offer {
    double value;
    uint32_t id, pad;                              // row of the group and token
};
__device__ __forceinline__ bool better(const Offer& a, const Offer& b) { return a.value > b.value || (a.value == b.value && a.id < b.id); }
// fp32 of a value, as a number that ascends with it: equal values have equal keys, a greater one's is not smaller.
__device__ __forceinline__ uint32_t key_of(double value) {
    const uint32_t u = __float_as_uint(static_cast<float>(value));
    return u ^ (static_cast<uint32_t>(static_cast<int>(u) >> 31) | 0x80000000u);
}
struct __attribute__((aligned(16))) Choice {       // in LDS, the rows' offers behind it
    uint32_t keys[kGroupThreads + 4];              // of all offers, one row's behind the other's
    uint16_t slots[kGroupThreads];
    int places[kGroupThreads], hits[kMostOut];
    uint16_t same[kMostOut][kSame];                // offers that share a place
    double offsets[kMostBeams];
    int counts[kMostBeams];
    Offer offers[1];
};
constexpr size_t choice_bytes(int beams) { return sizeof(Choice) + (static_cast<size_t>(beams) * kOffer - 1) * sizeof(Offer); }

// Row r of a group: its offers, by one wavefront.
__device__ __forceinline__ void pick_row(const BeamArgs& a, int64_t group, int r, const uint16_t* bins, PickRoom& room, Choice& to) {
    const int lane = threadIdx.x & 63;
    int n = pick(a.logits + (group * a.beams + r) * a.ld, a.vocab, a.tiles, bins, a.n_out, room);
    if (n > kOffer || a.beams > kGroupWaves) n = best_of(room.list, n, a.n_out);      // (many beams: see merge_many)
    if (lane < n) {
        const uint64_t c = room.list[lane];
        to.offers[r * kOffer + lane] = Offer{static_cast<double>(h_f(static_cast<uint16_t>(half_bits(static_cast<uint32_t>(c >> 32))))),
                                             static_cast<uint32_t>(r) << kIdBits | ~static_cast<uint32_t>(c), 0};
    }
    if (lane == 0) to.counts[r] = n;
}

__device__ __forceinline__ void put(const BeamArgs& a, int64_t group, int place, const Offer& o) {
    const int64_t to = group * a.n_out + place;
    a.out_score[to] = static_cast<float>(o.value);
    a.out_token[to] = static_cast<int>(o.id & ((1u << kIdBits) - 1));
    a.out_row[to] = static_cast<int>(group * a.beams) + static_cast<int>(o.id >> kIdBits);
}

// Of more beams than wavefronts, whose offers are in order each: an offer's place is its place in its own list and, of each other list, how
// many there are before it, by halves.  Returns the number of offers.
__device__ __forceinline__ int merge_many(const BeamArgs& a, int64_t group, Choice& c) {
    int all = 0;
    #pragma unroll 1
    for (int r = 0; r < a.beams; ++r) {
        if (!(fabs(c.offsets[r]) < __builtin_huge_val())) c.counts[r] = 0;        // (every thread the same)
        all += c.counts[r];
    }
    __syncthreads();
    #pragma unroll 1
    for (int z = threadIdx.x; z < a.beams * kOffer; z += kGroupThreads)
        if (z % kOffer < c.counts[z / kOffer]) c.offers[z].value += c.offsets[z / kOffer];
    __syncthreads();
    #pragma unroll 1
    for (int z = threadIdx.x; z < a.beams * kOffer; z += kGroupThreads) {
        const int r = z / kOffer, i = z % kOffer;
        if (i >= c.counts[r]) continue;
        const Offer own = c.offers[z];
        int place = i;
        #pragma unroll 1
        for (int o = 0; o < a.beams && place < a.n_out; ++o) {
            if (o == r) continue;
            int lo = 0, hi = c.counts[o];
            while (lo < hi) {
                const int mid = (lo + hi) / 2;
                const bool before = better(c.offers[o * kOffer + mid], own);
                lo = before ? mid + 1 : lo;
                hi = before ? hi : mid;
            }
            place += lo;
        }
        if (place < a.n_out) put(a, group, place, own);
    }
    return all;
}

// An offer's place among all: how many have a greater key, counted by all wavefronts, a part of the keys each.  Those that then share a
// place have equal keys and are told apart by their 64 bits and ids.
__device__ __forceinline__ int merge_few(const BeamArgs& a, int64_t group, Choice& c) {
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    // a wavefront's row, and where its offers come among all
    const bool good = lane < a.beams && fabs(c.offsets[lane < a.beams ? lane : 0]) < __builtin_huge_val();
    const int counts = good ? c.counts[lane] : 0, upto = scan(counts);
    const int all = __builtin_amdgcn_readlane(upto, 63), own = __builtin_amdgcn_readlane(counts, wave);
    const int base = __builtin_amdgcn_readlane(upto, wave) - own;
    if (lane < own) {
        Offer& o = c.offers[wave * kOffer + lane];
        o.value += c.offsets[wave];
        c.keys[base + lane] = key_of(o.value);
        c.slots[base + lane] = static_cast<uint16_t>(wave * kOffer + lane);
    }
    c.places[tid] = 0;
    if (tid < kMostOut) c.hits[tid] = 0;
    if (tid < 4) c.keys[all + tid] = 0;
    __syncthreads();
    const int chunks = (all + 63) / 64, shift = chunks > 1 ? 32 - __builtin_clz(chunks - 1) : 0;       // 2^shift times 64 offers are room for all
    const int parts = kGroupWaves >> shift, part = wave >> shift, mine = (wave - (part << shift)) * 64 + lane;
    if (mine < all) {
        const uint32_t key = c.keys[mine];
        int place = 0;
        #pragma unroll 4
        for (int z = 4 * part; z < all; z += 4 * parts) {
            const u32x4 other = *reinterpret_cast<const u32x4*>(&c.keys[z]);
            #pragma unroll
            for (int e = 0; e < 4; ++e) place += other[e] > key;
        }
        if (place) atomicAdd(&c.places[mine], place);
    }
    __syncthreads();
    int place = tid < all ? c.places[tid] : a.n_out;
    if (place < a.n_out) {
        const int nth = atomicAdd(&c.hits[place], 1);
        if (nth < kSame) c.same[place][nth] = static_cast<uint16_t>(tid);
    }
    __syncthreads();
    if (place < a.n_out) {
        const Offer o = c.offers[c.slots[tid]];
        const int hits = c.hits[place], shared = place;
        if (hits > 1 && hits <= kSame) {           // (two tokens of a row have the same logit, most often)
            #pragma unroll 1
            for (int z = 0; z < hits; ++z) place += better(c.offers[c.slots[c.same[shared][z]]], o);
        } else if (hits > 1) {
            const uint32_t key = c.keys[tid];
            #pragma unroll 1
            for (int z0 = 0; z0 < all; z0 += 4) {
                uint32_t same = 0;
                #pragma unroll
                for (int e = 0; e < 4; ++e) same |= static_cast<uint32_t>(c.keys[z0 + e] == key) << e;
                for (; same; same &= same - 1) {
                    const int z = z0 + __builtin_ctz(same);
                    if (z < all) place += better(c.offers[c.slots[z]], o);
                }
            }
        }
        if (place < a.n_out) put(a, group, place, o);
    }
    return all;
}

// The best n_out of all offers, by the block, behind a barrier.
__device__ __forceinline__ void merge(const BeamArgs& a, int64_t group, Choice& c) {
    const int all = a.beams > kGroupWaves ? merge_many(a, group, c) : merge_few(a, group, c);
    const int place = threadIdx.x;
    if (place >= all && place < a.n_out) {
        const int64_t to = group * a.n_out + place;
        a.out_score[to] = -__builtin_huge_valf();
        a.out_token[to] = a.out_row[to] = -1;
    }
}

__global__ __launch_bounds__(kGroupThreads) void beam_pick_kernel(const BeamArgs a, const float2* __restrict__ sums, const uint16_t* __restrict__ bins) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    __shared__ PickRoom rooms[kPickWaves];
    Choice& choice = *reinterpret_cast<Choice*>(lds);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t group = static_cast<int64_t>(a.first) + blockIdx.x;
    #pragma unroll 1
    for (int r = wave % kPickWaves; r < a.beams; r += kPickWaves) {
        const int64_t item = (static_cast<int64_t>(blockIdx.x) * a.beams + r) * a.tiles;
        if (wave < kPickWaves) pick_row(a, group, r, bins + item * kBins, rooms[wave], choice);
        else choice.offsets[r] = offset_of(sums + item, a.tiles, a.score[group * a.beams + r]);
    }
    __syncthreads();
    merge(a, group, choice);
}

// Everything in one block per group, for streams that have no workspace: row by row, sums and bins in LDS.
__global__ __launch_bounds__(kGroupThreads) void beam_alone_kernel(const BeamArgs a) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    __shared__ PickRoom room;
    auto* const sums = reinterpret_cast<float2*>(lds);
    auto* const bins = reinterpret_cast<uint16_t*>(sums + (a.tiles + 1) / 2 * 2);
    Choice& choice = *reinterpret_cast<Choice*>(bins + a.tiles * kBins);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int64_t group = blockIdx.x;
    for (int r = 0; r < a.beams; ++r) {
        const uint16_t* const row = a.logits + (group * a.beams + r) * a.ld;
        for (int t = wave; t < a.tiles; t += kGroupWaves) {
            const Scanned s = scan_tile(row, a.vocab, t);
            bins[t * kBins + lane] = static_cast<uint16_t>(s.bin);
            if (lane == 0) sums[t] = float2{s.top, s.sum};
        }
        __syncthreads();
        if (wave == 0) pick_row(a, group, r, bins, room, choice);
        else if (wave == 1) choice.offsets[r] = offset_of(sums, a.tiles, a.score[group * a.beams + r]);
        __syncthreads();
    }
    merge(a, group, choice);
}
constexpr size_t alone_bytes(int tiles) { return static_cast<size_t>((tiles + 1) / 2 * 2) * 8 + static_cast<size_t>(tiles) * kBins * 2; }
static_assert(alone_bytes(tiles_of_row(MI_BEAM_MAX_VOCAB)) + choice_bytes(kMostBeams) + sizeof(PickRoom) <= 160 * 1024, "fits LDS");
static_assert(choice_bytes(kMostBeams) + kPickWaves * sizeof(PickRoom) <= 160 * 1024, "fits LDS");
static_assert(groups_that_fit(kWorkspaceBytes, kMostBeams, MI_BEAM_MAX_VOCAB) >= 1, "a group fits the workspace");
static_assert(tiles_of_row(MI_BEAM_MAX_VOCAB) * kBins <= 65536, "a bin's number has 16 bits");
static_assert(kMostOut <= kOffer && kOffer == 64 && kMostOut + 64 <= kList && kMostBeams <= 64, "a lane each");
static_assert(MI_BEAM_MAX_VOCAB <= 1 << kIdBits && kMostBeams <= 1 << (32 - kIdBits), "an offer's number has 32 bits");

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
    if (static_cast<int64_t>(c.n_groups) * c.beams > 0x7fffffff || c.n_groups > 0x7fffffff / kGroupThreads) {
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
    const size_t choice = choice_bytes(c.beams);
    void* const workspace = stream_room(s).workspace;
    if (!workspace) {
        if (!MI_ONCE_OK(raise_lds(reinterpret_cast<const void*>(beam_alone_kernel),
                                  static_cast<int>(alone_bytes(tiles_of_row(MI_BEAM_MAX_VOCAB)) + choice_bytes(kMostBeams)))))
            return 0;
        hipLaunchKernelGGL(beam_alone_kernel, dim3(c.n_groups), dim3(kGroupThreads), alone_bytes(a.tiles) + choice, s, a);
        return MI_HIP_OK(hipGetLastError()) ? 1 : 0;
    }
    if (!MI_ONCE_OK(raise_lds(reinterpret_cast<const void*>(beam_pick_kernel), static_cast<int>(choice_bytes(kMostBeams))))) return 0;
    const int64_t fit = groups_that_fit(kWorkspaceBytes, c.beams, c.vocab);
    for (int64_t first = 0; first < c.n_groups; first += fit) {
        const int64_t n = c.n_groups - first < fit ? c.n_groups - first : fit, items = n * c.beams * a.tiles;
        a.first = static_cast<int>(first);
        a.rows = static_cast<int>(n * c.beams);
        auto* const bins = static_cast<uint16_t*>(workspace);
        auto* const sums = reinterpret_cast<float2*>(bins + items * kBins);
        hipLaunchKernelGGL(beam_scan_kernel, dim3(static_cast<unsigned>((items + kScanWaves - 1) / kScanWaves)), dim3(64 * kScanWaves), 0, s, a, sums,
                           bins);
        if (!MI_HIP_OK(hipGetLastError())) return 0;
        hipLaunchKernelGGL(beam_pick_kernel, dim3(static_cast<unsigned>(n)), dim3(kGroupThreads), choice, s, a, sums, bins);
        if (!MI_HIP_OK(hipGetLastError())) return 0;
    }
    return 1;
}
