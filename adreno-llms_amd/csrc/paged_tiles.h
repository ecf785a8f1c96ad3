// What the kernels of attention over a cache in pages (paged_attention.hip, paged_tree.hip) share: out = sum_j w_j v_j / sum_j w_j over the
// positions j that a row sees, w_j = exp(scale q k_j - their maximum), per query head; who does what, and a tile of keys and values
// from its pages to the matrix instructions' operands.
#pragma once
#include "device_math.h"
#include "paged.h"
#include "paged_plan.h"

#include <type_traits>

namespace mi {
namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef float floatx2 __attribute__((ext_vector_type(2)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef short short4v __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

constexpr float kNone = -__builtin_huge_valf();  // the score of a key that the query does not see
constexpr float kStart = -1.0e30f;               // the running maximum of a query that has seen no key
// Weights are exp2(score - base).  base is set to kHead below the greatest score so far and stays until a score is more than kHead + kSlack
// above it: so the greatest weight is between 2^7 and 2^15, fp16 holds weights down to 2^-21 of it at full precision, and the sums
// are rescaled only where the maximum has risen by more than kSlack.
constexpr float kHead = 7.0f, kSlack = 8.0f;
// Up to there (2^23, where fp32 counts in halves) a score times scale goes into its weight's exponent unrounded, by fma.  Beyond, what an
// unrounded product is apart from a rounded base may be more than fp16's whole range, so each product is rounded first: equal
// scores then have equal weights, of at most 2^kMost (a product just over base + kSlack + kHead may round to it; fp16 ends below 2^16).
constexpr float kFar = 8388608.0f, kMost = 15.9375f;
__device__ __forceinline__ float far_exponent(float score, float scale_log2, float base) {
    const float x = fabsf(base) < kFar ? fmaf(score, scale_log2, -base) : score * scale_log2 - base;
    return x > kMost ? kMost : x;                    // (a NaN stays one)
}
// The base for a greatest score `most`, from the product as far_exponent has it.
__device__ __forceinline__ float base_of(float most, float scale_log2) {
    const float rounded = most * scale_log2 - kHead;
    return fabsf(rounded) < kFar ? fmaf(most, scale_log2, -kHead) : rounded;
}

// The greater of a lane's value and those of the lanes 16, 32 and 48 away.
__device__ __forceinline__ float max_of_groups(float a) {
    unsigned u = __float_as_uint(a);
    auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    u = __float_as_uint(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
    r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
// The greatest of three, NaN where one is (one instruction; fmaxf would quieten signalling NaNs first, with another for each operand).
__device__ __forceinline__ float max3(float a, float b, float c) { return __builtin_elementwise_maximum(__builtin_elementwise_maximum(a, b), c); }
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(floatx2{a, b}, half2v));
}
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

// Sum of the lanes up to a lane's own.
__device__ __forceinline__ int scan(int x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);      // from 1, 2, 4, 8 lanes below, in rows of 16
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);      // row 0's last lane to row 1, 2's to 3
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);      // lane 31 to rows 2 and 3
    return x;
}
template <int CTRL, int ROWS>
__device__ __forceinline__ float add_dpp(float x) {
    return x + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, ROWS, 0xf, false));
}
// Sum of all lanes, in the last lane.
__device__ __forceinline__ float sum_to_last(float x) {
    x = add_dpp<0x111, 0xf>(x);
    x = add_dpp<0x112, 0xf>(x);
    x = add_dpp<0x114, 0xf>(x);
    x = add_dpp<0x118, 0xf>(x);
    x = add_dpp<0x142, 0xa>(x);
    return add_dpp<0x143, 0xc>(x);
}

// A masked key has weight 0, but 0 x inf and 0 x NaN are NaN.  So in a tile that is masked for some query the values are
// multiplied in four parts, if there are any that are not finite: the finite ones (the others as 0), and 1 for every infinity, every
// -infinity and every NaN: the sum of a query's weights for those, where it is not 0, says that the query sees one, which is
// then added to its output.
__device__ __forceinline__ uint32_t odd_halves(uint32_t x) { return ((x & 0x7c007c00u) + 0x04000400u) & 0x80008000u; }     // top bits of odd ones
__device__ __forceinline__ uint32_t whole_halves(uint32_t top) { return (top >> 15) * 0xffffu; }                         // top bits -> halves
__device__ __forceinline__ uint32_t odd_part(uint32_t x, int part) {
    const uint32_t odd = whole_halves(odd_halves(x)), nan = odd & whole_halves(((x & 0x03ff03ffu) + 0x7fff7fffu) & 0x80008000u);
    const uint32_t sign = whole_halves(x & 0x80008000u), inf = odd & ~nan;
    return part == 0 ? x & ~odd : (part == 1 ? inf & ~sign : part == 2 ? inf & sign : nan) & 0x3c003c00u;
}
__device__ __forceinline__ float with_odd(float sum, float found, int part) {
    if (part == 0) return sum + found;
    const float what = part == 1 ? __builtin_huge_valf() : part == 2 ? -__builtin_huge_valf() : __builtin_nanf("");
    return found != 0.0f ? sum + what : sum;
}

// A stored element as the number it stands for.
template <int KIND, int D>
__device__ __forceinline__ float element(const uint8_t* pool, const uint16_t* scales, int64_t row, int e) {
    if constexpr (KIND == MI_KV_F16) return h_f(reinterpret_cast<const uint16_t*>(pool)[row * D + e]);
    if constexpr (KIND == MI_KV_INT8)
        return static_cast<float>(static_cast<_Float16>(static_cast<float>(static_cast<int8_t>(pool[row * D + e])) * h_f(scales[row])));
    const int b = pool[(row * D + e) / 2], code = (e & 1 ? b >> 4 : b & 15) - 8;
    return static_cast<float>(static_cast<_Float16>(static_cast<float>(code) * h_f(scales[row * (D / 32) + e / 32])));
}

// ---- what a row sees ----------------------------------------------------------------------------------
//
// In a plain batch (AttentionArgs) token i of a sequence is at position pos + i and sees what lies before it.  In a tree of drafts (TreeArgs)
// the earlier positions are seen by the row's own place in its text, which the caller says, and the drafts by a bit for each: every tile
// that holds a draft is one where rows see different keys, the others are as they are in a plain batch.

template <class Args>
constexpr bool is_tree = std::is_same_v<Args, TreeArgs>;

// Of token `token` of a sequence.
__device__ __forceinline__ int position_of(const AttentionArgs&, const Span& s, int token) { return s.pos + token; }
__device__ __forceinline__ int position_of(const TreeArgs& a, const Span& s, int token) {
    const int p = a.window > 0 ? a.position[s.first + token] : s.pos;       // (without a window all earlier positions are seen)
    return p < s.pos ? s.pos : p > s.pos + (s.n - 1) ? s.pos + (s.n - 1) : p;
}
// The drafts at positions j0 .. j0 + 31 that it sees, as bits.  (0 before the first and behind the row's words.)
__device__ __forceinline__ uint32_t drafts_seen(const TreeArgs& a, const Span& s, int token, int j0) {
    const int first = j0 - s.pos, word = first >> 5, shift = first & 31;
    const uint32_t* const line = a.seen + static_cast<int64_t>(s.first + token) * a.words;
    const uint32_t lo = word >= 0 && word < a.words ? line[word] : 0u;
    const uint32_t hi = word >= -1 && word + 1 < a.words ? line[word + 1] : 0u;
    return static_cast<uint32_t>((static_cast<uint64_t>(hi) << 32 | lo) >> shift);
}

// ---- who does what --------------------------------------------------------------------------------------
//
// The lengths are known to the device alone.  A block works on some tiles of keys for a set of ROWS rows of one sequence and
// key/value head; how many tiles that are follows from the tiles of the whole batch, so that every block gets about as
// many whatever the mixture of lengths: `share` tiles, such that the items fit the `target` blocks that the chip holds plus
// one per set.  Every wavefront works that out for itself from q_start and kv_len: the loads are those that it
// needs anyway.

struct Item {
    int b = -1, set = 0, chunk = 0, share = 0, tiles = 0;
    Span s;
    int kvh = 0, id = 0;      // its key/value head, and its number over all of them: the parts of a set are n_kv_heads apart
};

// Item `y` of the batch (of any one key/value head); b = -1: there is none.  A q_start that goes down somewhere has more rows than the
// host counted blocks for, and a set whose parts are not all there would leave its counter up for the calls to come: then no block has
// anything (where keys are split every block looks at all of the batch; where they are not there are no counters).
//
// EVEN: where a block's share is long, the least share is looked for with which the items still fit the launch's blocks: the first one leaves
// a part of a share in the last part of each set, up to half of all (at 16 tiles and more: it takes about a microsecond).
// NEAR: which of a sequence's items a block has is as eight_apart says, and a part is what tree_worth says at least.  RESIDENT: shares are round_share's, for
// that many blocks to a compute unit (where they are more than 16 tiles, with one to a unit 16, and not all that a sequence has: the search takes a microsecond).
template <int ROWS, int KEYS, bool EVEN = false, bool NEAR = false, int RESIDENT = 0>
__device__ __forceinline__ Item item_of(const AttentionArgs& a, const Plan& plan, const int y) {
    const int lane = threadIdx.x & 63;
    bool down = false;
    auto span = [&](int b) {
        if (b >= a.p.n_seqs) return Span{};
        const int start = a.p.q_start[b], end = a.p.q_start[b + 1];
        down |= goes_down(start, end);
        return span_of(start, end, a.p.kv_len[b], a.p.n_tokens);
    };
    Item it;
    auto cost = [&](const Span& s) { return cost_of(plan, s, a.p.cap, a.window, a.sinks, ROWS, KEYS); };
    Span s = span(lane);
    Cost c = cost(s);
    it.share = 0x7fffffff;
    if (plan.target > 0) {
        float total = static_cast<float>(c.sets) * static_cast<float>(c.tiles);
        for (int b0 = 64; b0 < a.p.n_seqs; b0 += 64) {
            const Cost more = cost(span(b0 + lane));
            total += static_cast<float>(more.sets) * static_cast<float>(more.tiles);
        }
        it.share = uniform(share_of(__int_as_float(__builtin_amdgcn_readlane(__float_as_int(sum_to_last(total)), 63)), plan));
        if (EVEN && plan.target > 0 && a.p.n_seqs <= 64 && it.share >= 16) {
            it.share = uniform(even_share(it.share, static_cast<int>(gridDim.x) / a.p.n_kv_heads, [&](int share) {
                const float items = static_cast<float>(items_of(c, share));
                return static_cast<int>(__int_as_float(__builtin_amdgcn_readlane(__float_as_int(sum_to_last(items)), 63)));
            }));
        }
    }
    if (RESIDENT > 0 && plan.target > 0 && it.share + (RESIDENT == 1) > 4 * kWaves && a.p.n_seqs <= 64 && __any(c.tiles > it.share)) {
        const auto sum = [](float x) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(sum_to_last(x)), 63)); };
        const float sets = static_cast<float>(c.sets), tiles = static_cast<float>(c.tiles), worth = static_cast<float>(tree_worth(c.tiles));
        const auto items = [&](int share) {        // (a tile's half: the quotient is no whole number that its rounding could miss)
            return static_cast<int>(sum(sets * (floorf((tiles - 0.5f) * __builtin_amdgcn_rcpf(fmaxf(static_cast<float>(share), worth))) + 1.0f)));
        };
        const float most = wave_max(tiles);
        if (most < 1.0e6f)
            it.share = uniform(round_share(it.share, sum(sets * tiles), static_cast<int>(sum(sets)), static_cast<int>(most), plan, RESIDENT,
                                           static_cast<int>(gridDim.x) / a.p.n_kv_heads, items));
    }
    int before = 0;
    for (int b0 = 0;; ) {
        if (__any(down)) return it;
        int share = it.share;
        if constexpr (NEAR) {
            const int worth = plan.target > 0 ? tree_worth(c.tiles) : 0;
            if (share < worth) share = worth;
        }
        const int chunks = c.sets ? (c.tiles - 1) / share + 1 : 0, upto = scan(c.sets * chunks) + before;
        const uint64_t past = __ballot(upto > y);
        if (past) {
            const int l = uniform(__builtin_ctzll(past));
            it.b = b0 + l;
            it.s.first = __builtin_amdgcn_readlane(s.first, l);
            it.s.n = __builtin_amdgcn_readlane(s.n, l);
            it.s.pos = __builtin_amdgcn_readlane(s.pos, l);
            it.tiles = __builtin_amdgcn_readlane(c.tiles, l);
            const int n = __builtin_amdgcn_readlane(chunks, l), sets = __builtin_amdgcn_readlane(c.sets, l);
            const int own = y - (__builtin_amdgcn_readlane(upto, l) - sets * n);
            if constexpr (NEAR) {
                const unsigned heads = a.p.n_kv_heads;
                it.id = blockIdx.x;
                it.kvh = blockIdx.x - y * heads;
                if (sets > 1) {
                    const SetOfPair x = eight_apart(own * heads + it.kvh, sets, n * heads);
                    it.set = x.set;
                    it.chunk = x.pair / heads;
                    it.kvh = x.pair - it.chunk * heads;
                    it.id = (y - own + x.set * n + it.chunk) * heads + it.kvh;
                    it.share = (it.tiles - 1) / n + 1;
                    return it;
                }
            }
            const int set = sets == 1 ? 0 : own / n;
            it.chunk = own - set * n;
            it.set = sets - 1 - set;                                 // (the longest first)
            if (NEAR || n > 1) it.share = (it.tiles - 1) / n + 1;          // (the sequence's tiles in n equal parts)
            return it;
        }
        before = __builtin_amdgcn_readlane(upto, 63);
        b0 += 64;
        if (b0 >= a.p.n_seqs) return it;
        s = span(b0 + lane);
        c = cost(s);
    }
}

// ---- a tile of 32 keys as it comes from the cache, and as operands ------------------------------------------

// Keys as A operand of q k: of 16 n + i, n = 0, 1, pieces of 16 bytes (8 where a row has 32), the groups' side by side, so that
// a load of 64 lanes covers 64 bytes and more of a row at once (with a quarter of the row per group every lane was in a line of its
// own).  Which elements meet in one product does not matter as long as the query brings the same.  Values as A operand of
// the product with the weights: of keys 4 g .. and 16 + 4 g .., the elements i D / 16 .., D / 16 of them, which become row i of
// D / 16 operands: element m of the piece is row i of operand m.  The transpose is then one byte permute per two numbers.
template <int KIND, int D, bool PAGES16>
struct Tile {
    static constexpr int kK = row_bytes(KIND, D) / 4 / 4;      // words of a key's pieces
    static constexpr int kVBytes = row_bytes(KIND, D) / 16;    // bytes of a value's piece: 2, 4, 8, 16
    static constexpr int kV = (kVBytes + 3) / 4;
    uint32_t k[2][kK];
    std::conditional_t<kVBytes == 2, uint16_t, uint32_t> v[8][kV];
    uint16_t ks[2];                                            // the keys' scales
    // The values' scales, of four keys at a time as they are loaded: Q4 whole rows of them; int8 two to a word, or (keys looked up
    // one by one) one to a word.  pack_scales leaves the lane's, two to a word, in the first two.
    static constexpr int kVS = KIND == MI_KV_Q4 ? D / 16 : PAGES16 ? 2 : 4;
    uint32_t vs[2][kVS];
};

// N words, in pieces of four that are 4 STEP bytes apart.
template <int STEP, int N>
__device__ __forceinline__ void load_words(uint32_t (&w)[N], const uint8_t* p) {
    if constexpr (N % 4 == 0) {
        #pragma unroll
        for (int j = 0; j < N; j += 4) {
            const u32x4 x = *reinterpret_cast<const u32x4*>(p + STEP * j);
            w[j] = x[0]; w[j + 1] = x[1]; w[j + 2] = x[2]; w[j + 3] = x[3];
        }
    } else if constexpr (N == 2) {
        const u32x2 x = *reinterpret_cast<const u32x2*>(p);
        w[0] = x[0]; w[1] = x[1];
    } else {
        w[0] = *reinterpret_cast<const uint32_t*>(p);
    }
}

template <int N>
__device__ __forceinline__ void load_value(uint32_t (&w)[N], const uint8_t* p) { load_words<4>(w, p); }
__device__ __forceinline__ void load_value(uint16_t (&w)[1], const uint8_t* p) { w[0] = *reinterpret_cast<const uint16_t*>(p); }

// Codes as fp16 numbers, two to a word, times their scales: rounded once, to the number that the cache holds.
__device__ __forceinline__ uint32_t scaled(uint32_t codes, half2v scale) {
    return __builtin_bit_cast(uint32_t, __builtin_bit_cast(half2v, codes) * scale);
}
// Signed bytes LO of a and HI of b.  (Sub-word operands: an instruction per number, where building it under an exponent takes three
// for two.)
template <int LO, int HI>
__device__ __forceinline__ uint32_t from_bytes(uint32_t a, uint32_t b) {
    uint32_t r;
#define MI_BYTES(L, H)                                                                                                     \
    if constexpr (LO == L && HI == H)                                                                                      \
        asm("v_cvt_f16_i16_sdwa %0, sext(%1) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_" #L "\n\t"                 \
            "v_cvt_f16_i16_sdwa %0, sext(%2) dst_sel:WORD_1 dst_unused:UNUSED_PRESERVE src0_sel:BYTE_" #H                  \
            : "=&v"(r) : "v"(a), "v"(b))
    MI_BYTES(0, 0);
    MI_BYTES(1, 1);
    MI_BYTES(2, 2);
    MI_BYTES(3, 3);
    MI_BYTES(0, 1);
    MI_BYTES(2, 3);
#undef MI_BYTES
    return r;
}
// The nibbles at bits 0 and 16, less 8: under the exponent of 1024 a nibble is that number above 1024.  (Both constants cannot
// be scalars of one instruction: `exponent` is a vector register that holds 0x64006400.)
__device__ __forceinline__ uint32_t from_nibbles(uint32_t w, uint32_t exponent) {
    uint32_t r;
    asm("v_and_or_b32 %0, %1, %2, %3" : "=v"(r) : "v"(w), "s"(0x000f000fu), "v"(exponent));
    const half2v above = {static_cast<_Float16>(1032.0f), static_cast<_Float16>(1032.0f)};
    return __builtin_bit_cast(uint32_t, __builtin_bit_cast(half2v, r) - above);
}
__device__ __forceinline__ half2v both(uint16_t s) { return __builtin_bit_cast(half2v, s * 0x00010001u); }

// Operand j (8 elements) of a key's piece.  Q4: elements come as 0 4 1 5 2 6 3 7 of each 8, and so does the query.
template <int KIND, int N>
__device__ __forceinline__ half8 key_operand(const uint32_t (&w)[N], int j, uint16_t scale, uint32_t exponent) {
    if constexpr (KIND == MI_KV_F16) return __builtin_bit_cast(half8, u32x4{w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]});
    u32x4 r;
    const half2v s = both(scale);
    if constexpr (KIND == MI_KV_INT8) {
        #pragma unroll
        for (int h = 0; h < 2; ++h) {
            r[2 * h] = scaled(from_bytes<0, 1>(w[2 * j + h], w[2 * j + h]), s);
            r[2 * h + 1] = scaled(from_bytes<2, 3>(w[2 * j + h], w[2 * j + h]), s);
        }
    } else {
        #pragma unroll
        for (int h = 0; h < 4; ++h) r[h] = scaled(from_nibbles(w[j] >> (4 * h), exponent), s);
    }
    return __builtin_bit_cast(half8, r);
}

// (Lane i's elements i D / 16 .. of a Q4 row are in block i D / 16 / 32 of it.)
template <int KIND, int D, bool PAGES16>
__device__ __forceinline__ void pack_scales(Tile<KIND, D, PAGES16>& t, int i) {
    if constexpr (KIND == MI_KV_F16 || (KIND == MI_KV_INT8 && PAGES16)) return;
    constexpr int kWords = KIND == MI_KV_Q4 ? D / 64 : 1;          // of a key
    const uint32_t sel = KIND == MI_KV_Q4 && i & (8 / kWords) ? 0x07060302u : 0x05040100u;
    #pragma unroll
    for (int n = 0; n < 2; ++n) {
        uint32_t w[4];
        #pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = kWords == 1 || i < 8 ? t.vs[n][kWords * e] : t.vs[n][kWords * e + kWords - 1];
        t.vs[n][0] = __builtin_amdgcn_perm(w[1], w[0], sel);
        t.vs[n][1] = __builtin_amdgcn_perm(w[3], w[2], sel);
    }
}

// Keys 2 p and 2 p + 1 of the lane's values, element m of their pieces.
template <int KIND, int D, bool PAGES16>
__device__ __forceinline__ uint32_t value_pair(const Tile<KIND, D, PAGES16>& t, int p, int m, uint32_t exponent) {
    const auto &lo = t.v[2 * p], &hi = t.v[2 * p + 1];
    if constexpr (KIND == MI_KV_F16)
        return __builtin_amdgcn_perm(hi[m / 2], lo[m / 2], m & 1 ? 0x07060302u : 0x05040100u);
    const half2v s = __builtin_bit_cast(half2v, t.vs[p / 2][p % 2]);
    if constexpr (KIND == MI_KV_INT8) {
        const uint32_t a = lo[m / 4], b = hi[m / 4];
        return scaled(m % 4 == 0 ? from_bytes<0, 0>(a, b) : m % 4 == 1 ? from_bytes<1, 1>(a, b) : m % 4 == 2 ? from_bytes<2, 2>(a, b)
                                                                                                           : from_bytes<3, 3>(a, b), s);
    } else {
        const uint32_t two = __builtin_amdgcn_perm(static_cast<uint32_t>(hi[0]), static_cast<uint32_t>(lo[0]), m < 4 ? 0x05040100u : 0x07060302u);
        return scaled(from_nibbles(two >> (4 * (m % 4)), exponent), s);
    }
}

// Whether any of the lane's values that are in the cache (`there`, a mask for each pair of keys) may be an infinity or a NaN:
// of fp16 its greatest, else its scales (256 and more count, as their products may overflow).
template <int KIND, int D, bool PAGES16>
__device__ __forceinline__ bool odd_values(const Tile<KIND, D, PAGES16>& t, const uint32_t (&there)[4]) {
    uint16_t most = 0;
    #pragma unroll
    for (int e = 0; e < 8; ++e) {
        const uint16_t have = static_cast<uint16_t>(there[e / 2] >> (16 * (e & 1)));
        if constexpr (KIND == MI_KV_F16) {
            #pragma unroll
            for (int w = 0; w < Tile<KIND, D, PAGES16>::kV; ++w)
                #pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint16_t x = static_cast<uint16_t>(t.v[e][w] >> (16 * h)) & have & 0x7fffu;
                    most = x > most ? x : most;
                }
        } else {
            const uint16_t x = static_cast<uint16_t>(t.vs[e / 4][e / 2 % 2] >> (16 * (e & 1))) & have & 0x7fffu;
            most = x > most ? x : most;
        }
    }
    return most >= (KIND == MI_KV_F16 ? 0x7c00u : 0x5c00u);
}

}  // namespace
}  // namespace mi
