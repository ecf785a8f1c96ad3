// Attention of many sequences' new tokens over a cache in pages (mi_attention): out = sum_j w_j v_j / sum_j w_j over the
// positions j that a row sees, w_j = exp(scale q k_j - their maximum), per query head.
//
// The query heads that share a key/value head are rows of one matrix, token by token (row t * nrep + head), so that a key
// is fetched once for all of them: 16 rows are one operand of v_mfma_f32_16x16x32_f16.  Scores are computed transposed (A = keys,
// B = queries): lane (query i = lane % 16, group g = lane / 16) then holds keys 4 g .. 4 g + 3 of every 16 for its query, and
// two such quadruples are, as they stand, the B operand of the product with the values, whichever keys they are, as long as
// the A operand (values transposed) brings the same.  Probabilities never leave the registers.
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
};

// Item `y` of the batch (of any one key/value head); b = -1: there is none.  A q_start that goes down somewhere has more rows than the
// host counted blocks for, and a set whose parts are not all there would leave its counter up for the calls to come: then no block has
// anything (where keys are split every block looks at all of the batch; where they are not there are no counters).
template <int ROWS, int KEYS>
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
    }
    int before = 0;
    for (int b0 = 0;; ) {
        if (__any(down)) return it;
        const int chunks = c.sets ? (c.tiles - 1) / it.share + 1 : 0, upto = scan(c.sets * chunks) + before;
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
            const int set = sets == 1 ? 0 : own / n;
            it.chunk = own - set * n;
            it.set = sets - 1 - set;                                 // (the longest first)
            if (n > 1) it.share = (it.tiles - 1) / n + 1;          // (the sequence's tiles in n equal parts)
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

// ---- few rows: keys straight from memory to registers -----------------------------------------------------
//
// A block has 16 rows and a share of their tiles of 32 keys, which its four wavefronts take in turn, each with a maximum and sums of its
// own that meet in LDS at the end.  No barrier in the loop, and no LDS: keys and values go from memory to the registers that are the
// matrix instructions' operands, and as soon as a tile's keys are multiplied the next tile's are asked for into the same registers.
// Blocks that share a set leave sums in the workspace; the last to arrive adds them in their order, so the bits are the same again.
//
// What bounds it: memory where the cache is long (16 rows make 32 operations per byte of fp16, 1/8 of what the matrix cores take for
// each that memory gives): 656 MB of fp16 in 135.8 us, 4.84 TB/s, a large copy 4.93.  Where it is short, 7 us that do not depend on
// its length: launch 1.4, planning 0.9 to 1.3, the first page's number 0.6, parts to the workspace 0.8 to 1.1, arrival 0.4, the
// merge 1.6 to 2: 32 conversations of 14 heads over 2, 14 MB of int8, 8.7 us; 27 MB of Q4, 61 conversations, 15.0.  In Q4 codes to numbers
// keep the vector units busy 63 % of the time of a long step (fp16 8 %): 549 MB in 140 us, 3.9 TB/s; 545 MB of int8 4.65 TB/s.
// Planning looks at 64 sequences at a time, each a trip to memory: tokens behind 200 positions of 14 heads over 2, 32 / 64 / 65 / 128 sequences
// 5.5 / 5.6 / 6.1 / 7.0 us, and then with the bytes 256 / 512 / 1024 / 4096 13 / 27 / 65 / 339 (floors 5 / 11 / 21 / 85).
//
// Four wavefronts to a block; with eight those 32 conversations took 15.6 us for 9.9 (then).  A tile's memory in flight per wavefront is what its
// registers hold, so width 64 asks for four blocks to a compute unit and 128 for two.  Width 64 in fp16 with pages that end inside a
// tile asks for three: with four, 44 registers spilled (32 conversations to 4096 in pages of 100 13.8 us for 12.6, 16 to 8000 in pages of 50
// 15.9 for 14.6); in pages of whole sixteens 3 spill, and four are as fast or faster (61 to 2500 22.7, with three 23.6).

// PAGES16: pages are multiples of 16 positions long, so 16 keys lie in one page.
template <int KIND, int D, bool PAGES16>
__global__ __launch_bounds__(64 * kWaves, D == 128 ? 2 : KIND == MI_KV_F16 && !PAGES16 ? 3 : 4) void paged_step_kernel(const AttentionArgs a, const Plan plan, float* __restrict__ sums,
                                                                 uint32_t* __restrict__ counters) {
    constexpr int kOps = D / 32, kOuts = D / 16;   // operands of a key, of the values
    constexpr int kRow = row_bytes(KIND, D), kScales = row_scales(KIND, D);
    constexpr int kPiece = kRow >= 64 ? 16 : 8, kElems = kPiece * D / kRow;       // of a key: bytes, elements
    __shared__ float meet[kWaves][4 * kOuts + 2][64];
    __shared__ uint32_t arrived;
    const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
    const int i = lane & 15, g = lane >> 4;
    const int kvh = blockIdx.x % a.p.n_kv_heads, y = blockIdx.x / a.p.n_kv_heads;
    const Item it = item_of<kRows, kKeys>(a, plan, y);
    if (it.b < 0) return;
    const int rows = it.s.n * plan.nrep, r0 = it.set * kRows, r_end = r0 + kRows < rows ? r0 + kRows : rows;
    const int p_lo = it.s.pos + divide(r0, plan.rep), p_hi = it.s.pos + divide(r_end - 1, plan.rep);
    const Tiles tiles = tiles_of(p_lo, p_hi, a.p.cap, a.window, a.sinks, kKeys);
    const int parts = tiles.count > 0 ? (tiles.count - 1) / it.share + 1 : 1;
    if (it.chunk >= parts) return;
    const int first = parts == 1 ? 0 : it.chunk * it.share;
    const int last = tiles.count - first < it.share ? tiles.count : first + it.share;
    // the lane's query (past the last: that one, not stored)
    const bool live = r0 + i < r_end;
    const int row = live ? r0 + i : r_end - 1, token = divide(row, plan.rep), head = kvh * plan.nrep + (row - token * plan.nrep);
    const int my_pos = it.s.pos + token;
    // (a row before position 0 sees nothing; the window's far end, before the first position where there is none)
    const int before = (a.window > 0 && my_pos >= 0) ? my_pos - a.window : -1, sinks = a.window > 0 ? a.sinks : 0;
    half8 q[kOps];
    {
        const uint16_t* src = a.q + (it.s.first + token) * a.ld_q + head * D + g * kElems;
        const bool wide = reinterpret_cast<uintptr_t>(src) % 16 == 0;
        #pragma unroll
        for (int j = 0; j < kOps; ++j) {
            constexpr int kPer = kElems / 8;           // operands of a piece
            const uint16_t* at = src + j / kPer * (4 * kElems) + 8 * (j % kPer);
            half8 x;
            if (wide) x = *reinterpret_cast<const half8*>(at);
            else
                #pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = __builtin_bit_cast(_Float16, at[e]);
            q[j] = KIND == MI_KV_Q4 ? __builtin_shufflevector(x, x, 0, 4, 1, 5, 2, 6, 3, 7) : x;
        }
    }

    // (as constant memory: scalar loads where the page is one for the wavefront, which do not wait for the tile under way)
    const auto* const table = reinterpret_cast<const __attribute__((address_space(4))) int*>(
        reinterpret_cast<uintptr_t>(a.p.pages + static_cast<int64_t>(it.b) * a.p.max_pages));
    // Page numbers are asked for a tile ahead of what lies in them: two loads in a row would be waited for otherwise.
    struct Pages { int number[2]; };
    auto look_up = [&](int v) {
        Pages p;
        const int j0 = tile_at(tiles, v < last ? v : last - 1) * kKeys;
        #pragma unroll
        for (int n = 0; n < 2; ++n) {
            const int mine = j0 + 16 * n + (PAGES16 ? 0 : i), j = mine < tiles.end ? mine : tiles.end - 1;
            p.number[n] = table[divide(j, a.p.page)];
        }
        return p;
    };
    // A load's address is a base that is the same for the wavefront plus 32 bits of the lane's own.
    const uint32_t k_off = i * kRow + g * kPiece, v_off = 4 * g * kRow + i * (kRow / 16);
    const uint32_t ks_off = (i * kScales + kScales * g / 4) * 2, vs_off = 4 * g * kScales * 2;
    struct Rows {                                  // of a tile: where its two times 16 rows begin, and what is not in the pool:
        int64_t at[2];                             // (PAGES16: of 16 keys; else of the lane's key)
        uint32_t absent;                           // bit e of 8: key e of the lane's values
    };
    auto place = [&](int v, const Pages& pages) {
        Rows r;
        r.absent = 0;
        const int j0 = tile_at(tiles, v) * kKeys;
        #pragma unroll
        for (int n = 0; n < 2; ++n) {
            const int mine = j0 + 16 * n + (PAGES16 ? 0 : i), j = mine < tiles.end ? mine : tiles.end - 1;
            const int number = pages.number[n];
            const bool bad = static_cast<uint32_t>(number) >= static_cast<uint32_t>(a.p.n_pages);
            int slot = j - divide(j, a.p.page) * a.p.page.d;
            // (16 keys behind the end are read as the last 16 before it, and masked)
            if constexpr (PAGES16) slot &= ~15;
            r.at[n] = row_number(a.p, bad ? 0 : number, kvh, slot);
            if constexpr (PAGES16) {
                if (bad) r.absent |= 15u << (4 * n);
            } else {
                #pragma unroll
                for (int e = 0; e < 4; ++e) r.absent |= __shfl(bad ? 1u << (4 * n + e) : 0u, 4 * g + e);
            }
        }
        return r;
    };
    Tile<KIND, D, PAGES16> t;
    uint32_t exponent = 0x64006400u;               // see from_nibbles
    if constexpr (KIND == MI_KV_Q4) asm("" : "+v"(exponent));
    auto load_keys = [&](const Rows& r) {
        #pragma unroll
        for (int n = 0; n < 2; ++n) {
            if constexpr (PAGES16) {
                load_words<16>(t.k[n], a.p.k + r.at[n] * kRow + k_off);
                if constexpr (kScales > 0)
                    t.ks[n] = *reinterpret_cast<const uint16_t*>(reinterpret_cast<const uint8_t*>(a.p.k_scale + r.at[n] * kScales) + ks_off);
            } else {
                load_words<16>(t.k[n], a.p.k + r.at[n] * kRow + g * kPiece);
                if constexpr (kScales > 0) t.ks[n] = a.p.k_scale[r.at[n] * kScales + kScales * g / 4];
            }
        }
    };
    auto load_values = [&](const Rows& r) {
        #pragma unroll
        for (int n = 0; n < 2; ++n) {
            if constexpr (PAGES16 && kScales > 0)
                load_words<4>(t.vs[n], reinterpret_cast<const uint8_t*>(a.p.v_scale + r.at[n] * kScales) + vs_off);
            #pragma unroll
            for (int e = 0; e < 4; ++e) {
                if constexpr (PAGES16) {
                    load_value(t.v[4 * n + e], a.p.v + r.at[n] * kRow + v_off + e * kRow);
                } else {
                    const int lo = static_cast<int>(r.at[n]), hi = static_cast<int>(r.at[n] >> 32);
                    const int64_t from = static_cast<uint32_t>(__shfl(lo, 4 * g + e)) | static_cast<int64_t>(__shfl(hi, 4 * g + e)) << 32;
                    load_value(t.v[4 * n + e], a.p.v + from * kRow + i * (kRow / 16));
                    if constexpr (KIND == MI_KV_INT8) t.vs[n][e] = a.p.v_scale[from];
                    if constexpr (KIND == MI_KV_Q4)
                        #pragma unroll
                        for (int w = 0; w < D / 64; ++w)
                            t.vs[n][e * (D / 64) + w] = reinterpret_cast<const uint32_t*>(a.p.v_scale + from * kScales)[w];
                }
            }
        }
    };

    floatx4 acc[kOuts];
    #pragma unroll
    for (int m = 0; m < kOuts; ++m) acc[m] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
    float base = kStart;                           // see kHead
    floatx4 l = {0.0f, 0.0f, 0.0f, 0.0f};          // sum of the weights as they meet the values, the same in every register
    half8 ones;
    #pragma unroll
    for (int e = 0; e < 8; ++e) ones[e] = static_cast<_Float16>(1.0f);
    const float scale_log2 = a.scale * 1.44269504088896341f;
    bool far = false;                              // some query's base is beyond kFar

    // Tile v, whose rows are `r`; `more`: the keys and values of tile v + kWaves, at `next`, are asked for as soon as the registers of
    // tile v's are free, so that they are on their way meanwhile without registers of their own.
    auto multiply = [&](int v, const Rows& r, auto more, const Rows& next) {
        const int j0 = tile_at(tiles, v) * kKeys;
        floatx4 s[2];
        #pragma unroll
        for (int n = 0; n < 2; ++n) {
            s[n] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
            #pragma unroll
            for (int j = 0; j < kOps; ++j)
                s[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(key_operand<KIND>(t.k[n], j, t.ks[n], exponent), q[j], s[n], 0, 0, 0);
        }
        if constexpr (more.value) load_keys(next);
        bool masked = !all_seen(j0, kKeys, p_lo, p_hi, a.p.cap, a.window, a.sinks);
        masked |= PAGES16 ? r.absent != 0 : __any(r.absent);
        uint32_t there[4] = {};                    // halves of keys that are in the cache at all
        if (__builtin_expect(masked, 0)) {
            asm volatile("");                      // (a branch: most tiles are not)
            #pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int n = e / 4, j = j0 + 16 * n + 4 * g + e % 4;
                const bool have = (j < tiles.end) & ((r.absent >> e & 1) == 0);
                const bool see = have & (j <= my_pos) & ((j > before) | (j < sinks));
                s[n][e % 4] = see ? s[n][e % 4] : kNone;
                there[e / 2] |= have ? 0xffffu << (16 * (e & 1)) : 0u;
            }
        }
        float top = max3(max3(s[0][0], s[0][1], s[0][2]), max3(s[0][3], s[1][0], s[1][1]), max3(s[1][2], s[1][3], s[1][3]));
        if (__builtin_expect(__any(top * scale_log2 - kHead > base + kSlack), 0)) {
            top = fmaxf(base, max_of_groups(base_of(top, scale_log2)));
            const float alpha = __builtin_amdgcn_exp2f(base - top);
            l *= alpha;
            #pragma unroll
            for (int m = 0; m < kOuts; ++m) acc[m] *= alpha;
            base = top;
            far = __any(fabsf(base) >= kFar && base > kStart);
        }
        float by = scale_log2, from = base;
        if (__builtin_expect(far, 0)) {
            asm volatile("");
            #pragma unroll
            for (int e = 0; e < 8; ++e) s[e / 4][e % 4] = far_exponent(s[e / 4][e % 4], scale_log2, base);
            by = 1.0f;
            from = 0.0f;
        }
        float w[8];
        #pragma unroll
        for (int e = 0; e < 8; ++e) w[e] = __builtin_amdgcn_exp2f(fmaf(s[e / 4][e % 4], by, -from));
        pack_scales(t, i);
        const half8 pb = __builtin_bit_cast(half8, u32x4{pack2(w[0], w[1]), pack2(w[2], w[3]), pack2(w[4], w[5]), pack2(w[6], w[7])});
        l = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, pb, l, 0, 0, 0);
        if (!masked) {
            #pragma unroll
            for (int m = 0; m < kOuts; ++m)
                acc[m] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                    __builtin_bit_cast(half8, u32x4{value_pair(t, 0, m, exponent), value_pair(t, 1, m, exponent), value_pair(t, 2, m, exponent), value_pair(t, 3, m, exponent)}),
                    pb, acc[m], 0, 0, 0);
            if constexpr (more.value) load_values(next);
            return;
        }
        // What is not in the cache is taken as 0; for what is and is not finite see odd_part.
        auto product = [&](int m, floatx4 from, auto change) {
            u32x4 x;
            #pragma unroll
            for (int p = 0; p < 4; ++p) x[p] = change(value_pair(t, p, m, exponent) & there[p]);
            return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, x), pb, from, 0, 0, 0);
        };
        if (__builtin_expect(!__any(odd_values(t, there)), 1)) {
            #pragma unroll
            for (int m = 0; m < kOuts; ++m) acc[m] = product(m, acc[m], [](uint32_t x) { return x; });
        } else {
            #pragma unroll
            for (int m = 0; m < kOuts; ++m)
                #pragma unroll 1
                for (int part = 0; part < 4; ++part) {
                    const floatx4 none = {0.0f, 0.0f, 0.0f, 0.0f};
                    const floatx4 found = product(m, none, [&](uint32_t x) { return odd_part(x, part); });
                    #pragma unroll
                    for (int r = 0; r < 4; ++r) acc[m][r] = with_odd(acc[m][r], found[r], part);
                }
        }
        if constexpr (more.value) load_values(next);
    };

    if (first + wave < last) {
        int v = first + wave;
        Pages pages = look_up(v);
        Rows now = place(v, pages);
        load_keys(now);
        load_values(now);
        pages = look_up(v + kWaves);
        for (; v + kWaves < last; v += kWaves) {
            const Rows next = place(v + kWaves, pages);
            pages = look_up(v + 2 * kWaves);
            multiply(v, now, std::true_type{}, next);
            now = next;
        }
        multiply(v, now, std::false_type{}, now);
    }

    // The wavefronts' sums meet in LDS; wavefront w goes on with register w % 4 of some outputs, that is with kMine elements from
    // `element` on of query i.
    constexpr int kMine = kOuts * 4 / kWaves;
    const int reg = wave % 4, m0 = wave / 4 * kMine, element = (4 * g + reg) * kOuts + m0;
    float* const mine = &meet[wave][0][lane];
    mine[0] = base;
    mine[64] = l[0];
    #pragma unroll
    for (int m = 0; m < kOuts; ++m)
        #pragma unroll
        for (int r = 0; r < 4; ++r) mine[(2 + m * 4 + r) * 64] = acc[m][r];
    __syncthreads();
    float top = meet[0][0][lane];
    #pragma unroll
    for (int z = 1; z < kWaves; ++z) top = fmaxf(top, meet[z][0][lane]);
    float sum = 0.0f, o[kMine];
    #pragma unroll
    for (int m = 0; m < kMine; ++m) o[m] = 0.0f;
    #pragma unroll
    for (int z = 0; z < kWaves; ++z) {
        const float f = __builtin_amdgcn_exp2f(meet[z][0][lane] - top);
        sum += meet[z][1][lane] * f;
        #pragma unroll
        for (int m = 0; m < kMine; ++m) o[m] += meet[z][2 + (m0 + m) * 4 + reg][lane] * f;
    }

    if (parts > 1) {
        // The parts of a set meet in memory, at agent scope, which passes the XCDs' own L2s; the block that arrives last adds them up,
        // in their order.  No block waits for another.  The counter is 0 between launches.
        constexpr int kSlot = slot_floats(D) / 2;                    // pairs of floats
        auto* const slot = reinterpret_cast<uint64_t*>(sums) + static_cast<int64_t>(blockIdx.x) * kSlot;
        if (live) {
            #pragma unroll
            for (int m = 0; m < kMine; m += 2)
                __hip_atomic_store(slot + m / 2 * (64 * kWaves) + tid, __builtin_bit_cast(uint64_t, floatx2{o[m], o[m + 1]}), __ATOMIC_RELAXED,
                                   __HIP_MEMORY_SCOPE_AGENT);
            if (wave == 0 && g == 0)
                __hip_atomic_store(slot + 8 * D + i, __builtin_bit_cast(uint64_t, floatx2{top, sum}), __ATOMIC_RELAXED,
                                   __HIP_MEMORY_SCOPE_AGENT);
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        uint32_t* const counter = counters + (blockIdx.x - it.chunk * a.p.n_kv_heads);
        if (tid == 0) arrived = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __syncthreads();
        if (uniform(arrived) + 1 != static_cast<uint32_t>(parts)) return;
        asm volatile("" ::: "memory");
        if (tid == 0) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        const uint64_t* const slots = reinterpret_cast<const uint64_t*>(sums) +
                                      static_cast<int64_t>(blockIdx.x - it.chunk * a.p.n_kv_heads) * kSlot;
        const int64_t next = static_cast<int64_t>(a.p.n_kv_heads) * kSlot;
        const int col = live ? i : 0;
        auto pair_at = [&](int part, int at) {
            return __builtin_bit_cast(floatx2, __hip_atomic_load(slots + part * next + at, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
        };
        top = kStart;
        sum = 0.0f;
        #pragma unroll
        for (int m = 0; m < kMine; ++m) o[m] = 0.0f;
        const int at = live ? tid : tid & ~15;
        constexpr int kAhead = 32 / kMine;                     // parts asked for together
        for (int z0 = 0; z0 < parts; z0 += kAhead) {
            floatx2 bl[kAhead], x[kAhead][kMine / 2];
            #pragma unroll
            for (int z = 0; z < kAhead; ++z) {
                const int part = z0 + z < parts ? z0 + z : parts - 1;
                bl[z] = pair_at(part, 8 * D + col);
                #pragma unroll
                for (int m = 0; m < kMine; m += 2) x[z][m / 2] = pair_at(part, m / 2 * (64 * kWaves) + at);
            }
            #pragma unroll
            for (int z = 0; z < kAhead; ++z) {
                if (z0 + z >= parts) break;
                const float now = fmaxf(top, bl[z][0]), was = __builtin_amdgcn_exp2f(top - now), f = __builtin_amdgcn_exp2f(bl[z][0] - now);
                top = now;
                sum = sum * was + bl[z][1] * f;
                #pragma unroll
                for (int m = 0; m < kMine; ++m) o[m] = o[m] * was + x[z][m / 2][m & 1] * f;
            }
        }
    }
    if (!live) return;
    const float inv = __fdiv_rn(1.0f, sum);        // (not used where the sum is 0)
    uint16_t* const dst = a.out + (it.s.first + token) * a.ld_out + head * D + element;
    uint32_t h[kMine / 2];
    #pragma unroll
    for (int m = 0; m < kMine; m += 2) h[m / 2] = sum == 0.0f ? 0u : pack2(o[m] * inv, o[m + 1] * inv);      // (o may be NaN)
    if (reinterpret_cast<uintptr_t>(dst) % (2 * kMine) == 0) {
        if constexpr (kMine == 8) *reinterpret_cast<u32x4*>(dst) = u32x4{h[0], h[1], h[2], h[3]};
        else if constexpr (kMine == 4) *reinterpret_cast<u32x2*>(dst) = u32x2{h[0], h[1]};
        else *reinterpret_cast<uint32_t*>(dst) = h[0];
    } else {
        #pragma unroll
        for (int m = 0; m < kMine; ++m) dst[m] = static_cast<uint16_t>(h[m / 2] >> (16 * (m & 1)));
    }
}

// ---- many rows: tiles of keys in LDS, 32 rows per wavefront -------------------------------------------------
//
// A block has 128 or 64 rows of one sequence and key/value head, 32 per wavefront (v_mfma_f32_32x32x16_f16: twice the rows per
// operand that comes out of LDS), and takes its tiles of 64 keys through two buffers in LDS: while a tile is multiplied the next one
// is on its way to registers, and is written (int8 and Q4: as fp16, converted once for the block) behind it.  KS slices of a block
// take every KS-th tile, each with buffers of its own.
// Scores again transposed: lane (query = lane % 32, half h = lane / 32) has keys 8 a + 4 h + b of every 32, a, b = 0 .. 3, in
// registers 4 a + b, and registers 8 c .. 8 c + 7 are the B operand of the product with the values for keys 16 c + 4 h .. and 16 c + 8 +
// 4 h ..  The A operand, 4 keys of one element at a time, is what a transposed read from LDS gives.
// In a row of LDS the 16-byte piece p lies at p ^ twist(row): eight rows' pieces of one p, and four rows' two neighbouring pieces,
// are in different banks.
//
// What bounds it: a wavefront alone takes 1.3 us per tile at width 64, of which the matrix cores are busy 0.25 and the vector units
// (exponentials, maxima, conversions) 0.4; the rest is the chain barrier - keys from LDS - scores - weights - values - next tile to LDS, which
// only other wavefronts fill: matrix cores busy 25 % of the SIMD-cycles, vector units 34 %, LDS 38 % of the CU-cycles (a third of it
// bank conflicts) at 4096 rows of 32 heads over 8, width 128, window 1000 (0.55 PFLOP/s).  Tried and slower: the next tile's
// scores under this one's weights (32 or more registers), the next tile to LDS while scores are formed, all key operands read ahead.

constexpr int chunk_lds(int D) { return 2 * 2 * kChunkKeys * 2 * D; }          // of a slice's tiles
constexpr int chunk_lds_all(int D, int KS) { return KS * (chunk_lds(D) + 2 * kChunkKeys); }
constexpr int meet_floats(int D, int RW) { return RW * 64 * (D / 2 + 3); }         // of a slice's sums
__device__ __forceinline__ constexpr int twist(int row) { return (row & 3) * 2 + (row >> 2 & 1); }

// Dear: a row takes its keys one to a lane and its values one after the other.  A prompt of 2048 rows of 14 heads over 2 with one NaN among
// the values of a head's first, middle and last position 0.5, 3.2 and 5.5 ms instead of 0.03, 4096 rows of 32 over 8 0.8, 26 and 50 ms
// instead of 0.23 (single launches).
//
// Row `q` (fp16) of a query at position pos against tiles first .. last - 1 of a sequence, one key to a lane: where an infinity or a
// NaN in a place that some row must not see keeps the row off the matrix cores.  Leaves elements lane, lane + 64, .. of the sum of the
// weighted values, and the sums' base.
template <int KIND, int D>
__device__ __forceinline__ void row_by_itself(const AttentionArgs& a, const int* table, const Tiles& tiles, int first, int last, int pos, int kvh,
                                              const uint16_t* q, float (&o)[D / 64], float& base, float& sum) {
    const int lane = threadIdx.x & 63;
    base = kStart;
    sum = 0.0f;
    for (int d = 0; d < D / 64; ++d) o[d] = 0.0f;
    #pragma unroll 1
    for (int v = first; v < last; ++v) {
        const int j = tile_at(tiles, v) * 64 + lane;
        int lo = 0, hi = -1;                       // the key's row, in two halves; none
        float score = kNone;
        if (pos >= 0 && j < tiles.end && sees(pos, j, a.window, a.sinks)) {
            const int page = divide(j, a.p.page), number = table[page];
            if (static_cast<uint32_t>(number) < static_cast<uint32_t>(a.p.n_pages)) {
                const int64_t at = row_number(a.p, number, kvh, j - page * a.p.page.d);
                lo = static_cast<int>(at);
                hi = static_cast<int>(at >> 32);
                float dot = 0.0f;
                #pragma unroll 1
                for (int e = 0; e < D; ++e) dot = fmaf(h_f(q[e]), element<KIND, D>(a.p.k, a.p.k_scale, at, e), dot);
                score = dot * (a.scale * 1.44269504088896341f);
            }
        }
        const float now = fmaxf(base, wave_max(score) - kHead), was = __builtin_amdgcn_exp2f(base - now);
        const float w = hi < 0 ? 0.0f : static_cast<float>(static_cast<_Float16>(__builtin_amdgcn_exp2f(score - now)));
        base = now;
        sum *= was;
        for (int d = 0; d < D / 64; ++d) o[d] *= was;
        #pragma unroll 1
        for (int z = 0; z < 64; ++z) {
            const int zh = __builtin_amdgcn_readlane(hi, z);
            if (zh < 0) continue;
            const int64_t at = static_cast<uint32_t>(__builtin_amdgcn_readlane(lo, z)) | static_cast<int64_t>(zh) << 32;
            const float wz = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(w), z));
            sum += wz;
            for (int d = 0; d < D / 64; ++d) o[d] = fmaf(wz, element<KIND, D>(a.p.v, a.p.v_scale, at, lane + 64 * d), o[d]);
        }
    }
}

template <int KIND, int D, bool PAGES16, int RW, int KS>
__global__ __launch_bounds__(64 * RW * KS, 2) void paged_chunk_kernel(const AttentionArgs a, const Plan plan, float* __restrict__ partial,
                                                                          uint32_t* __restrict__ counters) {
    constexpr int kChunkWaves = RW, kChunkRows = 32 * RW;
    constexpr int kRow = row_bytes(KIND, D), kScales = row_scales(KIND, D);
    constexpr int kPiece = KIND == MI_KV_Q4 && D == 64 ? 8 : 16, kPieces = kRow / kPiece;      // of a row as it is stored
    constexpr int kPer = 64 * kChunkWaves / kPieces;                                           // rows that the block loads at a time
    constexpr int kLoads = kChunkKeys / kPer, kWords = kPiece / 4;
    static_assert(64 / kPieces <= 16, "a wavefront's rows of a load lie among 16");
    constexpr int kOps = D / 16, kOuts = D / 32;
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];                              // [2][keys, values][64][2 D]
    const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6) % kChunkWaves, slice = uniform(tid >> 6) / kChunkWaves;
    const int i = lane & 31, h = lane >> 5;
    const int kvh = blockIdx.x % a.p.n_kv_heads, y = blockIdx.x / a.p.n_kv_heads;
    const Item it = item_of<kChunkRows, kChunkKeys>(a, plan, y);
    if (it.b < 0) return;
    const int rows = it.s.n * plan.nrep, r0 = it.set * kChunkRows, r_end = r0 + kChunkRows < rows ? r0 + kChunkRows : rows;
    const Tiles tiles = tiles_of(it.s.pos + divide(r0, plan.rep), it.s.pos + divide(r_end - 1, plan.rep), a.p.cap, a.window, a.sinks, kChunkKeys);
    const int parts = tiles.count > 0 ? (tiles.count - 1) / it.share + 1 : 1;
    if (it.chunk >= parts) return;
    const int first = parts == 1 ? 0 : it.chunk * it.share;
    const int last = tiles.count - first < it.share ? tiles.count : first + it.share;
    // the wavefront's rows and the lane's query (past the last: that one, not stored)
    const int w0 = r0 + 32 * wave < r_end ? r0 + 32 * wave : r_end - 1, w_end = w0 + 32 < r_end ? w0 + 32 : r_end;
    const bool busy = r0 + 32 * wave < r_end, live = r0 + 32 * wave + i < r_end;
    const int row = w0 + i < w_end ? w0 + i : w_end - 1, token = divide(row, plan.rep), head = kvh * plan.nrep + (row - token * plan.nrep);
    const int my_pos = it.s.pos + token, p_lo = it.s.pos + divide(w0, plan.rep), p_hi = it.s.pos + divide(w_end - 1, plan.rep);
    const int before = (a.window > 0 && my_pos >= 0) ? my_pos - a.window : -1, sinks = a.window > 0 ? a.sinks : 0;
    half8 q[kOps];
    {
        const uint16_t* src = a.q + (it.s.first + token) * a.ld_q + head * D + 8 * h;
        const bool wide = reinterpret_cast<uintptr_t>(src) % 16 == 0;
        #pragma unroll
        for (int j = 0; j < kOps; ++j) {
            if (wide) q[j] = *reinterpret_cast<const half8*>(src + 16 * j);
            else
                #pragma unroll
                for (int e = 0; e < 8; ++e) q[j][e] = __builtin_bit_cast(_Float16, src[16 * j + e]);
        }
    }

    // ---- a tile from its pages to registers, and from there to LDS
    const auto* const table = reinterpret_cast<const __attribute__((address_space(4))) int*>(
        reinterpret_cast<uintptr_t>(a.p.pages + static_cast<int64_t>(it.b) * a.p.max_pages));
    const int my_row = wave * (64 / kPieces) + lane / kPieces, my_piece = lane % kPieces;      // of load 0; kPer rows on for the next
    struct Raw { uint32_t k[kLoads][kWords], v[kLoads][kWords]; uint16_t ks[kLoads], vs[kLoads]; uint32_t none; } raw;
    uint8_t* const own_lds = lds + slice * chunk_lds(D);
    uint8_t* const gone = lds + KS * chunk_lds(D) + slice * 2 * kChunkKeys;                                                  // [2][64]: keys that are not in the cache
    struct Pages { int number[kLoads]; };
    auto key_of = [&](int j0, int p) {             // PAGES16: of the wavefront, the first of its 16 rows; else the lane's
        const int r = p * kPer + (PAGES16 ? (wave * (64 / kPieces) & ~15) : my_row);
        return j0 + r < tiles.end ? j0 + r : tiles.end - 1;
    };
    auto look_up = [&](int v) {
        Pages g;
        const int j0 = tile_at(tiles, v < last ? v : last - 1) * kChunkKeys;
        #pragma unroll
        for (int p = 0; p < kLoads; ++p) g.number[p] = table[divide(key_of(j0, p), a.p.page)];
        return g;
    };
    auto fetch = [&](int v, const Pages& g) {
        const int j0 = tile_at(tiles, v) * kChunkKeys;
        raw.none = 0;
        #pragma unroll
        for (int p = 0; p < kLoads; ++p) {
            const int j = key_of(j0, p), number = g.number[p];
            const bool bad = static_cast<uint32_t>(number) >= static_cast<uint32_t>(a.p.n_pages);
            int slot = j - divide(j, a.p.page) * a.p.page.d;
            if constexpr (PAGES16) slot &= ~15;
            const int64_t at = row_number(a.p, bad ? 0 : number, kvh, slot);
            const uint32_t within = PAGES16 ? my_row & 15 : 0;
            const uint8_t *kb = a.p.k + at * kRow, *vb = a.p.v + at * kRow;
            const uint32_t off = within * kRow + my_piece * kPiece;
            load_words<4>(raw.k[p], kb + off);
            load_words<4>(raw.v[p], vb + off);
            if constexpr (kScales > 0) {
                const uint32_t so = (within * kScales + my_piece * kScales / kPieces) * 2;
                raw.ks[p] = *reinterpret_cast<const uint16_t*>(reinterpret_cast<const uint8_t*>(a.p.k_scale + at * kScales) + so);
                raw.vs[p] = *reinterpret_cast<const uint16_t*>(reinterpret_cast<const uint8_t*>(a.p.v_scale + at * kScales) + so);
            }
            // what is not in the cache becomes zeros
            if (bad || j0 + p * kPer + my_row >= tiles.end) raw.none |= 1u << p;
        }
    };
    uint32_t exponent = 0x64006400u;
    if constexpr (KIND == MI_KV_Q4) asm("" : "+v"(exponent));
    auto store = [&](uint8_t* to, const uint32_t (&w)[kWords], uint16_t scale, int r) {
        uint8_t* const line = to + r * (2 * D);
        auto put = [&](int piece, u32x4 x) { *reinterpret_cast<u32x4*>(line + 16 * (piece ^ twist(r))) = x; };
        if constexpr (KIND == MI_KV_F16) {
            put(my_piece, u32x4{w[0], w[1], w[2], w[3]});
        } else if constexpr (KIND == MI_KV_INT8) {
            #pragma unroll
            for (int e = 0; e < 2; ++e) {
                u32x4 x;
                #pragma unroll
                for (int z = 0; z < 2; ++z) {
                    x[2 * z] = scaled(from_bytes<0, 1>(w[2 * e + z], w[2 * e + z]), both(scale));
                    x[2 * z + 1] = scaled(from_bytes<2, 3>(w[2 * e + z], w[2 * e + z]), both(scale));
                }
                put(2 * my_piece + e, x);
            }
        } else {
            #pragma unroll
            for (int e = 0; e < kWords; ++e) {
                uint32_t c[4];
                #pragma unroll
                for (int z = 0; z < 4; ++z) c[z] = scaled(from_nibbles(w[e] >> (4 * z), exponent), both(scale));
                put(kWords * my_piece + e, u32x4{__builtin_amdgcn_perm(c[1], c[0], 0x05040100u), __builtin_amdgcn_perm(c[3], c[2], 0x05040100u),
                                                 __builtin_amdgcn_perm(c[1], c[0], 0x07060302u), __builtin_amdgcn_perm(c[3], c[2], 0x07060302u)});
            }
        }
    };
    auto stash = [&](int buf) {
        uint8_t* const kt = own_lds + buf * (chunk_lds(D) / 2);
        if (__builtin_expect(__any(raw.none), 0)) {
            #pragma unroll
            for (int p = 0; p < kLoads; ++p)
                if (raw.none >> p & 1) {
                    #pragma unroll
                    for (int e = 0; e < kWords; ++e) raw.k[p][e] = raw.v[p][e] = 0;
                    raw.ks[p] = raw.vs[p] = 0;
                }
        }
        #pragma unroll
        for (int p = 0; p < kLoads; ++p) {
            if (my_piece == 0) gone[buf * kChunkKeys + p * kPer + my_row] = raw.none >> p & 1;
            store(kt, raw.k[p], raw.ks[p], p * kPer + my_row);
            store(kt + chunk_lds(D) / 4, raw.v[p], raw.vs[p], p * kPer + my_row);
        }
    };

    floatx16 acc[kOuts];
    #pragma unroll
    for (int m = 0; m < kOuts; ++m)
        #pragma unroll
        for (int r = 0; r < 16; ++r) acc[m][r] = 0.0f;
    float base = kStart, sum = 0.0f;               // sum: of the lane's weights, as they meet the values
    const float scale_log2 = a.scale * 1.44269504088896341f;
    // lane addresses within a tile: of a key operand, piece 2 j + h of row i; of a value operand, 4 rows of 16 elements for 16 lanes
    const int vr = 4 * h + (lane & 15) / 4, vc = (lane >> 4 & 1) * 2 + (lane & 3) / 2, vo = (lane & 1) * 8;

    bool odd = false, far = false;                 // see below; some query's base is beyond kFar
    auto multiply = [&](int v, int buf) {
        const int j0 = tile_at(tiles, v) * kChunkKeys;
        const uint8_t* const kt = own_lds + buf * (chunk_lds(D) / 2);
        const uint8_t* const vt = kt + chunk_lds(D) / 4;
        floatx16 s[2];
        #pragma unroll
        for (int t = 0; t < 2; ++t) {
            #pragma unroll
            for (int r = 0; r < 16; ++r) s[t][r] = 0.0f;
            #pragma unroll
            for (int j = 0; j < kOps; ++j)
                s[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(
                    *reinterpret_cast<const half8*>(kt + (32 * t + i) * (2 * D) + 16 * ((2 * j + h) ^ twist(i))), q[j], s[t], 0, 0, 0);
        }
        const uint64_t absent = __ballot(gone[buf * kChunkKeys + lane] != 0);
        const bool masked = !all_seen(j0, kChunkKeys, p_lo, p_hi, a.p.cap, a.window, a.sinks) || absent != 0;
        if (__builtin_expect(masked, 0)) {
            asm volatile("");
            #pragma unroll
            for (int t = 0; t < 2; ++t)
                #pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int j = j0 + 32 * t + 8 * (r / 4) + 4 * h + r % 4;
                    const uint32_t out = static_cast<uint32_t>(absent >> (32 * t)) >> (4 * h) >> (8 * (r / 4) + r % 4) & 1;
                    const bool see = (out == 0) & (j <= my_pos) & ((j > before) | (j < sinks));
                    s[t][r] = see ? s[t][r] : kNone;
                }
        }
        float tops[4];
        #pragma unroll
        for (int z = 0; z < 4; ++z) tops[z] = max3(s[z / 2][8 * (z % 2)], s[z / 2][8 * (z % 2) + 1], s[z / 2][8 * (z % 2) + 2]);
        #pragma unroll
        for (int r = 3; r < 7; r += 2)
            #pragma unroll
            for (int z = 0; z < 4; ++z) tops[z] = max3(tops[z], s[z / 2][8 * (z % 2) + r], s[z / 2][8 * (z % 2) + r + 1]);
        float top = max3(max3(tops[0], s[0][7], tops[1]), max3(s[0][15], tops[2], s[1][7]), max3(tops[3], s[1][15], s[1][15]));
        if (__builtin_expect(__any(top * scale_log2 - kHead > base + kSlack), 0)) {
            unsigned u = __float_as_uint(base_of(top, scale_log2));
            const auto both_halves = __builtin_amdgcn_permlane32_swap(u, u, false, false);
            top = max3(base, __uint_as_float(both_halves[0]), __uint_as_float(both_halves[1]));
            const float alpha = __builtin_amdgcn_exp2f(base - top);
            sum *= alpha;
            #pragma unroll
            for (int m = 0; m < kOuts; ++m) acc[m] *= alpha;
            base = top;
            far = __any(fabsf(base) >= kFar && base > kStart);
        }
        float by = scale_log2, from = base;
        if (__builtin_expect(far, 0)) {
            asm volatile("");
            #pragma unroll
            for (int t = 0; t < 2; ++t)
                #pragma unroll
                for (int r = 0; r < 16; ++r) s[t][r] = far_exponent(s[t][r], scale_log2, base);
            by = 1.0f;
            from = 0.0f;
        }
        uint32_t w[2][8];                          // weights, two to a word
        float sums[4] = {sum, 0.0f, 0.0f, 0.0f};
        #pragma unroll
        for (int t = 0; t < 2; ++t)
            #pragma unroll
            for (int r = 0; r < 16; r += 2) {
                w[t][r / 2] = pack2(__builtin_amdgcn_exp2f(fmaf(s[t][r], by, -from)), __builtin_amdgcn_exp2f(fmaf(s[t][r + 1], by, -from)));
                float& part = sums[2 * t + r / 2 % 2];
                part = __builtin_amdgcn_fdot2(__builtin_bit_cast(half2v, w[t][r / 2]), half2v{static_cast<_Float16>(1.0f), static_cast<_Float16>(1.0f)}, part, false);
            }
        sum = (sums[0] + sums[1]) + (sums[2] + sums[3]);
        // operand m, keys 16 c ..: two reads of 4 keys
        auto values = [&](int m, int c) {
            u32x4 x;
            #pragma unroll
            for (int z = 0; z < 2; ++z) {
                const int r = 16 * c + 8 * z + vr;
                const short4v y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4v*)(
                    vt + r * (2 * D) + 16 * ((4 * m + vc) ^ twist(r)) + vo));
                const u32x2 two = __builtin_bit_cast(u32x2, y);
                x[2 * z] = two[0];
                x[2 * z + 1] = two[1];
            }
            return x;
        };
        auto weights = [&](int c) { return __builtin_bit_cast(half8, u32x4{w[c / 2][4 * (c % 2)], w[c / 2][4 * (c % 2) + 1], w[c / 2][4 * (c % 2) + 2], w[c / 2][4 * (c % 2) + 3]}); };
        if (__builtin_expect(masked, 0)) {
            // A masked key has weight 0, but 0 x inf and 0 x NaN are NaN: where there is an infinity or a NaN in a tile that is masked
            // for some query, the wavefront does its rows again in the end (row_by_itself), whatever comes out here.
            uint32_t most = 0;
            #pragma unroll
            for (int c = 0; c < 4; ++c)
                #pragma unroll
                for (int m = 0; m < kOuts; ++m) {
                    const u32x4 x = values(m, c);
                    #pragma unroll
                    for (int z = 0; z < 4; ++z) most |= odd_halves(x[z]);
                }
            odd |= __any(most) != 0;
        }
        #pragma unroll
        for (int c = 0; c < 4; ++c)
            #pragma unroll
            for (int m = 0; m < kOuts; ++m)
                acc[m] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8, values(m, c)), weights(c), acc[m], 0, 0, 0);
    };

    // registers -> LDS, the next tile requested, one barrier (a buffer is written again two barriers after it was last read),
    // the tile multiplied unless the wavefront's queries see nothing of it
    // (of KS slices: tiles first + slice, + KS, ..; past the last that one again, not multiplied)
    Pages pages;
    const int mine = first + slice;
    auto clamp = [&](int v) { return v < last ? v : last - 1; };
    if (first < last) {
        pages = look_up(mine);
        fetch(clamp(mine), pages);
        pages = look_up(mine + KS);
    }
    for (int v = mine, buf = 0; v - slice < last; v += KS, buf ^= 1) {
        stash(buf);
        if (v - slice + KS < last) {
            fetch(clamp(v + KS), pages);
            pages = look_up(v + 2 * KS);
        }
        __syncthreads();
        if (v < last) {
            const int j0 = tile_at(tiles, v) * kChunkKeys;
            const int w_first = a.window > 0 && p_lo >= a.window ? p_lo - a.window + 1 : 0;    // of the window of the wavefront's first query
            if (busy && j0 <= p_hi && (j0 + (kChunkKeys - 1) >= w_first || j0 < sinks)) multiply(v, buf);
        }
    }
    if constexpr (KS > 1) {
        // The other slices' sums come to the first by LDS, in their order.
        __syncthreads();
        constexpr int kBox = meet_floats(D, RW);
        float* const box = reinterpret_cast<float*>(lds) + wave * 64 * (D / 2 + 3) + lane;
        if (slice > 0) {
            float* const to = box + (slice - 1) * kBox;
            to[0] = base;
            to[64] = sum;
            to[128] = odd ? 1.0f : 0.0f;
            #pragma unroll
            for (int m = 0; m < kOuts; ++m)
                #pragma unroll
                for (int r = 0; r < 16; ++r) to[(3 + 16 * m + r) * 64] = acc[m][r];
        }
        __syncthreads();
        if (slice > 0) return;
        #pragma unroll
        for (int z = 0; z < KS - 1; ++z) {
            const float* const from = box + z * kBox;
            const float now = fmaxf(base, from[0]), was = __builtin_amdgcn_exp2f(base - now), f = __builtin_amdgcn_exp2f(from[0] - now);
            base = now;
            sum = sum * was + from[64] * f;
            odd |= __any(from[128] != 0.0f) != 0;
            #pragma unroll
            for (int m = 0; m < kOuts; ++m)
                #pragma unroll
                for (int r = 0; r < 16; ++r) acc[m][r] = acc[m][r] * was + from[(3 + 16 * m + r) * 64] * f;
        }
    }
    if (!busy) return;
    constexpr int kSlot = chunk_slot_floats(D, RW) / 2, kPairs = kOuts * 8;           // pairs of floats: of a block, of a lane
    auto* const all = reinterpret_cast<uint64_t*>(partial);
    const int64_t own = static_cast<int64_t>(blockIdx.x) * kSlot;
    const int at = wave * kPairs * 64 + lane, at_sum = kChunkWaves * kPairs * 64 + wave * 32 + i;
    if (__builtin_expect(odd, 0)) {
        #pragma unroll 1
        for (int z = 0; z < 32 && w0 + z < w_end; ++z) {
            const int r = w0 + z, t = divide(r, plan.rep), hd = kvh * plan.nrep + (r - t * plan.nrep);
            float o[D / 64], b, l;
            row_by_itself<KIND, D>(a, a.p.pages + static_cast<int64_t>(it.b) * a.p.max_pages, tiles, first, last, it.s.pos + t, kvh, a.q + (it.s.first + t) * a.ld_q + hd * D, o, b, l);
            #pragma unroll
            for (int e = 0; e < D / 64; ++e) {
                const int d = lane + 64 * e, reg = 4 * (d % 32 / 8) + d % 4, place = (d / 4 % 2) * 32 + z;   // as the others lie in the registers
                if (parts == 1)
                    a.out[(it.s.first + t) * a.ld_out + hd * D + d] = f_h(l == 0.0f ? 0.0f : o[e] / l);
                else
                    __hip_atomic_store(reinterpret_cast<float*>(all + own + wave * kPairs * 64 + (d / 32 * 8 + reg / 2) * 64 + place) + reg % 2, o[e],
                                       __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            }
            if (parts > 1 && lane == 0)
                __hip_atomic_store(all + own + kChunkWaves * kPairs * 64 + wave * 32 + z, __builtin_bit_cast(uint64_t, floatx2{b, l}), __ATOMIC_RELAXED,
                                   __HIP_MEMORY_SCOPE_AGENT);
        }
        if (parts == 1) return;
    } else {
        const auto halves = __builtin_amdgcn_permlane32_swap(__float_as_uint(sum), __float_as_uint(sum), false, false);
        sum = __uint_as_float(halves[0]) + __uint_as_float(halves[1]);
        if (parts > 1) {
            // (as in paged_step_kernel, but every wavefront for its own rows)
            #pragma unroll
            for (int m = 0; m < kOuts; ++m)
                #pragma unroll
                for (int r = 0; r < 16; r += 2)
                    __hip_atomic_store(all + own + at + (m * 8 + r / 2) * 64, __builtin_bit_cast(uint64_t, floatx2{acc[m][r], acc[m][r + 1]}),
                                       __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            if (h == 0)
                __hip_atomic_store(all + own + at_sum, __builtin_bit_cast(uint64_t, floatx2{base, sum}), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
    }
    if (parts > 1) {
        const int64_t zero_at = static_cast<int64_t>(blockIdx.x - it.chunk * a.p.n_kv_heads) * kSlot, next = static_cast<int64_t>(a.p.n_kv_heads) * kSlot;
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        uint32_t* const counter = counters + (blockIdx.x - it.chunk * a.p.n_kv_heads) * kChunkWaves + wave;
        uint32_t arrived = 0;
        if (lane == 0) arrived = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        if (static_cast<uint32_t>(uniform(arrived)) + 1 != static_cast<uint32_t>(parts)) return;
        asm volatile("" ::: "memory");
        if (lane == 0) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        auto pair_at = [&](int part, int64_t k) {
            return __builtin_bit_cast(floatx2, __hip_atomic_load(all + zero_at + part * next + k, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
        };
        base = kStart;
        sum = 0.0f;
        #pragma unroll
        for (int m = 0; m < kOuts; ++m)
            #pragma unroll
            for (int r = 0; r < 16; ++r) acc[m][r] = 0.0f;
        #pragma unroll 1
        for (int z = 0; z < parts; ++z) {
            const floatx2 bl = pair_at(z, at_sum);
            floatx2 x[kPairs];
            #pragma unroll
            for (int k = 0; k < kPairs; ++k) x[k] = pair_at(z, at + k * 64);
            const float now = fmaxf(base, bl[0]), was = __builtin_amdgcn_exp2f(base - now), f = __builtin_amdgcn_exp2f(bl[0] - now);
            base = now;
            sum = sum * was + bl[1] * f;
            #pragma unroll
            for (int m = 0; m < kOuts; ++m)
                #pragma unroll
                for (int r = 0; r < 16; ++r) acc[m][r] = acc[m][r] * was + x[m * 8 + r / 2][r & 1] * f;
        }
    }
    if (!live) return;
    const float inv = __fdiv_rn(1.0f, sum);        // (not used where the sum is 0)
    uint16_t* const dst = a.out + (it.s.first + token) * a.ld_out + head * D + 4 * h;
    const bool wide = reinterpret_cast<uintptr_t>(dst) % 8 == 0;
    #pragma unroll
    for (int m = 0; m < kOuts; ++m)
        #pragma unroll
        for (int e = 0; e < 4; ++e) {
            u32x2 x = {pack2(acc[m][4 * e] * inv, acc[m][4 * e + 1] * inv), pack2(acc[m][4 * e + 2] * inv, acc[m][4 * e + 3] * inv)};
            if (sum == 0.0f) x = u32x2{0, 0};      // (acc may be NaN)
            uint16_t* const to = dst + 32 * m + 8 * e;
            if (wide) {
                *reinterpret_cast<u32x2*>(to) = x;
            } else {
                #pragma unroll
                for (int z = 0; z < 4; ++z) to[z] = static_cast<uint16_t>(x[z / 2] >> (16 * (z & 1)));
            }
        }
}

struct PartRoom {             // of the stream: where parts of a sequence's keys meet (null: nowhere)
    float* sums = nullptr;
    uint32_t* counters = nullptr;
};

template <int KIND, int D>
bool launch_step(hipStream_t s, const AttentionArgs& a, const PartRoom& room, const PagedLaunch& l) {
    auto go = [&](auto kern) {
        hipLaunchKernelGGL(kern, dim3(static_cast<unsigned>(l.blocks)), dim3(l.threads), 0, s, a, l.plan, room.sums, room.counters);
    };
    if (a.p.page.d % 16 == 0) go(paged_step_kernel<KIND, D, true>);
    else go(paged_step_kernel<KIND, D, false>);
    return MI_HIP_OK(hipGetLastError());
}

template <int KIND, int D, int RW, int KS>
bool launch_chunk(hipStream_t s, const AttentionArgs& a, const PartRoom& room, const PagedLaunch& l) {
    constexpr int lds = chunk_lds_all(D, KS);
    static_assert(lds <= 160 * 1024 && (KS - 1) * meet_floats(D, RW) * 4 <= KS * chunk_lds(D), "tiles and sums fit");
    auto go = [&](auto pages16) {                  // (a type of its own for each, so that each has its attribute set once)
        const auto kern = paged_chunk_kernel<KIND, D, decltype(pages16)::value, RW, KS>;
        if (lds > 65536 && !MI_ONCE_OK(MI_HIP_OK(hipFuncSetAttribute(reinterpret_cast<const void*>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, lds))))
            return false;
        hipLaunchKernelGGL(kern, dim3(static_cast<unsigned>(l.blocks)), dim3(l.threads), lds, s, a, l.plan, room.sums, room.counters);
        return MI_HIP_OK(hipGetLastError());
    };
    return a.p.page.d % 16 == 0 ? go(std::true_type{}) : go(std::false_type{});
}

// One of the launches that paged_plan.h chooses: of the kernel for many rows, blocks of 64 rows in four slices of keys (width 64), of
// 128 in two (width 128) or in one.
template <int KIND, int D>
bool launch(hipStream_t s, const AttentionArgs& a, const PartRoom& room, const PagedLaunch& l) {
    constexpr int kWavesSliced = D == 64 ? 2 : 4, kSlices = D == 64 ? 4 : 2;
    if (l.wavefronts == 0) return launch_step<KIND, D>(s, a, room, l);
    return l.slices == 1 ? launch_chunk<KIND, D, 4, 1>(s, a, room, l) : launch_chunk<KIND, D, kWavesSliced, kSlices>(s, a, room, l);
}

}  // namespace

bool launch_paged_attention(hipStream_t s, const AttentionArgs& a, const StreamRoom& own) {
    PartRoom room;
    if (own.workspace && own.sums) room = {static_cast<float*>(own.sums), slice_counters(own.workspace)};
    const AttentionSize size = {a.p.n_seqs, a.p.n_tokens, a.max_tokens, a.p.cap, a.n_heads, a.p.n_kv_heads, a.head_dim, a.window, a.sinks};
    const PagedLaunches all = attention_launches(size, room.sums ? Room{kPartialBytes, kSliceCounters} : Room{}, device_info().cus);
    if (const int64_t blocks = too_many_blocks(all)) {     // (of any of the launches, before the first is enqueued)
        MI_ERROR_FMT("mi_attention: %lld blocks are more than a launch counts", static_cast<long long>(blocks));
        return false;
    }
    const bool wide = a.head_dim == 128;
    for (int i = 0; i < all.n; ++i) {
        const PagedLaunch& l = all.of[i];
        const bool ok = a.kind == MI_KV_F16    ? wide ? launch<MI_KV_F16, 128>(s, a, room, l) : launch<MI_KV_F16, 64>(s, a, room, l)
                        : a.kind == MI_KV_INT8 ? wide ? launch<MI_KV_INT8, 128>(s, a, room, l) : launch<MI_KV_INT8, 64>(s, a, room, l)
                                               : wide ? launch<MI_KV_Q4, 128>(s, a, room, l) : launch<MI_KV_Q4, 64>(s, a, room, l);
        if (!ok) return false;
    }
    return true;
}

}  // namespace mi
