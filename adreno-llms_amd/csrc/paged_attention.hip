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

namespace mi {
namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef float floatx2 __attribute__((ext_vector_type(2)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

constexpr float kNone = -__builtin_huge_valf();  // the score of a key that the query does not see
constexpr float kStart = -1.0e30f;               // the running maximum of a query that has seen no key
// Weights are exp2(score - base) with base between 2^-7 and 2^8 .. below the greatest: between 2^7 and 2^15 for the greatest
// score, so that fp16 holds weights down to 2^-21 of it at full precision, and the maximum may rise by 2^kSlack before the
// sums are rescaled.
constexpr float kHead = 7.0f, kSlack = 8.0f;

// The greater of a lane's value and those of the lanes 16, 32 and 48 away.
__device__ __forceinline__ float max_of_groups(float a) {
    unsigned u = __float_as_uint(a);
    auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    u = __float_as_uint(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
    r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
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
__device__ __forceinline__ float wave_sum(float x) {
    #pragma unroll
    for (int s = 32; s > 0; s /= 2) x += __shfl_xor(x, s);
    return x;
}

// ---- who does what --------------------------------------------------------------------------------------
//
// The lengths are known to the device alone.  A block works on some tiles of keys for 16 ROWS-row sets of one sequence and
// key/value head; how many tiles that are follows from the tiles of the whole batch, so that every block gets about as
// many whatever the mixture of lengths: `share` tiles, such that the items fit the `target` blocks that the chip holds plus
// one per set.  Every wavefront works that out for itself from q_start and kv_len: the loads are those that it
// needs anyway.

struct Plan {                 // from the host
    int target;               // items per key/value head beside one per set; 0: keys are not split
    int least;                // tiles of keys that a block is worth
    int nrep;
    Divider rep;              // by nrep
};
struct Item {
    int b = -1, set = 0, chunk = 0, share = 0;
    Span s;
};

struct Cost { int sets, tiles; };
template <int ROWS, int KEYS>
__device__ __forceinline__ Cost cost_of(const AttentionArgs& a, const Plan& plan, const Span& s) {
    if (s.n <= 0) return {0, 0};
    const int count = tiles_of(s.pos, s.pos + s.n - 1, a.p.cap, a.window, a.sinks, KEYS).count;
    return {(s.n * plan.nrep + ROWS - 1) / ROWS, count > 0 ? count : 1};
}

// Item `y` of the batch (of any one key/value head); b = -1: there is none.
template <int ROWS, int KEYS>
__device__ __forceinline__ Item item_of(const AttentionArgs& a, const Plan& plan, const int y) {
    const int lane = threadIdx.x & 63;
    auto span = [&](int b) {
        return b < a.p.n_seqs ? span_of(a.p.q_start[b], a.p.q_start[b + 1], a.p.kv_len[b], a.p.n_tokens) : Span{};
    };
    Item it;
    Span s = span(lane);
    Cost c = cost_of<ROWS, KEYS>(a, plan, s);
    it.share = 0x7fffffff;
    if (plan.target > 0) {
        float total = static_cast<float>(c.sets) * static_cast<float>(c.tiles);
        for (int b0 = 64; b0 < a.p.n_seqs; b0 += 64) {
            const Cost more = cost_of<ROWS, KEYS>(a, plan, span(b0 + lane));
            total += static_cast<float>(more.sets) * static_cast<float>(more.tiles);
        }
        // (a hundred-thousandth more: the sum's rounding must not make an item too many)
        const float each = wave_sum(total) * 1.00001f / static_cast<float>(plan.target);
        it.share = each < 1.0e9f ? static_cast<int>(each) + 1 : 0x7fffffff;
        if (it.share < plan.least) it.share = plan.least;
        it.share = uniform(it.share);
    }
    int before = 0;
    for (int b0 = 0;; ) {
        const int chunks = c.sets ? (c.tiles - 1) / it.share + 1 : 0, upto = scan(c.sets * chunks) + before;
        const uint64_t past = __ballot(upto > y);
        if (past) {
            const int l = uniform(__builtin_ctzll(past));
            it.b = b0 + l;
            it.s.first = __builtin_amdgcn_readlane(s.first, l);
            it.s.n = __builtin_amdgcn_readlane(s.n, l);
            it.s.pos = __builtin_amdgcn_readlane(s.pos, l);
            const int n = __builtin_amdgcn_readlane(chunks, l), sets = __builtin_amdgcn_readlane(c.sets, l);
            const int own = y - (__builtin_amdgcn_readlane(upto, l) - sets * n);
            it.set = sets == 1 ? 0 : own / n;
            it.chunk = own - it.set * n;
            return it;
        }
        before = __builtin_amdgcn_readlane(upto, 63);
        b0 += 64;
        if (b0 >= a.p.n_seqs) return it;
        s = span(b0 + lane);
        c = cost_of<ROWS, KEYS>(a, plan, s);
    }
}

// ---- a tile of 32 keys as it comes from the cache, and as operands ------------------------------------------

// Keys as A operand of q k: of 16 n + i, n = 0, 1, the elements g D / 4 .. (every group a quarter, so that pieces of rows are long;
// which elements meet in one product does not matter as long as the query brings the same).  Values as A operand of
// the product with the weights: of keys 4 g .. and 16 + 4 g .., the elements i D / 16 .., D / 16 of them, which become row i of
// D / 16 operands: element m of the piece is row i of operand m.  The transpose is then one byte permute per two numbers.
template <int KIND, int D>
struct Tile {
    static constexpr int kK = row_bytes(KIND, D) / 4 / 4;      // words of a key's piece
    static constexpr int kVBytes = row_bytes(KIND, D) / 16;    // bytes of a value's piece: 2, 4, 8, 16
    static constexpr int kV = (kVBytes + 3) / 4;
    uint32_t k[2][kK], v[8][kV];
    uint16_t ks[2], vs[8];                                     // their scales
    bool bad[2];                                               // 16 keys whose page is not in the pool (pages by 16 keys)
    uint32_t absent;                                           // bit e: key e of the lane's values, bit 8 + n: its key n has no page
};

template <int N>
__device__ __forceinline__ void load_words(uint32_t (&w)[N], const uint8_t* p) {
    if constexpr (N % 4 == 0) {
        #pragma unroll
        for (int j = 0; j < N; j += 4) {
            const u32x4 x = *reinterpret_cast<const u32x4*>(p + 4 * j);
            w[j] = x[0]; w[j + 1] = x[1]; w[j + 2] = x[2]; w[j + 3] = x[3];
        }
    } else if constexpr (N == 2) {
        const u32x2 x = *reinterpret_cast<const u32x2*>(p);
        w[0] = x[0]; w[1] = x[1];
    } else {
        w[0] = *reinterpret_cast<const uint32_t*>(p);
    }
}

// Codes as fp16 numbers: a byte (plus 128) or nibble (plus 8) under the exponent of 1024 is that number above 1024.
__device__ __forceinline__ uint32_t from_codes(uint32_t w, _Float16 above, half2v scale) {
    const half2v x = (__builtin_bit_cast(half2v, w) - half2v{above, above}) * scale;
    return __builtin_bit_cast(uint32_t, x);
}
__device__ __forceinline__ half2v both(uint16_t s) { return __builtin_bit_cast(half2v, s * 0x00010001u); }

// Operand j (8 elements) of a key's piece.  Q4: elements come as 0 4 1 5 2 6 3 7 of each 8, and so does the query.
template <int KIND, int N>
__device__ __forceinline__ half8 key_operand(const uint32_t (&w)[N], int j, uint16_t scale) {
    if constexpr (KIND == MI_KV_F16) return __builtin_bit_cast(half8, u32x4{w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]});
    u32x4 r;
    const half2v s = both(scale);
    if constexpr (KIND == MI_KV_INT8) {
        #pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint32_t u = w[2 * j + h];
            r[2 * h] = from_codes(__builtin_amdgcn_perm(0, u, 0x0c010c00u) ^ 0x64806480u, static_cast<_Float16>(1152.0f), s);
            r[2 * h + 1] = from_codes(__builtin_amdgcn_perm(0, u, 0x0c030c02u) ^ 0x64806480u, static_cast<_Float16>(1152.0f), s);
        }
    } else {
        #pragma unroll
        for (int h = 0; h < 4; ++h)
            r[h] = from_codes(((w[j] >> (4 * h)) & 0x000f000fu) | 0x64006400u, static_cast<_Float16>(1032.0f), s);
    }
    return __builtin_bit_cast(half8, r);
}

// Keys 2 p and 2 p + 1 of the lane's values, element m of their pieces.
template <int KIND, int D>
__device__ __forceinline__ uint32_t value_pair(const Tile<KIND, D>& t, int p, int m) {
    const auto &lo = t.v[2 * p], &hi = t.v[2 * p + 1];
    if constexpr (KIND == MI_KV_F16)
        return __builtin_amdgcn_perm(hi[m / 2], lo[m / 2], m & 1 ? 0x07060302u : 0x05040100u);
    const half2v s = __builtin_bit_cast(half2v, static_cast<uint32_t>(t.vs[2 * p]) | static_cast<uint32_t>(t.vs[2 * p + 1]) << 16);
    if constexpr (KIND == MI_KV_INT8) {
        const uint32_t sel = 0x0c040c00u + 0x00010001u * (m % 4);
        return from_codes(__builtin_amdgcn_perm(hi[m / 4], lo[m / 4], sel) ^ 0x64806480u, static_cast<_Float16>(1152.0f), s);
    } else {
        const uint32_t two = __builtin_amdgcn_perm(hi[0], lo[0], m < 4 ? 0x05040100u : 0x07060302u);
        return from_codes(((two >> (4 * (m % 4))) & 0x000f000fu) | 0x64006400u, static_cast<_Float16>(1032.0f), s);
    }
}

// Whether any of the lane's values that are in the cache (`there`, a mask for each pair of keys) may be an infinity or a NaN:
// of fp16 its greatest, else its scales (256 and more count, as their products may overflow).
template <int KIND, int D>
__device__ __forceinline__ bool odd_values(const Tile<KIND, D>& t, const uint32_t (&there)[4]) {
    uint16_t most = 0;
    #pragma unroll
    for (int e = 0; e < 8; ++e) {
        const uint16_t have = static_cast<uint16_t>(there[e / 2] >> (16 * (e & 1)));
        if constexpr (KIND == MI_KV_F16) {
            #pragma unroll
            for (int w = 0; w < Tile<KIND, D>::kV; ++w)
                #pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint16_t x = static_cast<uint16_t>(t.v[e][w] >> (16 * h)) & have & 0x7fffu;
                    most = x > most ? x : most;
                }
        } else {
            const uint16_t x = t.vs[e] & have & 0x7fffu;
            most = x > most ? x : most;
        }
    }
    return most >= (KIND == MI_KV_F16 ? 0x7c00u : 0x5c00u);
}

// ---- few rows: keys straight from memory to registers -----------------------------------------------------

constexpr int kRows = 16, kKeys = 32;
constexpr int kWaves = 4;                          // wavefronts per block; they take the block's tiles in turn
constexpr int slot_floats(int D) { return 16 * D + 32; }

// PAGES16: pages are multiples of 16 positions long, so 16 keys lie in one page.
template <int KIND, int D, bool PAGES16>
__global__ __launch_bounds__(64 * kWaves, D == 128 ? 2 : 3) void paged_step_kernel(const AttentionArgs a, const Plan plan, float* __restrict__ sums,
                                                                 uint32_t* __restrict__ counters) {
    constexpr int kOps = D / 32, kOuts = D / 16;   // operands of a key, of the values
    constexpr int kRow = row_bytes(KIND, D), kScales = row_scales(KIND, D);
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
    half8 q[kOps];
    {
        const uint16_t* src = a.q + (it.s.first + token) * a.ld_q + head * D + g * (D / 4);
        const bool wide = reinterpret_cast<uintptr_t>(src) % 16 == 0;
        #pragma unroll
        for (int j = 0; j < kOps; ++j) {
            half8 x;
            if (wide) x = *reinterpret_cast<const half8*>(src + 8 * j);
            else
                #pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = __builtin_bit_cast(_Float16, src[8 * j + e]);
            q[j] = KIND == MI_KV_Q4 ? __builtin_shufflevector(x, x, 0, 4, 1, 5, 2, 6, 3, 7) : x;
        }
    }

    const int* const table = a.p.pages + static_cast<int64_t>(it.b) * a.p.max_pages;
    auto fetch = [&](Tile<KIND, D>& t, int v) {
        const int j0 = tile_at(tiles, v) * kKeys;
        t.absent = 0;
        t.bad[0] = t.bad[1] = false;
        #pragma unroll
        for (int n = 0; n < 2; ++n) {
            const uint8_t *kp, *vp[4];
            const uint16_t *ksp = nullptr, *vsp[4] = {};
            if constexpr (PAGES16) {
                const int j = j0 + 16 * n < tiles.end ? j0 + 16 * n : j0;
                const int page = divide(j, a.p.page);
                int number = uniform(table[page]);
                t.bad[n] = number < 0 || number >= a.p.n_pages;
                number = t.bad[n] ? 0 : number;
                const int64_t at = row_number(a.p, number, kvh, j - page * a.p.page.d);
                kp = a.p.k + at * kRow + i * kRow + g * (kRow / 4);
                const uint8_t* vb = a.p.v + at * kRow + 4 * g * kRow + i * (kRow / 16);
                #pragma unroll
                for (int e = 0; e < 4; ++e) vp[e] = vb + e * kRow;
                if constexpr (kScales > 0) {
                    ksp = a.p.k_scale + at * kScales + i * kScales;
                    const uint16_t* vsb = a.p.v_scale + at * kScales + 4 * g * kScales;
                    #pragma unroll
                    for (int e = 0; e < 4; ++e) vsp[e] = vsb + e * kScales;
                }
            } else {
                const int mine = j0 + 16 * n + i, j = mine < tiles.end ? mine : tiles.end - 1;
                const int page = divide(j, a.p.page), number = table[page];
                const bool none = number < 0 || number >= a.p.n_pages;
                if (none) t.absent |= 256u << n;
                const int64_t at = row_number(a.p, none ? 0 : number, kvh, j - page * a.p.page.d);
                kp = a.p.k + at * kRow + g * (kRow / 4);
                ksp = a.p.k_scale + at * kScales;
                const int at_lo = static_cast<int>(at), at_hi = static_cast<int>(at >> 32);
                #pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int64_t from = static_cast<uint32_t>(__shfl(at_lo, 4 * g + e)) | static_cast<int64_t>(__shfl(at_hi, 4 * g + e)) << 32;
                    if (__shfl(static_cast<int>(none), 4 * g + e)) t.absent |= 1u << (4 * n + e);
                    vp[e] = a.p.v + from * kRow + i * (kRow / 16);
                    vsp[e] = a.p.v_scale + from * kScales;
                }
            }
            load_words(t.k[n], kp);
            #pragma unroll
            for (int e = 0; e < 4; ++e) {
                if constexpr (Tile<KIND, D>::kVBytes == 2) t.v[4 * n + e][0] = *reinterpret_cast<const uint16_t*>(vp[e]);
                else load_words(t.v[4 * n + e], vp[e]);
            }
            if constexpr (kScales > 0) {
                t.ks[n] = ksp[kScales * g / 4];
                #pragma unroll
                for (int e = 0; e < 4; ++e) t.vs[4 * n + e] = vsp[e][kScales * i / 16];
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

    auto multiply = [&](const Tile<KIND, D>& t, int v) {
        const int j0 = tile_at(tiles, v) * kKeys;
        floatx4 s[2];
        #pragma unroll
        for (int n = 0; n < 2; ++n) {
            s[n] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
            #pragma unroll
            for (int j = 0; j < kOps; ++j)
                s[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(key_operand<KIND>(t.k[n], j, t.ks[n]), q[j], s[n], 0, 0, 0);
        }
        bool masked = !all_seen(j0, kKeys, p_lo, p_hi, a.p.cap, a.window, a.sinks);
        if constexpr (PAGES16) masked |= t.bad[0] || t.bad[1];
        else masked |= __any(t.absent);
        uint32_t there[4];                         // halves of keys that are in the cache at all
        if (masked) {
            #pragma unroll
            for (int n = 0; n < 2; ++n) {
                #pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int j = j0 + 16 * n + 4 * g + r, e = 4 * n + r;
                    const bool have = j < tiles.end && !(PAGES16 ? t.bad[n] : (t.absent >> e & 1) != 0);
                    if (!have || !sees(my_pos, j, a.window, a.sinks)) s[n][r] = kNone;
                    const uint32_t half = have ? 0xffffu << (16 * (e & 1)) : 0u;
                    there[e / 2] = e & 1 ? there[e / 2] | half : half;
                }
            }
        }
        float top = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])), fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
        top = top * scale_log2 - kHead;
        if (__any(top > base + kSlack)) {
            top = fmaxf(base, max_of_groups(top));
            const float alpha = __builtin_amdgcn_exp2f(base - top);
            l *= alpha;
            #pragma unroll
            for (int m = 0; m < kOuts; ++m) acc[m] *= alpha;
            base = top;
        }
        float w[8];
        #pragma unroll
        for (int e = 0; e < 8; ++e) w[e] = __builtin_amdgcn_exp2f(fmaf(s[e / 4][e % 4], scale_log2, -base));
        const half8 pb = __builtin_bit_cast(half8, u32x4{pack2(w[0], w[1]), pack2(w[2], w[3]), pack2(w[4], w[5]), pack2(w[6], w[7])});
        l = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, pb, l, 0, 0, 0);
        if (!masked) {
            #pragma unroll
            for (int m = 0; m < kOuts; ++m)
                acc[m] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                    __builtin_bit_cast(half8, u32x4{value_pair(t, 0, m), value_pair(t, 1, m), value_pair(t, 2, m), value_pair(t, 3, m)}),
                    pb, acc[m], 0, 0, 0);
            return;
        }
        // A masked key has weight 0, but 0 x inf and 0 x NaN are NaN.  What is not in the cache is taken as 0; where there is
        // anything else that is not finite, the tile is multiplied once per query, with what that query does not see as zeros, and
        // the query's column kept.
        auto product = [&](int m, const uint32_t (&mask)[4]) {
            u32x4 x;
            #pragma unroll
            for (int p = 0; p < 4; ++p) x[p] = value_pair(t, p, m) & mask[p];
            return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, x), pb, acc[m], 0, 0, 0);
        };
        if (!__any(odd_values(t, there))) {
            #pragma unroll
            for (int m = 0; m < kOuts; ++m) acc[m] = product(m, there);
            return;
        }
        #pragma unroll 1
        for (int z = 0; z < kRows; ++z) {
            const int pos = __builtin_amdgcn_readlane(my_pos, z);
            uint32_t mask[4];
            #pragma unroll
            for (int e = 0; e < 8; ++e) {
                const bool see = sees(pos, j0 + 16 * (e / 4) + 4 * g + e % 4, a.window, a.sinks);
                const uint32_t half = see ? there[e / 2] & (0xffffu << (16 * (e & 1))) : 0u;
                mask[e / 2] = e & 1 ? mask[e / 2] | half : half;
            }
            #pragma unroll
            for (int m = 0; m < kOuts; ++m) {
                const floatx4 mine = product(m, mask);
                if (i == z) acc[m] = mine;
            }
        }
    };

    // One tile on its way while the one before it is multiplied (past the last: that one again, from the cache).
    if (first + wave < last) {
        Tile<KIND, D> x, z;
        int v = first + wave;
        fetch(x, v);
        for (;;) {
            fetch(z, v + kWaves < last ? v + kWaves : v);
            multiply(x, v);
            v += kWaves;
            if (v >= last) break;
            fetch(x, v + kWaves < last ? v + kWaves : v);
            multiply(z, v);
            v += kWaves;
            if (v >= last) break;
        }
    }

    // The wavefronts' sums meet in LDS; wavefront w goes on with register w of every output, that is with elements
    // (4 g + w) D / 16 .. of query i.
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
    float sum = 0.0f, o[kOuts];
    #pragma unroll
    for (int m = 0; m < kOuts; ++m) o[m] = 0.0f;
    #pragma unroll
    for (int z = 0; z < kWaves; ++z) {
        const float f = __builtin_amdgcn_exp2f(meet[z][0][lane] - top);
        sum += meet[z][1][lane] * f;
        #pragma unroll
        for (int m = 0; m < kOuts; ++m) o[m] += meet[z][2 + m * 4 + wave][lane] * f;
    }

    if (parts > 1) {
        // The parts of a set meet in memory, at agent scope, which passes the XCDs' own L2s; the block that arrives last adds them up,
        // in their order.  No block waits for another.  The counter is 0 between launches.
        constexpr int kSlot = slot_floats(D) / 2;                    // pairs of floats
        auto* const slot = reinterpret_cast<uint64_t*>(sums) + static_cast<int64_t>(blockIdx.x) * kSlot;
        if (live) {
            #pragma unroll
            for (int m = 0; m < kOuts; m += 2)
                __hip_atomic_store(slot + m / 2 * 256 + tid, __builtin_bit_cast(uint64_t, floatx2{o[m], o[m + 1]}), __ATOMIC_RELAXED,
                                   __HIP_MEMORY_SCOPE_AGENT);
            if (wave == 0 && g == 0)
                __hip_atomic_store(slot + kOuts / 2 * 256 + i, __builtin_bit_cast(uint64_t, floatx2{top, sum}), __ATOMIC_RELAXED,
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
        #pragma unroll 4
        for (int z = 0; z < parts; ++z) top = fmaxf(top, pair_at(z, kOuts / 2 * 256 + col)[0]);
        sum = 0.0f;
        #pragma unroll
        for (int m = 0; m < kOuts; ++m) o[m] = 0.0f;
        const int at = live ? tid : tid & ~15;
        #pragma unroll 4
        for (int z = 0; z < parts; ++z) {
            const floatx2 bl = pair_at(z, kOuts / 2 * 256 + col);
            const float f = __builtin_amdgcn_exp2f(bl[0] - top);
            sum += bl[1] * f;
            #pragma unroll
            for (int m = 0; m < kOuts; m += 2) {
                const floatx2 x = pair_at(z, m / 2 * 256 + at);
                o[m] += x[0] * f;
                o[m + 1] += x[1] * f;
            }
        }
    }
    if (!live) return;
    const float inv = sum == 0.0f ? 0.0f : __fdiv_rn(1.0f, sum);
    uint16_t* const dst = a.out + (it.s.first + token) * a.ld_out + head * D + (4 * g + wave) * kOuts;
    uint32_t h[kOuts / 2];
    #pragma unroll
    for (int m = 0; m < kOuts; m += 2) h[m / 2] = pack2(o[m] * inv, o[m + 1] * inv);
    if (reinterpret_cast<uintptr_t>(dst) % (2 * kOuts) == 0) {
        if constexpr (kOuts == 8) *reinterpret_cast<u32x4*>(dst) = u32x4{h[0], h[1], h[2], h[3]};
        else *reinterpret_cast<u32x2*>(dst) = u32x2{h[0], h[1]};
    } else {
        #pragma unroll
        for (int m = 0; m < kOuts; ++m) dst[m] = static_cast<uint16_t>(h[m / 2] >> (16 * (m & 1)));
    }
}

template <int KIND, int D>
bool launch_step(hipStream_t s, const AttentionArgs& a, void* workspace) {
    Plan plan{};
    plan.nrep = a.n_heads / a.p.n_kv_heads;
    plan.rep = make_divider(plan.nrep);
    plan.least = 8;
    // Sets of 16 rows: at most one more per sequence than full ones.
    const int64_t rows = static_cast<int64_t>(a.p.n_tokens) * plan.nrep, seqs = a.p.n_seqs < a.p.n_tokens ? a.p.n_seqs : a.p.n_tokens;
    const int64_t sets = (rows - seqs) / kRows + seqs;
    // Items beside one per set: as many blocks as the chip holds.
    const int64_t slots = workspace ? static_cast<int64_t>(kWorkspaceBytes / (slot_floats(D) * sizeof(float))) : 0;
    int64_t blocks = sets * a.p.n_kv_heads;
    const int64_t want = 4 * device_info().cus, room = (slots < kSliceCounters ? slots : kSliceCounters) - blocks;
    const int64_t target = (want < room ? want : room) / a.p.n_kv_heads;
    plan.target = target > 0 ? static_cast<int>(target) : 0;
    blocks += static_cast<int64_t>(plan.target) * a.p.n_kv_heads;
    const dim3 grid(static_cast<unsigned>(blocks)), block(64 * kWaves);
    auto go = [&](auto kern) {
        hipLaunchKernelGGL(kern, grid, block, 0, s, a, plan, static_cast<float*>(workspace), workspace ? slice_counters(workspace) : nullptr);
    };
    if (a.p.page.d % 16 == 0) go(paged_step_kernel<KIND, D, true>);
    else go(paged_step_kernel<KIND, D, false>);
    return MI_HIP_OK(hipGetLastError());
}

}  // namespace

bool launch_paged_attention(hipStream_t s, const AttentionArgs& a, void* workspace) {
    const bool wide = a.head_dim == 128;
    if (a.kind == MI_KV_F16) return wide ? launch_step<MI_KV_F16, 128>(s, a, workspace) : launch_step<MI_KV_F16, 64>(s, a, workspace);
    if (a.kind == MI_KV_INT8) return wide ? launch_step<MI_KV_INT8, 128>(s, a, workspace) : launch_step<MI_KV_INT8, 64>(s, a, workspace);
    return wide ? launch_step<MI_KV_Q4, 128>(s, a, workspace) : launch_step<MI_KV_Q4, 64>(s, a, workspace);
}

}  // namespace mi
