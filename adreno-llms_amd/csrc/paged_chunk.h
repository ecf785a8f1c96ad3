// The kernel for many rows of attention over a cache in pages: of plain batches (paged_attention.hip) and of trees (paged_tree_many.hip).
#pragma once
#include "paged_tiles.h"

namespace mi {
namespace {

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
__device__ const __attribute__((aligned(16))) uint32_t kNothing[4] = {0, 0, 0, 0};
// 16 bytes from each lane's place in memory to LDS, the lanes' side by side from `to` on (which is the wavefront's).
__device__ __forceinline__ void lds_fill(const uint8_t* from, uint8_t* to) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) uint8_t*)from, (__attribute__((address_space(3))) uint8_t*)to, 16, 0, 0);
}
__device__ __forceinline__ constexpr int twist(int row) { return (row & 3) * 2 + (row >> 2 & 1); }

// Dear: a row takes its keys one to a lane and its values one after the other.  A prompt of 2048 rows of 14 heads over 2 with one NaN among
// the values of a head's first, middle and last position 0.5, 3.2 and 5.5 ms instead of 0.03, 4096 rows of 32 over 8 0.8, 26 and 50 ms
// instead of 0.23 (single launches).
//
// Row `q` (fp16) of token `token` of a sequence against tiles first .. last - 1, one key to a lane: where an infinity or a
// NaN in a place that some row must not see keeps the row off the matrix cores.  Leaves elements lane, lane + 64, .. of the sum of the
// weighted values, and the sums' base.
template <int KIND, int D, class Args>
__device__ __forceinline__ void row_by_itself(const Args& a, const Span& span, int token, const int* table, const Tiles& tiles, int first, int last, int kvh,
                                              const uint16_t* q, float (&o)[D / 64], float& base, float& sum) {
    const int lane = threadIdx.x & 63, pos = position_of(a, span, token);
    base = kStart;
    sum = 0.0f;
    for (int d = 0; d < D / 64; ++d) o[d] = 0.0f;
    #pragma unroll 1
    for (int v = first; v < last; ++v) {
        const int j = tile_at(tiles, v) * 64 + lane;
        int lo = 0, hi = -1;                       // the key's row, in two halves; none
        float score = kNone;
        bool see;
        if constexpr (is_tree<Args>) see = j < span.pos ? sees(pos, j, a.window, a.sinks) : (drafts_seen(a, span, token, j) & 1) != 0;
        else see = pos >= 0 && sees(pos, j, a.window, a.sinks);
        if (j < tiles.end && see) {
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

template <int KIND, int D, bool PAGES16, int RW, int KS, class Args>
__global__ __launch_bounds__(64 * RW * KS, is_tree<Args> && D == 64 ? 3 : 2) void paged_chunk_kernel(const Args a, const Plan plan, float* __restrict__ partial,
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
    const Item it = item_of<kChunkRows, kChunkKeys, is_tree<Args>>(a, plan, y);
    if (it.b < 0) return;
    const int rows = it.s.n * plan.nrep, r0 = it.set * kChunkRows, r_end = r0 + kChunkRows < rows ? r0 + kChunkRows : rows;
    constexpr bool kTree = is_tree<Args>;          // (a tree's rows lie anywhere among its positions)
    const int tree_end = it.s.pos + (it.s.n - 1);
    const Tiles tiles = tiles_of(kTree ? it.s.pos : it.s.pos + divide(r0, plan.rep), kTree ? tree_end : it.s.pos + divide(r_end - 1, plan.rep), a.p.cap, a.window,
                                 a.sinks, kChunkKeys);
    const int parts = tiles.count > 0 ? (tiles.count - 1) / it.share + 1 : 1;
    if (it.chunk >= parts) return;
    const int first = parts == 1 ? 0 : it.chunk * it.share;
    const int last = tiles.count - first < it.share ? tiles.count : first + it.share;
    // the wavefront's rows and the lane's query (past the last: that one, not stored)
    const int w0 = r0 + 32 * wave < r_end ? r0 + 32 * wave : r_end - 1, w_end = w0 + 32 < r_end ? w0 + 32 : r_end;
    const bool busy = r0 + 32 * wave < r_end, live = r0 + 32 * wave + i < r_end;
    const int row = w0 + i < w_end ? w0 + i : w_end - 1, token = divide(row, plan.rep), head = kvh * plan.nrep + (row - token * plan.nrep);
    const int my_pos = position_of(a, it.s, token), p_lo = kTree ? it.s.pos : it.s.pos + divide(w0, plan.rep);
    const int p_hi = kTree ? tree_end : it.s.pos + divide(w_end - 1, plan.rep);
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
    // A tree's tile in fp16 goes from its pages to LDS by itself, a row's piece p ^ twist(row) to the place p (what is not in the cache from a
    // piece of zeros).
    auto fill = [&](int v, const Pages& g, int buf) {
        const int j0 = tile_at(tiles, v) * kChunkKeys;
        uint8_t* const kt = own_lds + buf * (chunk_lds(D) / 2) + wave * 1024;
        #pragma unroll
        for (int p = 0; p < kLoads; ++p) {
            const int j = key_of(j0, p), number = g.number[p], row = p * kPer + my_row;
            const bool bad = static_cast<uint32_t>(number) >= static_cast<uint32_t>(a.p.n_pages), none = bad || j0 + row >= tiles.end;
            int slot = j - divide(j, a.p.page) * a.p.page.d;
            if constexpr (PAGES16) slot &= ~15;
            const int64_t at = row_number(a.p, bad ? 0 : number, kvh, slot);
            const uint32_t off = (PAGES16 ? my_row & 15 : 0) * kRow + (my_piece ^ twist(my_row)) * kPiece;
            const uint8_t *kb = a.p.k + at * kRow + off, *vb = a.p.v + at * kRow + off;
            if (none) kb = vb = reinterpret_cast<const uint8_t*>(kNothing);
            lds_fill(kb, kt + p * kPer * (2 * D));
            lds_fill(vb, kt + p * kPer * (2 * D) + chunk_lds(D) / 4);
            if (my_piece == 0) gone[buf * kChunkKeys + row] = none;
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
        // (a tree's wavefront goes first while it feeds the matrix cores: 8 trees of 64 behind 16384 117 -> 112 us, int8 111 -> 102)
        if constexpr (kTree) __builtin_amdgcn_s_setprio(1);
        #pragma unroll
        for (int t = 0; t < 2; ++t) {
            #pragma unroll
            for (int r = 0; r < 16; ++r) s[t][r] = 0.0f;
            #pragma unroll
            for (int j = 0; j < kOps; ++j)
                s[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(
                    *reinterpret_cast<const half8*>(kt + (32 * t + i) * (2 * D) + 16 * ((2 * j + h) ^ twist(i))), q[j], s[t], 0, 0, 0);
        }
        if constexpr (kTree) __builtin_amdgcn_s_setprio(0);
        const uint64_t absent = __ballot(gone[buf * kChunkKeys + lane] != 0);
        const bool masked = !all_seen(j0, kChunkKeys, kTree ? p_lo - 1 : p_lo, p_hi, a.p.cap, a.window, a.sinks) || absent != 0;
        if (__builtin_expect(masked, 0)) {
            asm volatile("");
            #pragma unroll
            for (int t = 0; t < 2; ++t) {
                uint32_t drafts = 0;
                if constexpr (kTree) {
                    if (j0 + 32 * t + 31 >= it.s.pos) drafts = drafts_seen(a, it.s, token, j0 + 32 * t) >> (4 * h);
                }
                #pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int j = j0 + 32 * t + 8 * (r / 4) + 4 * h + r % 4;
                    const uint32_t out = static_cast<uint32_t>(absent >> (32 * t)) >> (4 * h) >> (8 * (r / 4) + r % 4) & 1;
                    bool see;
                    if constexpr (kTree) see = (out == 0) & (j < it.s.pos ? (j > before) | (j < sinks) : (drafts >> (8 * (r / 4) + r % 4) & 1) != 0);
                    else see = (out == 0) & (j <= my_pos) & ((j > before) | (j < sinks));
                    s[t][r] = see ? s[t][r] : kNone;
                }
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
        if constexpr (kTree) __builtin_amdgcn_s_setprio(1);
        #pragma unroll
        for (int c = 0; c < 4; ++c)
            #pragma unroll
            for (int m = 0; m < kOuts; ++m)
                acc[m] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8, values(m, c)), weights(c), acc[m], 0, 0, 0);
        if constexpr (kTree) __builtin_amdgcn_s_setprio(0);
    };

    // registers -> LDS, the next tile requested, one barrier (a buffer is written again two barriers after it was last read),
    // the tile multiplied unless the wavefront's queries see nothing of it
    // (of KS slices: tiles first + slice, + KS, ..; past the last that one again, not multiplied)
    Pages pages;
    const int mine = first + slice;
    auto clamp = [&](int v) { return v < last ? v : last - 1; };
    constexpr bool kStraight = kTree && KIND == MI_KV_F16 && KS == 1;
    if (first < last) {
        pages = look_up(mine);
        if constexpr (kStraight) fill(mine, pages, 0);
        else fetch(clamp(mine), pages);
        pages = look_up(mine + KS);
    }
    for (int v = mine, buf = 0; v - slice < last; v += KS, buf ^= 1) {
        if constexpr (kStraight) {
            // (this tile is there, and the one before it done with, for all wavefronts)
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();
            if (v + 1 < last) {
                fill(v + 1, pages, buf ^ 1);
                pages = look_up(v + 2);
            }
        } else {
            stash(buf);
            if (v - slice + KS < last) {
                fetch(clamp(v + KS), pages);
                pages = look_up(v + 2 * KS);
            }
            __syncthreads();
        }
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
            row_by_itself<KIND, D>(a, it.s, t, a.p.pages + static_cast<int64_t>(it.b) * a.p.max_pages, tiles, first, last, kvh, a.q + (it.s.first + t) * a.ld_q + hd * D, o, b, l);
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
        constexpr int kAhead = kTree ? 2 : 1;      // parts asked for together
        #pragma unroll 1
        for (int z0 = 0; z0 < parts; z0 += kAhead) {
            floatx2 bl[kAhead], x[kAhead][kPairs];
            #pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                const int z = kAhead == 1 || z0 + u < parts ? z0 + u : parts - 1;
                bl[u] = pair_at(z, at_sum);
                #pragma unroll
                for (int k = 0; k < kPairs; ++k) x[u][k] = pair_at(z, at + k * 64);
            }
            #pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                if (kAhead > 1 && z0 + u >= parts) break;
                const float now = fmaxf(base, bl[u][0]), was = __builtin_amdgcn_exp2f(base - now), f = __builtin_amdgcn_exp2f(bl[u][0] - now);
                base = now;
                sum = sum * was + bl[u][1] * f;
                #pragma unroll
                for (int m = 0; m < kOuts; ++m)
                    #pragma unroll
                    for (int r = 0; r < 16; ++r) acc[m][r] = acc[m][r] * was + x[u][m * 8 + r / 2][r & 1] * f;
            }
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

template <int KIND, int D, int RW, int KS, class Args>
bool launch_chunk(hipStream_t s, const Args& a, const PartRoom& room, const PagedLaunch& l) {
    constexpr int lds = chunk_lds_all(D, KS);
    static_assert(lds <= 160 * 1024 && (KS - 1) * meet_floats(D, RW) * 4 <= KS * chunk_lds(D), "tiles and sums fit");
    auto go = [&](auto pages16) {                  // (a type of its own for each, so that each has its attribute set once)
        const auto kern = paged_chunk_kernel<KIND, D, decltype(pages16)::value, RW, KS, Args>;
        if (lds > 65536 && !MI_ONCE_OK(MI_HIP_OK(hipFuncSetAttribute(reinterpret_cast<const void*>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, lds))))
            return false;
        hipLaunchKernelGGL(kern, dim3(static_cast<unsigned>(l.blocks)), dim3(l.threads), lds, s, a, l.plan, room.sums, room.counters);
        return MI_HIP_OK(hipGetLastError());
    };
    return a.p.page.d % 16 == 0 ? go(std::true_type{}) : go(std::false_type{});
}

}  // namespace
}  // namespace mi
