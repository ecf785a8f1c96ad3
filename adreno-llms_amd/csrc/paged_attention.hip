// Attention of many sequences' new tokens over a cache in pages (mi_attention): out = sum_j w_j v_j / sum_j w_j over the
// positions j that a row sees, w_j = exp(scale q k_j - their maximum), per query head.
//
// The query heads that share a key/value head are rows of one matrix, token by token (row t * nrep + head), so that a key
// is fetched once for all of them: 16 rows are one operand of v_mfma_f32_16x16x32_f16.  Scores are computed transposed (A = keys,
// B = queries): lane (query i = lane % 16, group g = lane / 16) then holds keys 4 g .. 4 g + 3 of every 16 for its query, and
// two such quadruples are, as they stand, the B operand of the product with the values, whichever keys they are, as long as
// the A operand (values transposed) brings the same.  Probabilities never leave the registers.
#include "paged_chunk.h"

namespace mi {
namespace {

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

template <int KIND, int D>
bool launch_step(hipStream_t s, const AttentionArgs& a, const PartRoom& room, const PagedLaunch& l) {
    auto go = [&](auto kern) {
        hipLaunchKernelGGL(kern, dim3(static_cast<unsigned>(l.blocks)), dim3(l.threads), 0, s, a, l.plan, room.sums, room.counters);
    };
    if (a.p.page.d % 16 == 0) go(paged_step_kernel<KIND, D, true>);
    else go(paged_step_kernel<KIND, D, false>);
    return MI_HIP_OK(hipGetLastError());
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
