// Attention of drafted tokens over a cache in pages (mi_attention_tree): the earlier positions are seen by the row's place in its text, the
// drafts by a bit for each.
//
// A sequence has a few dozen to a few hundred rows here (drafts times the query heads of a group) before thousands of keys: too
// many to fetch and convert the keys again for every 16 of them, too few for blocks of 128 rows to fill the chip.  So a
// wavefront streams its tiles of 32 keys from memory to the operands of the matrix instructions, without LDS or barriers as the kernel
// for few rows of a plain batch does, and multiplies each of them with SETS times 16 rows.
//
// What bounds it: launch, planning, queries and the meeting of parts, about 7 us whatever the lengths (16 drafts of 14 heads over 2 behind 900: 7.0);
// beyond, the vector units and the wait for memory.  With two sets in int8 a tile that all rows see is 194 vector instructions, 16 of them
// exponentials, 100 scalar ones and 16 matrix products; a launch has 273 and 159 for each tile, planning, queries, masks and sums counted in.  Counters
// of 32 trees of 24 drafts behind 4096, int8, 22.5 us: vector units busy 54 % of the SIMD-cycles, matrix cores 11 %; of the wavefronts' time, 2.3 to
// a SIMD, 40 % are instructions, 34 % waits for memory (a tile's keys are asked for behind the last one's key products, its values
// behind its value products) and 26 % for their turn.  13 of 100 in a window of 1024, Q4, pages of 48, 20.2 us: 54 %, 8 %; 2.5 to a SIMD, 36, 40 and 24 %.
#include "paged_tiles.h"

namespace mi {
namespace {

// The sum of a lane's value and those of the lanes 16, 32 and 48 away.
__device__ __forceinline__ float sum_of_groups(float a) {
    unsigned u = __float_as_uint(a);
    auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    u = __float_as_uint(__uint_as_float(r[0]) + __uint_as_float(r[1]));
    r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

constexpr int tree_lds(int D, int SETS) { return kWaves * SETS * (D / 4 + 2) * 64 * 4; }
// Blocks to a compute unit that the registers have to do for.  Two sets of width 64 in pages of whole sixteens: three, with 11 registers
// spilled in fp16 (32 trees of 24 drafts behind 4096 positions 25.6 us, with two 28.8; int8 and Q4 spill none), else two; of width 128
// one (264 to 320 registers, no spills, but 48 bytes of scratch memory: the division by nrep in the end is a call there, which takes the plan by its address).
constexpr int tree_blocks(int KIND, int D, bool PAGES16, int SETS) {
    if (D == 128) return SETS == 1 ? 2 : 1;
    return SETS == 2 ? PAGES16 ? 3 : 2 : KIND == MI_KV_F16 && !PAGES16 ? 3 : 4;
}

template <int KIND, int D, bool PAGES16, int SETS>
__global__ __launch_bounds__(64 * kWaves, tree_blocks(KIND, D, PAGES16, SETS)) void paged_tree_kernel(
    const TreeArgs a, const Plan plan, float* __restrict__ sums, uint32_t* __restrict__ counters) {
    constexpr int kOps = D / 32, kOuts = D / 16;   // operands of a key, of the values
    constexpr int kRow = row_bytes(KIND, D), kScales = row_scales(KIND, D);
    constexpr int kPiece = kRow >= 64 ? 16 : 8, kElems = kPiece * D / kRow;       // of a key: bytes, elements
    extern __shared__ __attribute__((aligned(16))) float meet[];                  // [kWaves][SETS][4 kOuts + 2][64]
    __shared__ uint32_t arrived;
    const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
    const int i = lane & 15, g = lane >> 4;
    const Item it = item_of<kRows * SETS, kKeys, false, true, D == 64 ? 0 : SETS == 1 ? 2 : 1>(a, plan, blockIdx.x / a.p.n_kv_heads);
    if (it.b < 0) return;
    const int kvh = it.kvh;
    const int rows = it.s.n * plan.nrep, r0 = it.set * (kRows * SETS), r_end = r0 + kRows * SETS < rows ? r0 + kRows * SETS : rows;
    const int base_pos = it.s.pos, p_hi = it.s.pos + (it.s.n - 1);                // of the first draft, of the last
    const Tiles tiles = tiles_of(base_pos, p_hi, a.p.cap, a.window, a.sinks, kKeys);
    const int parts = tiles.count > 0 ? (tiles.count - 1) / it.share + 1 : 1;
    if (it.chunk >= parts) return;
    const int first = parts == 1 ? 0 : it.chunk * it.share;
    const int last = tiles.count - first < it.share ? tiles.count : first + it.share;
    // the lane's queries (past the last: that one, not stored)
    auto row_of = [&](int u) { return r0 + kRows * u + i < r_end ? r0 + kRows * u + i : r_end - 1; };
    half8 q[SETS][kOps];
    int before[SETS], tokens[SETS];                // the window's far end, before the first position where there is none
    #pragma unroll
    for (int u = 0; u < SETS; ++u) {
        const int row = row_of(u), token = divide(row, plan.rep), head = kvh * plan.nrep + (row - token * plan.nrep);
        tokens[u] = token;
        before[u] = -1;
        if (a.window > 0) {
            const int mine = position_of(a, it.s, token);
            if (mine >= 0) before[u] = mine - a.window;
        }
        const uint16_t* src = a.q + (it.s.first + token) * a.ld_q + head * D + g * kElems;
        const bool wide = reinterpret_cast<uintptr_t>(src) % 16 == 0;
        #pragma unroll
        for (int j = 0; j < kOps; ++j) {
            constexpr int kPer = kElems / 8;       // operands of a piece
            const uint16_t* at = src + j / kPer * (4 * kElems) + 8 * (j % kPer);
            half8 x;
            if (wide) x = *reinterpret_cast<const half8*>(at);
            else
                #pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = __builtin_bit_cast(_Float16, at[e]);
            q[u][j] = KIND == MI_KV_Q4 ? __builtin_shufflevector(x, x, 0, 4, 1, 5, 2, 6, 3, 7) : x;
        }
    }
    const int sinks = a.window > 0 ? a.sinks : 0;

    // ---- a tile's pages and loads, as in paged_step_kernel
    const auto* const table = reinterpret_cast<const __attribute__((address_space(4))) int*>(
        reinterpret_cast<uintptr_t>(a.p.pages + static_cast<int64_t>(it.b) * a.p.max_pages));
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
    const uint32_t k_off = i * kRow + g * kPiece, v_off = 4 * g * kRow + i * (kRow / 16);
    const uint32_t ks_off = (i * kScales + kScales * g / 4) * 2, vs_off = 4 * g * kScales * 2;
    struct Rows {
        int64_t at[2];
        uint32_t absent;
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

    floatx4 acc[SETS][kOuts];
    float l[SETS];                                 // sums of the lane's weights, as they meet the values
    float base[SETS];                              // see kHead
    const floatx4 none = {0.0f, 0.0f, 0.0f, 0.0f};
    #pragma unroll
    for (int u = 0; u < SETS; ++u) {
        #pragma unroll
        for (int m = 0; m < kOuts; ++m) acc[u][m] = none;
        l[u] = 0.0f;
        base[u] = kStart;
    }
    const float scale_log2 = a.scale * 1.44269504088896341f;
    bool far = false;                              // some query's base is beyond kFar

    // Tile v, whose rows are `r`; `more`: the keys and values of the wavefront's next tile, at `next`, are asked for as soon as the
    // registers of this one's are free.
    auto multiply = [&](int v, const Rows& r, auto more, const Rows& next) {
        const int j0 = tile_at(tiles, v) * kKeys;
        floatx4 s[SETS][2];
        #pragma unroll
        for (int n = 0; n < 2; ++n) {
            #pragma unroll
            for (int u = 0; u < SETS; ++u) s[u][n] = none;
            #pragma unroll
            for (int j = 0; j < kOps; ++j) {
                const half8 key = key_operand<KIND>(t.k[n], j, t.ks[n], exponent);
                #pragma unroll
                for (int u = 0; u < SETS; ++u) s[u][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(key, q[u][j], s[u][n], 0, 0, 0);
            }
        }
        if constexpr (more.value) load_keys(next);
        __builtin_amdgcn_sched_barrier(0);
        bool masked = !all_seen(j0, kKeys, base_pos - 1, p_hi, a.p.cap, a.window, a.sinks);
        masked |= PAGES16 ? r.absent != 0 : __any(r.absent);
        uint32_t there[4] = {};                    // halves of keys that are in the cache at all
        if (__builtin_expect(masked, 0)) {
            asm volatile("");                      // (a branch: most tiles are not)
            uint32_t have = 0;                     // bit e: key e of the lane's values
            #pragma unroll
            for (int e = 0; e < 8; ++e) {
                const bool in = (j0 + 16 * (e / 4) + 4 * g + e % 4 < tiles.end) & ((r.absent >> e & 1) == 0);
                have |= in ? 1u << e : 0u;
                there[e / 2] |= in ? 0xffffu << (16 * (e & 1)) : 0u;
            }
            #pragma unroll
            for (int u = 0; u < SETS; ++u) {
                const uint32_t drafts = j0 + (kKeys - 1) < base_pos ? 0u : drafts_seen(a, it.s, tokens[u], j0) >> (4 * g);
                #pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int at = 16 * (e / 4) + e % 4, j = j0 + at + 4 * g;
                    const bool see = j < base_pos ? (j > before[u]) | (j < sinks) : (drafts >> at & 1) != 0;
                    s[u][e / 4][e % 4] = (see & ((have >> e & 1) != 0)) ? s[u][e / 4][e % 4] : kNone;
                }
            }
        }
        float top[SETS];
        bool higher = false;
        #pragma unroll
        for (int u = 0; u < SETS; ++u) {
            top[u] = max3(max3(s[u][0][0], s[u][0][1], s[u][0][2]), max3(s[u][0][3], s[u][1][0], s[u][1][1]), max3(s[u][1][2], s[u][1][3], s[u][1][3]));
            higher |= top[u] * scale_log2 - kHead > base[u] + kSlack;
        }
        if (__builtin_expect(__any(higher), 0)) {
            far = false;
            #pragma unroll
            for (int u = 0; u < SETS; ++u) {
                const float now = fmaxf(base[u], max_of_groups(base_of(top[u], scale_log2)));
                const float alpha = __builtin_amdgcn_exp2f(base[u] - now);
                l[u] *= alpha;
                #pragma unroll
                for (int m = 0; m < kOuts; ++m) acc[u][m] *= alpha;
                base[u] = now;
                far |= __any(fabsf(now) >= kFar && now > kStart) != 0;
            }
        }
        half8 pb[SETS];
        #pragma unroll
        for (int u = 0; u < SETS; ++u) {
            float by = scale_log2, from = base[u];
            if (__builtin_expect(far, 0)) {
                asm volatile("");
                #pragma unroll
                for (int e = 0; e < 8; ++e) s[u][e / 4][e % 4] = far_exponent(s[u][e / 4][e % 4], scale_log2, base[u]);
                by = 1.0f;
                from = 0.0f;
            }
            float w[8];
            #pragma unroll
            for (int e = 0; e < 8; ++e) w[e] = __builtin_amdgcn_exp2f(fmaf(s[u][e / 4][e % 4], by, -from));
            const uint32_t two[4] = {pack2(w[0], w[1]), pack2(w[2], w[3]), pack2(w[4], w[5]), pack2(w[6], w[7])};
            const half2v ones = {static_cast<_Float16>(1.0f), static_cast<_Float16>(1.0f)};
            #pragma unroll
            for (int e = 0; e < 4; ++e) l[u] = __builtin_amdgcn_fdot2(__builtin_bit_cast(half2v, two[e]), ones, l[u], false);
            pb[u] = __builtin_bit_cast(half8, u32x4{two[0], two[1], two[2], two[3]});
            __builtin_amdgcn_sched_barrier(0);
        }
        pack_scales(t, i);
        if (!masked) {
            #pragma unroll
            for (int m = 0; m < kOuts; ++m) {
                const half8 value = __builtin_bit_cast(half8, u32x4{value_pair(t, 0, m, exponent), value_pair(t, 1, m, exponent),
                                                                    value_pair(t, 2, m, exponent), value_pair(t, 3, m, exponent)});
                #pragma unroll
                for (int u = 0; u < SETS; ++u) acc[u][m] = __builtin_amdgcn_mfma_f32_16x16x32_f16(value, pb[u], acc[u][m], 0, 0, 0);
            }
            if constexpr (more.value) load_values(next);
            return;
        }
        // What is not in the cache is taken as 0; for what is and is not finite see odd_part.
        auto operand = [&](int m, auto change) {
            u32x4 x;
            #pragma unroll
            for (int p = 0; p < 4; ++p) x[p] = change(value_pair(t, p, m, exponent) & there[p]);
            return __builtin_bit_cast(half8, x);
        };
        if (__builtin_expect(!__any(odd_values(t, there)), 1)) {
            #pragma unroll
            for (int m = 0; m < kOuts; ++m) {
                const half8 value = operand(m, [](uint32_t x) { return x; });
                #pragma unroll
                for (int u = 0; u < SETS; ++u) acc[u][m] = __builtin_amdgcn_mfma_f32_16x16x32_f16(value, pb[u], acc[u][m], 0, 0, 0);
            }
        } else {
            #pragma unroll
            for (int m = 0; m < kOuts; ++m)
                #pragma unroll 1
                for (int part = 0; part < 4; ++part) {
                    const half8 value = operand(m, [&](uint32_t x) { return odd_part(x, part); });
                    #pragma unroll
                    for (int u = 0; u < SETS; ++u) {
                        const floatx4 found = __builtin_amdgcn_mfma_f32_16x16x32_f16(value, pb[u], none, 0, 0, 0);
                        #pragma unroll
                        for (int e = 0; e < 4; ++e) acc[u][m][e] = with_odd(acc[u][m][e], found[e], part);
                    }
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

    // The wavefronts' sums meet in LDS.  Wavefront w goes on with set w % SETS, and of it with kMine registers: kMine elements from `element`
    // on of query i.
    constexpr int kBox = (4 * kOuts + 2) * 64, kMine = 4 * kOuts * SETS / kWaves, kRegs = kMine / kOuts ? kMine / kOuts : 1;
    static_assert(kWaves % SETS == 0 && kMine % kOuts == 0, "whole registers of all outputs");
    #pragma unroll
    for (int u = 0; u < SETS; ++u) {
        float* const mine = meet + (wave * SETS + u) * kBox + lane;
        mine[0] = base[u];
        mine[64] = sum_of_groups(l[u]);
        #pragma unroll
        for (int m = 0; m < kOuts; ++m)
            #pragma unroll
            for (int r = 0; r < 4; ++r) mine[(2 + m * 4 + r) * 64] = acc[u][m][r];
    }
    __syncthreads();
    const int set = wave % SETS, reg = wave / SETS * kRegs;            // registers reg .. reg + kRegs - 1 of all outputs
    const bool live = r0 + kRows * set + i < r_end;
    const float* const box = meet + set * kBox + lane;
    float high = box[0];
    #pragma unroll
    for (int z = 1; z < kWaves; ++z) high = fmaxf(high, box[z * SETS * kBox]);
    float sum = 0.0f, o[kRegs][kOuts];
    #pragma unroll
    for (int r = 0; r < kRegs; ++r)
        #pragma unroll
        for (int m = 0; m < kOuts; ++m) o[r][m] = 0.0f;
    #pragma unroll
    for (int z = 0; z < kWaves; ++z) {
        const float* const from = box + z * SETS * kBox;
        const float f = __builtin_amdgcn_exp2f(from[0] - high);
        sum += from[64] * f;
        #pragma unroll
        for (int r = 0; r < kRegs; ++r)
            #pragma unroll
            for (int m = 0; m < kOuts; ++m) o[r][m] += from[(2 + m * 4 + reg + r) * 64] * f;
    }

    if (parts > 1) {
        // The parts of a set meet in memory, at agent scope, which passes the XCDs' own L2s; the block that arrives last adds them up,
        // in their order.  No block waits for another.  The counter is 0 between launches.
        constexpr int kPairs = kMine / 2, kSlot = SETS * slot_floats(D) / 2;     // pairs of floats: of a lane, of a block
        auto* const slot = reinterpret_cast<uint64_t*>(sums) + static_cast<int64_t>(it.id) * kSlot;
        const int at_sum = kPairs * 64 * kWaves + set * 16 + i;
        if (live) {
            #pragma unroll
            for (int k = 0; k < kPairs; ++k)
                __hip_atomic_store(slot + k * (64 * kWaves) + tid, __builtin_bit_cast(uint64_t, floatx2{o[2 * k / kOuts][2 * k % kOuts], o[2 * k / kOuts][2 * k % kOuts + 1]}),
                                   __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            if (wave < SETS && g == 0)
                __hip_atomic_store(slot + at_sum, __builtin_bit_cast(uint64_t, floatx2{high, sum}), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        uint32_t* const counter = counters + (it.id - it.chunk * a.p.n_kv_heads);
        if (tid == 0) arrived = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __syncthreads();
        if (uniform(arrived) + 1 != static_cast<uint32_t>(parts)) return;
        asm volatile("" ::: "memory");
        if (tid == 0) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        const uint64_t* const slots = reinterpret_cast<const uint64_t*>(sums) + static_cast<int64_t>(it.id - it.chunk * a.p.n_kv_heads) * kSlot;
        const int64_t next = static_cast<int64_t>(a.p.n_kv_heads) * kSlot;
        auto pair_at = [&](int part, int at) {
            return __builtin_bit_cast(floatx2, __hip_atomic_load(slots + part * next + at, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
        };
        high = kStart;
        sum = 0.0f;
        #pragma unroll
        for (int r = 0; r < kRegs; ++r)
            #pragma unroll
            for (int m = 0; m < kOuts; ++m) o[r][m] = 0.0f;
        const int at = live ? tid : tid & ~15, col = live ? at_sum : at_sum - i;
        constexpr int kAhead = kPairs <= 4 ? 8 : kPairs <= 8 ? 6 : 4;              // parts asked for together
        #pragma unroll 1
        for (int z0 = 0; z0 < parts; z0 += kAhead) {
            floatx2 bl[kAhead], x[kAhead][kPairs];
            #pragma unroll
            for (int z = 0; z < kAhead; ++z) {
                const int part = z0 + z < parts ? z0 + z : parts - 1;
                bl[z] = pair_at(part, col);
                #pragma unroll
                for (int k = 0; k < kPairs; ++k) x[z][k] = pair_at(part, k * (64 * kWaves) + at);
            }
            #pragma unroll
            for (int z = 0; z < kAhead; ++z) {
                if (z0 + z >= parts) break;
                const float now = fmaxf(high, bl[z][0]), was = __builtin_amdgcn_exp2f(high - now), f = __builtin_amdgcn_exp2f(bl[z][0] - now);
                high = now;
                sum = sum * was + bl[z][1] * f;
                #pragma unroll
                for (int k = 0; k < kMine; ++k) o[k / kOuts][k % kOuts] = o[k / kOuts][k % kOuts] * was + x[z][k / 2][k & 1] * f;
            }
        }
    }
    if (!live) return;
    const float inv = __fdiv_rn(1.0f, sum);        // (not used where the sum is 0)
    const int row = row_of(set), token = divide(row, plan.rep), head = kvh * plan.nrep + (row - token * plan.nrep);
    uint16_t* const dst = a.out + (it.s.first + token) * a.ld_out + head * D + (4 * g + reg) * kOuts;
    const bool wide = reinterpret_cast<uintptr_t>(dst) % (2 * kOuts) == 0;
    #pragma unroll
    for (int r = 0; r < kRegs; ++r) {
        uint32_t h[kOuts / 2];
        #pragma unroll
        for (int m = 0; m < kOuts; m += 2) h[m / 2] = sum == 0.0f ? 0u : pack2(o[r][m] * inv, o[r][m + 1] * inv);      // (o may be NaN)
        uint16_t* const to = dst + r * kOuts;
        if (wide) {
            if constexpr (kOuts == 8) *reinterpret_cast<u32x4*>(to) = u32x4{h[0], h[1], h[2], h[3]};
            else *reinterpret_cast<u32x2*>(to) = u32x2{h[0], h[1]};
        } else {
            #pragma unroll
            for (int m = 0; m < kOuts; ++m) to[m] = static_cast<uint16_t>(h[m / 2] >> (16 * (m & 1)));
        }
    }
}

template <int KIND, int D, int SETS>
bool launch(hipStream_t s, const TreeArgs& a, float* sums, uint32_t* counters, const PagedLaunch& l) {
    constexpr int lds = tree_lds(D, SETS);
    static_assert(lds <= 160 * 1024 - 64, "sums fit");
    auto go = [&](auto pages16) {                  // (a type of its own for each, so that each has its attribute set once)
        const auto kern = paged_tree_kernel<KIND, D, decltype(pages16)::value, SETS>;
        if (lds > 65536 - 64 && !MI_ONCE_OK(MI_HIP_OK(hipFuncSetAttribute(reinterpret_cast<const void*>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, lds))))
            return false;
        hipLaunchKernelGGL(kern, dim3(static_cast<unsigned>(l.blocks)), dim3(l.threads), lds, s, a, l.plan, sums, counters);
        return MI_HIP_OK(hipGetLastError());
    };
    return a.p.page.d % 16 == 0 ? go(std::true_type{}) : go(std::false_type{});
}
template <int KIND, int D>
bool launch_sets(hipStream_t s, const TreeArgs& a, float* sums, uint32_t* counters, const PagedLaunch& l) {
    return l.sets == 1 ? launch<KIND, D, 1>(s, a, sums, counters, l) : launch<KIND, D, 2>(s, a, sums, counters, l);
}

}  // namespace

bool launch_paged_tree(hipStream_t s, const TreeArgs& a, const StreamRoom& own) {
    const bool room = own.workspace && own.sums;
    const AttentionSize size = {a.p.n_seqs, a.p.n_tokens, a.max_tokens, a.p.cap, a.n_heads, a.p.n_kv_heads, a.head_dim, a.window, a.sinks,
                                a.kind == MI_KV_F16};
    PagedLaunches all;
    all.n = 1;
    const PagedLaunch& l = all.of[0] = tree_launch(size, room ? Room{kPartialBytes, kSliceCounters} : Room{}, device_info().cus);
    if (const int64_t blocks = too_many_blocks(all)) {
        MI_ERROR_FMT("mi_attention_tree: %lld blocks are more than a launch counts", static_cast<long long>(blocks));
        return false;
    }
    auto* const sums = room ? static_cast<float*>(own.sums) : nullptr;
    uint32_t* const counters = room ? slice_counters(own.workspace) : nullptr;
    if (l.wavefronts) return launch_paged_tree_many(s, a, sums, counters, l);
    const bool wide = a.head_dim == 128;
    return a.kind == MI_KV_F16    ? wide ? launch_sets<MI_KV_F16, 128>(s, a, sums, counters, l) : launch_sets<MI_KV_F16, 64>(s, a, sums, counters, l)
           : a.kind == MI_KV_INT8 ? wide ? launch_sets<MI_KV_INT8, 128>(s, a, sums, counters, l) : launch_sets<MI_KV_INT8, 64>(s, a, sums, counters, l)
                                  : wide ? launch_sets<MI_KV_Q4, 128>(s, a, sums, counters, l) : launch_sets<MI_KV_Q4, 64>(s, a, sums, counters, l);
}

}  // namespace mi
