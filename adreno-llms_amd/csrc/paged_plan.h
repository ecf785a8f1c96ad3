// Which kernels serve a call of mi_attention (paged_attention.hip) or mi_attention_tree (paged_tree.hip), with how many blocks, and how the keys of sequences are shared
// out to them: everything that follows from the numbers the host has, and from a sequence's lengths.  Plain C++ (constexpr makes
// device code as well).
#pragma once
#include "paged_rule.h"

#include <cstddef>

namespace mi {

// The kernel for few rows: sets of 16 rows, tiles of 32 keys, four wavefronts.  The one for many: 32 rows per wavefront, tiles of 64.
constexpr int kRows = 16, kKeys = 32, kWaves = 4;
constexpr int kChunkKeys = 64;
// Floats of a block's sums in the workspace, for width D (and RW wavefronts of 32 rows).
constexpr int slot_floats(int D) { return 16 * D + 32; }
constexpr int chunk_slot_floats(int D, int RW) { return 32 * RW * (D + 2); }

struct Plan {
    int target = 0;           // items per key/value head beside one per set; 0: keys are not split
    int least = 0;            // tiles of keys that a block is worth
    int from = 0, to = 0;     // sequences of that many rows (new tokens times nrep) are the launch's
    int nrep = 1;
    Divider rep;              // by nrep
};

// What a sequence is to a launch: sets of rows, and tiles of keys that each has at most.
struct Cost {
    int sets = 0, tiles = 0;
};
constexpr Cost cost_of(const Plan& plan, const Span& s, int cap, int window, int sinks, int rows_per_set, int keys) {
    if (s.n <= 0 || s.n * plan.nrep < plan.from || s.n * plan.nrep > plan.to) return {};
    const int count = tiles_of(s.pos, s.pos + s.n - 1, cap, window, sinks, keys).count;
    return {(s.n * plan.nrep + rows_per_set - 1) / rows_per_set, count > 0 ? count : 1};
}
// Tiles that a block takes, of `all` tiles of all sets.  (A hundred-thousandth more: the sum's rounding must not make an item too many.)
constexpr int share_of(float all, const Plan& plan) {
    if (plan.target <= 0) return 0x7fffffff;
    const float each = all * 1.00001f / static_cast<float>(plan.target);
    const int share = each < 1.0e9f ? static_cast<int>(each) + 1 : 0x7fffffff;
    return share < plan.least ? plan.least : share;
}

// Items of a sequence where a block takes `share` tiles; and the least share, down to half of `share`, with which all sequences' items
// (items(share), fewer the greater it is) are no more than `blocks`: `share` itself is known to fit.
constexpr int items_of(const Cost& c, int share) { return c.sets ? c.sets * ((c.tiles - 1) / share + 1) : 0; }
template <class Items>
constexpr int even_share(int share, int blocks, const Items& items) {
    int low = share / 2;                           // (not known to)
    while (share - low > 1) {
        const int mid = low + (share - low) / 2;
        if (items(mid) <= blocks) share = mid;
        else low = mid;
    }
    return share;
}

// The sets of a sequence read the same keys.  Blocks go to the eight XCDs in turn, each with an L2 of its own: so that a part of the keys of a
// key/value head (a pair) meets all its sets in one L2, they are eight blocks apart, one behind the other.  The sets and pairs of a sequence's blocks in
// their order, block `in`; pairs behind the last whole eight lie side by side.
// With the sets as far apart as a head has parts it is chance whether they share an XCD, and key/value heads that do not go into eight spread them over
// all; besides, they read their keys at other times.  us for few rows (paged_tree.hip), that way / eight apart: 32 trees of 24, 15 heads over 5, behind 4096, fp16
// 38.7 / 32.5; 8 of 16 behind 16384, 28 over 7, width 128 fp16 102 / 67, int8 61 / 50; one tree of 24 behind 16384, 12 over 6 25.6 / 18.0, 14 over 2 22.9 / 18.8,
// 32 over 8 22.0 / 19.5, width 128 47.2 / 47.5; 3 of 16 behind 9000, 32 over 8 23.2 / 19.3.  Over 576 cases of 1, 2, 4 and 8 key/value heads 0.82 to 1.07,
// on average 0.99 of the time.  For many rows (paged_tree_many.hip) nothing: 0.96 to 1.05.
struct SetOfPair {
    unsigned set, pair;
};
constexpr SetOfPair eight_apart(unsigned in, unsigned sets, unsigned pairs) {
    const unsigned group = 8 * sets, whole = pairs / 8 * group;
    if (in < whole) {
        const unsigned at = in / group, within = in - at * group;
        return {within / 8, at * 8 + within % 8};
    }
    const unsigned rest = pairs % 8, set = (in - whole) / rest;
    return {set, pairs / 8 * 8 + (in - whole - set * rest)};
}

// The least share with which all items are no more than `blocks`, which are not fewer than the sets: items(share), fewer the greater it is, are at most
// all / share + sets, and `most` leaves one per set.
template <class Items>
constexpr int fitting_share(float all, int sets, int blocks, int most, const Items& items) {
    const float least = all / static_cast<float>(blocks), enough = blocks > sets ? all * 1.00001f / static_cast<float>(blocks - sets) + 1.0f : 1.0e9f;
    int low = static_cast<int>(least * 0.99999f) - 1, share = enough < static_cast<float>(most) ? static_cast<int>(enough) : most;
    if (low < 0) low = 0;                          // (not known to fit)
    while (share - low > 1) {
        const int mid = low + (share - low) / 2;
        if (items(mid) <= blocks) share = mid;
        else low = mid;
    }
    return share;
}

// The share for a launch of which a compute unit holds r blocks, one or two, and whose target is so many: by `share`, what share_of says, the last round of blocks
// may be nearly empty.  Tried are the least shares that make one round and (r = 1) two, or (r = 2) one block for each unit; a tile's time is taken as
// 3 + j where a unit has j blocks, a block's start and end as 12 tiles.  `blocks`: per key/value head of the launch, which items must not exceed.
// us for few rows of width 128, with `share` / so: 4 trees of 64 behind 5474, 16 heads over 4, fp16 33.9 / 24.2; 8 of 32 behind 5165, 14 over 2, int8 29.9 / 21.9; 4 of 16
// behind 13281, 32 over 8, fp16 46.6 / 38.4; 8 of 16 behind 34190, 8 over 1, int8 45.0 / 34.7; 8 of 64 behind 3494, 12 heads of their own, Q4 22.0 / 24.9 (the
// worst: what tells such a batch from the others beforehand is not known).  At width 64, whose units hold two to four blocks, the same made 210 batches 3 % slower.
template <class Items>
constexpr int round_share(int share, float all, int sets, int most, const Plan& plan, int r, int blocks, const Items& items) {
    const int unit = plan.target / r;
    if (unit < 1) return share;
    const auto time = [&](int j, int of) { return static_cast<float>(j <= r ? 3 + j : (3 + r) * ((j + r - 1) / r)) * static_cast<float>(of + 12); };
    float best = 3.0e38f;
    int found = share;
    for (int k = 0; k < 2; ++k) {
        const int j = k == 0 ? r : 3 - r, room = j * unit;
        if (sets > room || room > blocks) continue;
        const int least = fitting_share(all, sets, room, most, items), of = least < plan.least ? plan.least : least;
        if (time(j, of) < best) {
            best = time(j, of);
            found = of;
        }
        if (all >= 0.85f * static_cast<float>(of) * static_cast<float>(room)) return found;
    }
    return time((items(share) + unit - 1) / unit, share) < best ? share : found;
}

// Tiles of 32 keys that a block is worth of a sequence that has so many (paged_tree.hip): fewer are a shorter chain of tiles, more are fewer parts for a set's last
// block to add up, about a microsecond for eight.  us at 4 / 8 / 16 / 32 / 48 tiles, one tree of 4 of 14 heads over 2, width 64, fp16: behind 150 positions 7.2 / 6.8 /
// 6.5 / - / -; 1000 7.4 / 7.7 / 9.0 / 9.8; 2000 8.2 / 7.6 / 8.9 / 11.6; 4000 9.8 / 8.7 / 8.7 / 11.3; 8000 13.7 / 10.4 / 9.5 / 11.1; 16000 21.1 / 14.0 / 11.5 / 12.1.
// Batches of 8 to 32 and 32 to 100 tiles of 16 rows to a compute unit, times the best: 2000 1.23 / 1.04 / 1.09 / 1.41 and 1.22 / 1.11 / 1.05 / 1.30; 8000 1.45 / 1.22 /
// 1.01 / 1.12 and 1.23 / 1.19 / 1.11 / 1.07; 16000 1.61 / 1.35 / 1.07 / 1.02 and 1.35 / 1.30 / 1.17 / 1.01; 32000 1.93 / 1.56 / 1.17 / 1.02 / 1.06 and 1.35 / 1.31 /
// 1.22 / 1.07 / 1.08.
constexpr int tree_worth(int tiles) {
    return tiles <= 12 ? 12 : tiles <= 48 ? 4 : tiles <= 96 ? 8 : tiles <= 375 ? 16 : tiles <= 750 ? 32 : tiles <= 1500 ? 48 : 64;
}

// Sets of rows_per_set rows that a launch over sequences of `from` to `to` rows has at most, whatever the lengths: every set full but
// one of each sequence, of which there are no more than tokens and than times that `from` goes into all rows; and none longer than `to`.
constexpr int64_t sets_at_most(int64_t n_tokens, int64_t n_seqs, int nrep, int rows_per_set, int from, int to) {
    const int64_t rows = n_tokens * nrep;
    int64_t seqs = n_seqs < n_tokens ? n_seqs : n_tokens;
    if (from > 0 && rows / from < seqs) seqs = rows / from;
    const int64_t full = (rows - seqs) / rows_per_set + seqs, longest = seqs * ((to - 1) / rows_per_set + 1);
    return longest < full ? longest : full;
}

// What the host knows of a call.
struct AttentionSize {
    int n_seqs = 0, n_tokens = 0, max_tokens = 0, cap = 0;
    int n_heads = 1, n_kv_heads = 1, head_dim = 64;
    int window = 0, sinks = 0;
    bool fp16 = true;         // the cache's kind, else int8 or Q4
};
struct Room {                 // of the stream's workspace: for sums, and counters
    size_t bytes = 0;
    int counters = 0;
};
struct PagedLaunch {
    int wavefronts = 0;       // of 32 rows in a block of the kernel for many rows, 0: the kernel for few
    int slices = 1;           // of keys in such a block
    int sets = 1;             // of 16 rows, of a wavefront of the kernel for trees
    Plan plan;
    int64_t blocks = 0;
    int threads = 0;
};
struct PagedLaunches {
    int n = 0;
    PagedLaunch of[2];
};

// A launch over sets of rows_per_set rows: one item per set and key/value head, and where there is room for the sums of parts (of
// `floats` floats and `counters` counters a block), `want` more, as far as it reaches.
constexpr PagedLaunch make_launch(const AttentionSize& a, int rows_per_set, int from, int to, int64_t want, const Room& room, int floats, int counters) {
    PagedLaunch l;
    l.plan.from = from;
    l.plan.to = to;
    l.plan.nrep = a.n_heads / a.n_kv_heads;
    l.plan.rep = make_divider(l.plan.nrep);
    const int64_t sums = static_cast<int64_t>(room.bytes / (static_cast<size_t>(floats) * sizeof(float))), counted = room.counters / counters;
    l.blocks = sets_at_most(a.n_tokens, a.n_seqs, l.plan.nrep, rows_per_set, from, to) * a.n_kv_heads;
    if (l.blocks == 0) return l;
    const int64_t left = (sums < counted ? sums : counted) - l.blocks, target = (want < left ? want : left) / a.n_kv_heads;
    l.plan.target = target > 0 ? static_cast<int>(target) : 0;
    l.blocks += static_cast<int64_t>(l.plan.target) * a.n_kv_heads;
    return l;
}

// Three blocks per compute unit beside one per set, but no block for fewer than 16 tiles (four per wavefront).  With 1 / 2 / 3 / 4 per
// compute unit, us: fp16, 656 MB 154 / 141 / 136.5 / 135; 16 conversations of 6676 in Q4, every head its own, 27 / 22.9 / 21.9 / 25.1; a window
// over int8, 34 MB, 12.2 / 13.2 / 13.2 / 13.4.  With at least 8 / 16 / 32 tiles: 32 conversations in int8 10.4 / 9.2 / 11.3; 3 of 2611, every
// head its own, 9.2 / 8.45 / 10.5.
constexpr PagedLaunch step_launch(const AttentionSize& a, const Room& room, int64_t cus, int to) {
    PagedLaunch l = make_launch(a, kRows, 0, to, 3 * cus, room, slot_floats(a.head_dim), 1);
    l.plan.least = 16;
    l.threads = 64 * kWaves;
    return l;
}

constexpr PagedLaunch slices_launch(const AttentionSize& a, const Room& room, int wavefronts, int slices, int from, int64_t want) {
    PagedLaunch l = make_launch(a, 32 * wavefronts, from, 0x7fffffff, want, room, chunk_slot_floats(a.head_dim, wavefronts), wavefronts);
    l.plan.least = 4;
    l.wavefronts = wavefronts;
    l.slices = slices;
    l.threads = 64 * wavefronts * slices;
    return l;
}

// A set's tiles are one chain of about 1.3 us each (width 128: twice that), so where there are few sets several wavefronts take them
// in turn.  A block of eight wavefronts is alone on its CU, of four wavefronts two are resident; sums of slices meet in LDS,
// of parts in memory, 33 KB per block.  Measured, us, width 64, 128 rows / 64 in four slices: 2048 rows of 14 heads over 2 (224
// sets) 28.5 / 33.5: blocks enough; 676 of 16 over 8 in a window of 435 (88 sets) 19.4 / 14.9; 14 sequences of 9 over 3 in a window
// of 137 21.4 / 16.6.
// Width 128, 128 rows / in two slices: 17 conversations of 32 heads over 8 (320 sets as counted here, 208 there are) 125 / 100, 14 of 16 over
// 8 90 / 74; 1024 sets 109 / -.
//
// Beside one block per set, as many as fill the chip, and at least half as many as it has CUs: sequences of other lengths need parts
// to be of one length.  None at least / half / one per CU: 32 sequences of 14 tokens to 3000 35.1 / 22.3 / 29.7; 14 of 64 tokens to 4000
// 41.6 / 26.9 / 32.6; 12 of 100, Q4, width 128, to 2500 60 / 41 / 53; 16 of 40 to 1500 38.1 / 35.2 / 37.4; one of 1000 tokens behind
// 5000 61.1 / 60.6 / 67.4; chunks and single tokens, 17 sequences, 96.8 / 97.4 / 109.
constexpr PagedLaunch chunk_launch(const AttentionSize& a, const Room& room, int64_t cus, int from) {
    const int64_t sets = sets_at_most(a.n_tokens, a.n_seqs, a.n_heads / a.n_kv_heads, 128, from, 0x7fffffff) * a.n_kv_heads, half = cus / 2;
    const auto most = [](int64_t x, int64_t y) { return x > y ? x : y; };
    if (a.head_dim == 64) {
        if (sets <= half) return slices_launch(a, room, 2, 4, from, most(cus - 2 * sets, half));
    } else {
        if (sets <= 3 * half) return slices_launch(a, room, 4, 2, from, most(cus - sets, half));
    }
    return slices_launch(a, room, 4, 1, from, 2 * cus);
}

// Which kernel.  The one for few rows reads the keys again for every 16 rows and has no start to pay for, the one for many
// rows takes a tile for 64 or 128 and first fills its LDS: about 1.3 us per tile, 4 to 6 us before the first.  So what counts is
// the work, in tiles of 16 rows by 32 keys: up to kEachCu per compute unit the whole batch is for the kernel for few rows, and
// above that only its sequences of up to kFew rows.  Kernel for few rows / for many, us, fp16:
//   14 heads over 2, width 64, 1 sequence: 112 sets of 16 rows at 1000 positions (14 tiles per compute unit) 8.9 / 12.4,
//     224 (28) 11.9 / 13.6, 448 (55) 19.1 / 14.3; 28 at 16000 (55) 23.5 / 29.2, 56 (109) 35 / 25.4, 112 (219) 56 / 28.6.
//   32 sequences: 448 sets at 500 (27) 9.9 / 11.5, 896 (55) 13.1 / 12.9, 1792 (110) 18.9 / 15.2;
//     256 at 3000 (94) 19.8 / 16.9, 448 (164) 24.4 / 21.3, 896 (328) 40 / 23.
//   32 heads over 8, width 128, 1 sequence: 256 sets at 1000 (31) 16.4 / 22.8, 512 (62) 28.8 / 23.7; 64 at 16000 (125) 47.7 / 64.2, 128 (250) 79 / 55.
//   16 heads of their own, width 128: 512 sets at 600 (38) 15.8 / 20.8, 1024 (76) 23.8 / 21.8.
//   300 tokens of 14 heads behind 900, int8 12.8 / 14.0.
//   Up to 32 rows, at any length: 8 sequences of 28 rows at 2000 8.6 / 13.1; 32 rows, width 128, at 2000 11.9 / 19.5.
// The work alone does not tell it all: few sets behind many positions (28 and 64 at 16000) are sent to the slower side, as the kernel for many
// rows adds the parts of a set one after another.
// The host knows the lengths' bound alone, the page table's width (or the window): a table much wider than its sequences are
// long moves them to the kernel for many rows sooner.
constexpr int kFew = 32, kEachCu = 48;
constexpr PagedLaunches attention_launches(const AttentionSize& a, const Room& room, int64_t cus) {
    PagedLaunches r;
    const auto add = [&](const PagedLaunch& l) {
        if (l.blocks > 0) r.of[r.n++] = l;
    };
    const int nrep = a.n_heads / a.n_kv_heads;
    const int64_t most = static_cast<int64_t>(a.max_tokens) * nrep;
    const int64_t sets = sets_at_most(a.n_tokens, a.n_seqs, nrep, kRows, 0, 0x7fffffff) * a.n_kv_heads;
    int64_t keys = a.cap;
    if (a.window > 0) {
        const int64_t seen = static_cast<int64_t>(a.window) + a.sinks + a.max_tokens;
        if (seen < keys) keys = seen;
    }
    if (most <= kFew || sets * (keys / kKeys + 1) <= kEachCu * cus) {
        add(step_launch(a, room, cus, 0x7fffffff));
    } else if (a.n_seqs == 1 || static_cast<int64_t>(a.max_tokens) * a.n_seqs == a.n_tokens) {
        add(chunk_launch(a, room, cus, 0));
    } else {
        add(chunk_launch(a, room, cus, kFew + 1));
        add(step_launch(a, room, cus, kFew));
    }
    return r;
}

// Which kernel serves a call of mi_attention_tree, always one for the whole batch: the one for few rows with 16 rows of a tree (its drafts times
// the heads of a group) per wavefront or with 32 (paged_tree.hip), or the one for many rows in blocks of 128 (paged_tree_many.hip).  The
// first reads and converts the keys again for every 16 or 32 rows, the last has a chain of 1.3 us (width 128: 2.6) per tile of 64 keys.
// us, 16 rows / 32 / 128, W: tiles of 16 rows by 32 keys per compute unit, B: blocks of 128 rows, by the host's bounds of rows and lengths:
//   width 64: 1 tree of 112 rows at 916 (W 2) 7.0 / 8.7 / 12.7; 2 of 100 at 2372, int8 (49) 11.3 / 13.4 / 18.8; 4 of 400 at 914 (45) 12.2 / 11.0 / 17.2; 4 of 300
//     at 6949, Q4 (194) 24.2 / 22.0 / 31.7; 32 of 168 at 4096 (355) int8 24.9 / 22.7 / 25.1, fp16 33.7 / 25.6 / 25.3; 32 of 192 at 2367 (333, B 192) fp16
//     37.1 / 29.3 / 24.6; 8 of 400 at 4015, Q4 (788) 48.9 / 34.2 / 35.0; 32 of 300 at 2696 (606) 54 / 43 / 32.5.
//   width 128: 4 of 96 at 3710, Q4 (49) 15.8 / 19.1 / 29; 1 of 400 at 5044 (64) 26.4 / 23.9 / 42; 4 of 96 at 5793, Q4 (54) 18.3 / 19.7 / 34.7; 8 of 512 at 3600 (77)
//     21.4 / 19.5 / 30.7; 1 of 256 at 8519 (136) fp16 45.8 / 33.9 / 53.7; 4 of 400 at 1883 (136) int8 29.4 / 37.8 / 32.6; 8 of 512 at 7286 (152) 32.0 / 25.7 / 46.2;
//     16 of 512 at 5548, Q4 (241) 39.0 / 41.6 / 50.0; 16 of 256 at 2083, int8 (196, B 144) 34.5 / 44.2 / 35.0; 8 of 400 at 4558 (303, B 92) 72 / 55 / 45.8; 2 of 128 at
//     24969, int8 (294, B 24) 59 / 52 / 71; 32 of 192 at 2276 (409, B 310) 114 / 84 / 45; 8 of 224 at 27113 (525, B 32) 88 / 64 / 97; 16 of 128 at 5583 (542, B 208)
//     91 / 79 / 51.
// Over 150 batches of each width (W 16 or 40 to 700) this takes 1.01 and 1.02 times the best of the three.  Four sets of 16 rows to a wavefront spill registers
// and took 31 us for the 22.7 above.  In batches of more than little work a block has 16 tiles at least, whatever tree_worth says: 16 trees of 16 of 15 heads over 5 behind
// 1203, int8 10.2, with 8 11.2; 4 of 2 of 12 heads of their own, width 128, behind 3432 13.7 and 17.7.
constexpr int kTreeFew = 64, kTreeLittle = 16, kTreeMuch = 440;
// W up to which 16 rows to a wavefront are better, and from which 128 are if there are blocks for a part of the units.
constexpr int one_set_up_to(int D, bool fp16) { return D == 64 ? fp16 ? 30 : 60 : fp16 ? 60 : 250; }
constexpr bool blocks_enough(int D, bool fp16, int64_t work, int64_t blocks, int64_t cus) {
    return work > 250 * cus && (D == 128 ? 4 * blocks >= cus : fp16 && 2 * blocks >= cus);
}
constexpr PagedLaunch tree_launch(const AttentionSize& a, const Room& room, int64_t cus) {
    const int nrep = a.n_heads / a.n_kv_heads;
    const int64_t rows = static_cast<int64_t>(a.max_tokens) * nrep;
    int64_t keys = a.cap;
    if (a.window > 0) {
        const int64_t seen = static_cast<int64_t>(a.window) + a.sinks + a.max_tokens;
        if (seen < keys) keys = seen;
    }
    const int64_t work = sets_at_most(a.n_tokens, a.n_seqs, nrep, kRows, 0, 0x7fffffff) * a.n_kv_heads * (keys / kKeys + 1);
    const int64_t many = sets_at_most(a.n_tokens, a.n_seqs, nrep, 128, 0, 0x7fffffff) * a.n_kv_heads;
    if ((work > kTreeMuch * cus && rows > kRows) || (rows > kTreeFew && blocks_enough(a.head_dim, a.fp16, work, many, cus)))
        return slices_launch(a, room, 4, 1, 0, 2 * cus);
    const int sets = rows > kTreeFew && work > one_set_up_to(a.head_dim, a.fp16) * cus ? 2 : 1;
    const int64_t want = a.head_dim == 64 ? (sets == 1 ? 4 : 2) * cus : (sets == 1 ? 2 : 1) * cus;
    PagedLaunch l = make_launch(a, kRows * sets, 0, 0x7fffffff, want, room, sets * slot_floats(a.head_dim), 1);
    l.plan.least = work > kTreeLittle * cus ? 4 * kWaves : 1;
    l.sets = sets;
    l.threads = 64 * kWaves;
    return l;
}

// The blocks of a launch that has more threads than a grid counts; 0: none has.
constexpr int64_t too_many_blocks(const PagedLaunches& all) {
    for (int i = 0; i < all.n; ++i)
        if (all.of[i].blocks > 0xffffffffll / all.of[i].threads) return all.of[i].blocks;
    return 0;
}

}  // namespace mi
