// Which kernels serve a call of mi_attention (paged_attention.hip), with how many blocks, and how the keys of sequences are shared
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
};
struct Room {                 // of the stream's workspace: for sums, and counters
    size_t bytes = 0;
    int counters = 0;
};
struct PagedLaunch {
    int wavefronts = 0;       // of 32 rows in a block of the kernel for many rows, 0: the kernel for few
    int slices = 1;           // of keys in such a block
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

// The blocks of a launch that has more threads than a grid counts; 0: none has.
constexpr int64_t too_many_blocks(const PagedLaunches& all) {
    for (int i = 0; i < all.n; ++i)
        if (all.of[i].blocks > 0xffffffffll / all.of[i].threads) return all.of[i].blocks;
    return 0;
}

}  // namespace mi
