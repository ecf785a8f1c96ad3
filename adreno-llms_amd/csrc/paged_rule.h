// What the kernels over a paged cache (kv_cache.hip, paged_attention.hip) take from the numbers that a call leaves in device
// memory: where a row lies, what a query sees, which tiles of keys a group of queries has, and how tiles are shared out to
// blocks.  Every such number is checked here, so that no value of it leads out of the caller's arrays.  Plain C++
// (constexpr makes device code as well).
#pragma once
#include <cstdint>

namespace mi {

// n / d for 0 <= n < 2^31 and d >= 1, without a division: n * mul >> (32 + shift), mul = ceil(2^(32 + shift) / d),
// 2^shift < d <= 2^(shift + 1) (d = 1: shift 0, taken apart).  mul < 2^32, and n * (mul * d - 2^(32 + shift)) < 2^31 * d
// <= 2^(32 + shift), so the error never reaches the next quotient.
struct Divider {
    int d = 1;
    uint32_t mul = 0;
    int shift = 0;
};
constexpr Divider make_divider(int d) {
    Divider r{};
    r.d = d;
    if (d == 1) return r;
    while ((2ll << r.shift) < d) ++r.shift;
    r.mul = static_cast<uint32_t>(((1ull << (32 + r.shift)) + static_cast<uint64_t>(d) - 1) / static_cast<uint64_t>(d));
    return r;
}
constexpr int divide(int n, const Divider& v) {
    return v.d == 1 ? n
                    : static_cast<int>(static_cast<uint32_t>((static_cast<uint64_t>(static_cast<uint32_t>(n)) * v.mul) >> 32) >> v.shift);
}

// Rows first .. first + n - 1 of the batch, the first of them at position `pos`.
struct Span {
    int first = 0, n = 0, pos = 0;
};
constexpr Span span_of(int start, int end, int len, int n_tokens) {
    Span s{};
    s.first = start < 0 ? 0 : start > n_tokens ? n_tokens : start;
    const int e = end < s.first ? s.first : end > n_tokens ? n_tokens : end;
    s.n = e - s.first;
    s.pos = (len < 0 ? 0 : len) - s.n;             // (n >= 0: no overflow; negative where a sequence has more rows than positions)
    return s;
}
// Whether a sequence's rows end before they begin.  Where none does, no two sequences have a row in common, and what is computed from
// n_tokens (blocks, room for sums) is enough for all of them.
constexpr bool goes_down(int start, int end) { return end < start; }

// Positions that a table of max_pages pages has, as far as an int counts them.
constexpr int capacity(int max_pages, int page_size) {
    const long long c = static_cast<long long>(max_pages) * page_size;
    return c < 0x7fffffffll ? static_cast<int>(c) : 0x7fffffff;
}

// Whether a query at position p (p >= 0) sees position j (j >= 0), as far as the mask goes.
constexpr bool sees(int p, int j, int window, int sinks) {
    return j <= p && (window <= 0 || j > p - window || j < sinks);
}

// Tiles of `size` keys that queries at positions p_lo .. p_hi see anything of: tiles 0 .. head - 1 (sinks alone) and from `from`
// on, `count` in all, numbered through (tile_at).  `end`: one past the last position that any of them sees.
struct Tiles {
    int head = 0, from = 0, count = 0, end = 0;
};
constexpr Tiles tiles_of(int p_lo, int p_hi, int cap, int window, int sinks, int size) {
    Tiles t{};
    if (p_hi < 0) return t;
    t.end = p_hi < cap ? p_hi + 1 : cap;
    const int first = window > 0 && p_lo >= window ? p_lo - window + 1 : 0;    // of the window, for the first query
    const int stay = sinks < first ? sinks : first;
    const int last = (t.end - 1) / size + (t.end > 0);                         // tiles up to the end (without end + size - 1: no overflow)
    t.head = stay > 0 ? (stay - 1) / size + 1 : 0;
    t.from = first / size;
    if (t.from > last) t.from = last;
    if (t.head >= t.from) t.head = t.from = 0;
    t.count = t.head + last - t.from;
    return t;
}
constexpr int tile_at(const Tiles& t, int i) { return i < t.head ? i : i - t.head + t.from; }

// Whether every query at p_lo .. p_hi sees all `size` keys from j0 on, all within the window or all among the sinks.
constexpr bool all_seen(int j0, int size, int p_lo, int p_hi, int cap, int window, int sinks) {
    const int last = j0 + (size - 1);
    return last <= p_lo && last < cap && (window <= 0 || j0 > p_hi - window || last < sinks);
}

}  // namespace mi
