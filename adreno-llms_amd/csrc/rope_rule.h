// The angle of a rotary pair (rope.hip), as exact as fp32's cosine and sine can tell at any position.  Plain C++ (constexpr makes device code
// as well).
#pragma once

namespace mi {

// position * inv_freq / 2 pi less the nearest integer, in turns from -1/2 to 1/2, within 2^-53 and 2^-102 of the turns that were taken off.  A position
// has 31 bits and inv_freq 24, so their product is one number of 53 bits and what its rounding left, which fma gives exactly; so it is with the
// product by 1 / 2 pi, of which there are two numbers.  (With products rounded to 53 bits alone an angle of 2^31 is 4 10^-7 off, seven of fp32's steps,
// and more with an inv_freq above 1.  What it costs shows where angles are most of the work: 30000 rows of two heads of 128 14.1 -> 14.5 us; 4096 of 40 are
// 13.8 either way.)
template <class Wide = double>                     // (constexpr takes fma and rint in templates alone)
constexpr Wide turns_of(int position, float inv_freq) {
    constexpr Wide kTurn = 0x1.45f306dc9c883p-3, kRest = -0x1.6b01ec5417056p-57;     // 1 / 2 pi
    const Wide p = static_cast<Wide>(position), f = static_cast<Wide>(inv_freq);
    const Wide angle = p * f, left = __builtin_fma(p, f, -angle);
    const Wide turns = angle * kTurn, rest = __builtin_fma(angle, kTurn, -turns) + __builtin_fma(angle, kRest, left * kTurn);
    const Wide part = (turns - __builtin_rint(turns)) + rest;
    return part - __builtin_rint(part);
}

}  // namespace mi
