// Which of several passes over a reduction a step belongs to, as plain arithmetic.
#pragma once

#include <stdint.h>

namespace ct {

// Division by `one`: value = 2^(32 + shift) / one, rounded up, with 2^shift < one <= 2^(shift + 1), so that it
// fills 32 bits. 0 for one <= 1, which needs none.
struct TermDivisor {
    uint32_t value;
    int shift;
};
constexpr TermDivisor term_divisor(int one) {
    int shift = 0;
    while (shift < 30 && (2 << shift) < one) ++shift;
    return one > 1 ? TermDivisor{(uint32_t)(((uint64_t{1} << (32 + shift)) - 1) / (uint32_t)one + 1), shift} : TermDivisor{0, 0};
}

struct TermStep {
    int product, at;
};

// t = product * one + at with 0 <= at < one, for 0 <= t < 8 one and one < 2^27. The value is too large by e / one
// with e < one, the quotient's fraction at most 1 - 1 / one: exact while t e < 2^(32 + shift), and
// t e < 8 one^2 <= 2^(shift + 4) one. (A correction by comparison instead of the shift costs 3% of the float32
// products, a reciprocal without either is one too large from 26992 steps on.)
constexpr TermStep term_step(int t, int one, TermDivisor by) {
    const int s = one > 1 ? (int)((uint64_t)(uint32_t)t * by.value >> 32) >> by.shift : t;
    return TermStep{s, t - s * one};
}

}  // namespace ct
