// A cache of keys and values in 8 bits: blocks of 64 tokens of a head, one scale for a block's keys and one for its values.
// Of a block the keys are [64][width] and the values, transposed, [width][64]: what a lane multiplies with is 16 bytes in a
// row of both.  The last 128 tokens of a sequence are kept in the activations' type as well, token p in row p % 128 of a
// tail; those of a block that is not complete are read there.
#pragma once
#include "common.hpp"

namespace lrqk {

constexpr int kByBlock = 64, kByTail = 128;

// Width that rows are held in.
static inline int by_width(int d) { return d <= 64 ? 64 : d <= 128 ? 128 : 256; }

}  // namespace lrqk
