// w4_chain.h -- INT4 group sums beside the matrix instructions of the chain that follows.
#pragma once

namespace hkq {

// A chain's 16 values per lane are added to the sums during the next chain of ch matrix
// instructions: values [chain_added(s, ch), chain_added(s + 1, ch)) beside instruction s,
// none beside the first, when the chain's own last instruction is still on its way.
constexpr int chain_added(int s, int ch) { return s == 0 ? 0 : (s - 1) * 16 / (ch - 1); }

constexpr bool chain_adds_each_once(int ch) {
    if (chain_added(1, ch) != 0 || chain_added(ch, ch) != 16) return false;
    for (int s = 0; s < ch; ++s)
        if (chain_added(s, ch) < 0 || chain_added(s + 1, ch) < chain_added(s, ch)) return false;
    return true;
}
static_assert(chain_adds_each_once(2) && chain_adds_each_once(4) && chain_adds_each_once(8), "groups of 32, 64, 128 values");

}  // namespace hkq
