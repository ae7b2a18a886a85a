// How long a wait inside a tile kernel may last before it gives up. No counterpart in the reference.
#pragma once
#include <cstdint>

namespace purlin {

// An epilogue waits for whole main loops, which take as long as their sums: 2^29 tokens are 2^23 k-blocks of a weight's gradient, 2 to 3 s at 450 cycles
// each. So: two seconds, and 4096 ns for each k-block that a CTA (or pair) walks, several times what one takes (0.2 to 1.2 us).
inline uint64_t waitLimitNs(int64_t kBlocks) { return 2000000000ull + 4096ull * uint64_t(kBlocks > 0 ? kBlocks : 0); }

}  // namespace purlin
