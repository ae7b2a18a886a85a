// Host-only unit test of the limit of waits (purlin/wait_limit.hpp): never below two seconds, above every main loop that the sizes allow, and no wrap.
#include <cstdio>
#include <initializer_list>

#include "purlin/wait_limit.hpp"

using purlin::waitLimitNs;

static int g_failures = 0;
#define CHECK(cond, what)                                                                        \
  do {                                                                                           \
    if (!(cond)) { std::printf("FAIL  %s (%s:%d)\n", what, __FILE__, __LINE__); ++g_failures; }  \
  } while (0)

int main() {
  CHECK(waitLimitNs(0) == 2000000000ull && waitLimitNs(-5) == 2000000000ull, "two seconds at least");
  // the longest sums: 2^29 tokens (k-blocks of 64), 2^31 columns in 4 bits (k-blocks of 256); a k-block takes up to 1.2 us
  for (long long kBlocks : {1ll, 128ll, 1ll << 20, 1ll << 23})
    CHECK(double(waitLimitNs(kBlocks)) > 2e9 + 3 * 1200.0 * double(kBlocks), "three times a main loop's time, and two seconds");
  CHECK(waitLimitNs(1ll << 40) > waitLimitNs(1ll << 39), "no wrap for many long tiles");
  std::printf(g_failures ? "%d FAILURES\n" : "PASSED\n", g_failures);
  return g_failures ? 1 : 0;
}
