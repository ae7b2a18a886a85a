// Host-only unit test of the feed-forward block's schedule (purlin/ffn_schedule.hpp): every accumulator of every tile and part of k is walked exactly
// once whatever the sizes, tiles and number of pairs, parts of k meet without a gap, no pair is left with much more than its share, and the
// choice of a tile holds to what the kernel has room for.
#include <cstdio>
#include <map>
#include <random>
#include <tuple>
#include <vector>

#include "purlin/ffn_schedule.hpp"

using namespace purlin::ffn;

static int g_failures = 0;
#define CHECK(cond, what)                                                                        \
  do {                                                                                           \
    if (!(cond)) { std::printf("FAIL  %s (%s:%d)\n", what, __FILE__, __LINE__); ++g_failures; }  \
  } while (0)

static Tiles tiled(Sizes z, const Shape& s, int split) {
  const int rows = kBM * s.ctas * s.accs;
  return Tiles{z.M, z.N, z.K, (z.M + rows - 1) / rows, (z.N + s.bn - 1) / s.bn, split};
}

template <int CTAS, int ACCS> static void walkOnce(const std::vector<Sizes>& z, Shape s, int sms, int epi) {
  Tiles g[kMaxGroups] = {};
  const int n = int(z.size());
  int64_t tiles = 0;
  double total = 0, longest = 0;
  for (int i = 0; i < n; ++i) {
    g[i] = tiled(z[i], s, i ? 1 : s.split);
    tiles += int64_t(g[i].tilesM) * g[i].tilesN * g[i].split;
    const double c = tileCycles(Sizes{z[i].M, z[i].N, (z[i].K + g[i].split - 1) / g[i].split}, s, epi);
    total += c * double(g[i].tilesM) * g[i].tilesN * g[i].split;
    longest = std::max(longest, c);
  }
  const int units = int(std::min<int64_t>(sms / CTAS, tiles));
  Schedule p{};
  shareOut(p, g, n, s, units, epi);
  CHECK(p.segments >= 1 && p.segments <= kMaxSegments, "segments fit their table");
  std::map<std::tuple<int, int, int, int>, int> seen;          // (group, part, first row of an accumulator, column) -> how often
  double worst = 0;
  for (int u = 0; u < units; ++u) {
    double cost = 0;
    forItems<CTAS, ACCS>(p, s.bn, u, units, [&](int i) -> const Tiles& { return g[i]; }, [&](const Item& m) {
      CHECK(m.count >= 1 && m.count <= ACCS && m.part >= 0 && m.part < g[m.group].split && m.col < z[m.group].N && m.row < z[m.group].M, "an item lies inside its product");
      for (int a = 0; a < m.count; ++a) ++seen[{m.group, m.part, m.row + a * CTAS * kBM, m.col}];
      cost += tileCycles(Sizes{z[m.group].M, z[m.group].N, (z[m.group].K + g[m.group].split - 1) / g[m.group].split}, s, epi) * m.count / ACCS;
      return true;
    });
    worst = std::max(worst, cost);
  }
  int64_t want = 0;
  bool once = true;
  for (int i = 0; i < n; ++i)
    for (int part = 0; part < g[i].split; ++part)
      for (int row = 0; row < z[i].M; row += CTAS * kBM)
        for (int col = 0; col < z[i].N; col += s.bn) {
          ++want;
          const auto at = seen.find({i, part, row, col});
          once = once && at != seen.end() && at->second == 1;
        }
  CHECK(once && int64_t(seen.size()) == want, "every accumulator of every part exactly once");
  CHECK(worst <= total / units + 2.01 * longest, "no pair has much more than its share");
  for (int i = 0; i < n; ++i) {
    int end = 0;
    for (int part = 0; part < g[i].split; ++part) {
      const KRange k = kRangeOf(g[i], part);
      CHECK(k.begin == end && k.end > k.begin, "the parts of k meet, none is empty");
      end = k.end;
    }
    CHECK(end == (z[i].K + kBK - 1) / kBK, "the parts of k cover it");
  }
}

static void walk(const std::vector<Sizes>& z, const Shape& s, int sms, int epi) {
  if (s.accs == 2) walkOnce<2, 2>(z, s, sms, epi);
  else if (s.ctas == 2) walkOnce<2, 1>(z, s, sms, epi);
  else walkOnce<1, 1>(z, s, sms, epi);
}

int main() {
  std::mt19937 rng(5);
  auto between = [&](int lo, int hi) { return int(std::uniform_int_distribution<int>(lo, hi)(rng)); };
  auto size = [&](int most) { int v = most; for (int i = between(0, 9); i > 0; --i) v = std::max(1, v / 2); return between(1, v); };
  int walks = 0;
  for (int round = 0; round < 1500; ++round) {
    const int tokens = size(9000), hidden = 8 * size(700), intermediate = 16 * size(400), sms = round % 3 ? 148 : between(2, 160);
    const std::vector<Sizes> grads = {{tokens, hidden, 2 * intermediate}, {2 * intermediate, hidden, tokens}, {hidden, intermediate, tokens}};
    const Sizes up{tokens, 2 * intermediate, hidden}, gate{tokens, intermediate, hidden};
    for (int epi : {kStore, kGate, kGateGrad}) {
      std::vector<Sizes> z;
      if (epi == kStore) for (const Sizes& g : grads) { if (between(0, 3)) z.push_back(g); }
      else z.push_back(epi == kGate ? up : gate);
      if (z.empty()) continue;
      const Shape s = chooseShape(z.data(), int(z.size()), sms, epi, epi == kStore && z[0].K == 2 * intermediate);
      CHECK(s.bn % 64 == 0 && s.bn <= 256 && (s.ctas == 1 || s.bn % 128 == 0) && (epi != kGate || s.bn % 128 == 0), "a tile the kernel has");
      CHECK((s.ctas == 2 && s.accs == 2) || (s.ctas == 2 && s.accs == 1) || (s.ctas == 1 && s.accs == 1), "a tile the kernel has");
      CHECK(s.split >= 1 && s.split <= kMaxSplit && partialBytes(z[0], s) <= kMaxPartial, "the parts fit the workspace");
      walk(z, s, sms, epi);
      // any tile, whether it would be chosen or not
      const Shape any[] = {{2, 2, 256, 1}, {2, 2, 128, 1}, {2, 1, 256, 1}, {1, 1, 256, 1}, {1, 1, 128, 1}};
      walk(z, any[between(0, 4)], sms, epi);
      walks += 2;
    }
  }
  std::printf("%d schedules\n", walks);
  std::printf(g_failures ? "%d FAILURES\n" : "PASSED\n", g_failures);
  return g_failures ? 1 : 0;
}
