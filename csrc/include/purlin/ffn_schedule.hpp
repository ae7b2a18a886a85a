// How the products of the gated feed-forward block (csrc/src/gated_ffn.cu) are cut into tiles and shared out over the GPU: the choice of a tile, the
// parts of a long sum, the walk of a CTA pair. Host arithmetic and a walk that the host can do too, so that both are tested without a
// GPU (csrc/tests/ffn_schedule_test.cpp). No counterpart in the reference.
#pragma once
#include <algorithm>
#include <cstddef>
#include <cstdint>

#include "constants.hpp"

namespace purlin {
namespace ffn {

constexpr int kBM = 128, kBK = 64;
enum { kStore = 0, kGate = 1, kGateGrad = 2 };

// One product of a launch: its size, its tiles, and the parts of its k (a tile of work each).
struct Tiles { int M, N, K, tilesM, tilesN, split; };

// Work [start, start + count) of a group (tiles, times the parts of k; with `halves` their accumulators one by one, 2 * count of them) in turn over
// `pairs` CTA pairs (or CTAs) from number `first` on, wrapping around.
struct Segment { int group, start, count, first, pairs, halves; };
constexpr int kMaxGroups = 3, kMaxSegments = 3 * kMaxGroups;
struct Schedule { Segment seg[kMaxSegments]; int segments; };

// Tile t -> (row block, column block), rows fastest inside bands of row blocks: the tiles in flight share operands in L2
constexpr int kBand = 8;
PURLIN_HD inline void tileCoord(const Tiles& g, int t, int& mIdx, int& nIdx) {
  const int perBand = kBand * g.tilesN, band = t / perBand, within = t - band * perBand, first = band * kBand;
  const int rows = g.tilesM - first < kBand ? g.tilesM - first : kBand;
  mIdx = first + within % rows;
  nIdx = within / rows;
}
// first row of the pair's accumulators, first column, number of accumulators
struct Item { int group, tile, part, row, col, count; };
struct KRange { int begin, end; };       // k-blocks of a part
PURLIN_HD inline KRange kRangeOf(const Tiles& g, int part) {
  const int blocks = (g.K + kBK - 1) / kBK;
  return KRange{int(int64_t(blocks) * part / g.split), int(int64_t(blocks) * (part + 1) / g.split)};
}
// The work of pair `idx` of `units`, in the order in which all warps of it walk it; body returns false to stop. group(i): the tiles of group i.
template <int CTAS, int ACCS, typename G, typename F> PURLIN_HD inline void forItems(const Schedule& p, int bn, int idx, int units, G&& group, F&& body) {
  for (int s = 0; s < p.segments; ++s) {
    const Segment& seg = p.seg[s];
    const Tiles& g = group(seg.group);
    const int at = idx - seg.first + (idx < seg.first ? units : 0);
    if (at >= seg.pairs) continue;
    const int n = ACCS == 2 && seg.halves ? 2 * seg.count : seg.count;
    for (int i = at; i < n; i += seg.pairs) {
      Item m;
      int mIdx, nIdx, first = 0;
      m.group = seg.group;
      m.tile = seg.start + (ACCS == 2 && seg.halves ? i >> 1 : i);
      m.part = 0;
      if (g.split > 1) { const int tiles = g.tilesM * g.tilesN; m.part = m.tile / tiles; m.tile -= m.part * tiles; }
      tileCoord(g, m.tile, mIdx, nIdx);
      m.count = 1;
      if constexpr (ACCS == 2) {
        if (seg.halves) first = i & 1;
        else m.count = (mIdx * ACCS + 1) * CTAS * kBM < g.M ? 2 : 1;      // rows of the last tile that end in its first accumulator
      }
      m.row = (mIdx * ACCS + first) * CTAS * kBM;
      m.col = nIdx * bn;
      if (m.row < g.M && !body(m)) return;
    }
  }
}

struct Shape { int ctas, accs, bn, split; };     // split: parts of the first product's k

struct Sizes { int M, N, K; };
inline int64_t tilesOf(const Sizes& z, const Shape& s) {
  const int tileRows = kBM * s.ctas * s.accs;
  return int64_t((z.M + tileRows - 1) / tileRows) * ((z.N + s.bn - 1) / s.bn);
}
// Expected cycles of a tile. A k-block (64 of k) takes the longest of its MMAs (bn / 2 cycles per 16 of k and accumulator, more where they all go
// into one), its loads from L2 (50 bytes a cycle and SM) and a round trip through the ring. The epilogue follows the main loop of a tile of two
// accumulators and hides under the next one's with one. The constants are fitted to 326 random sizes, each tile timed on each (a sweep on one B200, no part of the tests); over 180 others the
// choice takes 3.2 % (gate and up), 2.0 % (gate's gradient) and 2.9 % (the other gradients) longer than the best tile, where constants from
// reasoning took 5 and 3 and 5 %. us under the power cap, 512 x 256 / 256 x 256 per pair / 128 x 256 per CTA: gradient of the gate 1000 x 3584,
// k 8192 99 / 66 / 79; 8192 x 4096, k 1024 124 / 113 / 110; gate and up 4099 x 4096, k 7168 201 / 216 / 262; 2595 x 46560, k 424 196 / 183 / 219.
// In short bursts, 128 x 128 / 128 x 64 per CTA / the best wider tile: gradient of the gate 111 x 7168, k 6368 33.4 / 27.5 / 42.2.
inline double tileCycles(const Sizes& z, const Shape& s, int epi) {
  const double kBlocks = (z.K + kBK - 1) / kBK;
  const double mma = 4.0 * s.accs * s.bn / 2 * (s.accs == 2 ? 1.0 : 1.25);
  const double load = (s.accs * std::min(z.M, kBM) + s.bn / s.ctas) * 128.0 / 50;
  const double column = epi == kStore ? (s.accs == 2 ? 34 : s.ctas == 2 ? 4 : 10) : epi == kGate ? (s.accs == 2 ? 50 : s.ctas == 2 ? 24 : 31) : s.accs == 2 ? 160 : s.ctas == 2 ? 50 : 51;
  const double epilogue = s.bn * column, main = kBlocks * std::max({mma, load, 450.0});
  return s.accs == 2 ? main + 1600 + epilogue : std::max(main + 400, epilogue + 500);
}
inline size_t partialBytes(const Sizes& z, const Shape& s) { return s.split > 1 ? size_t(s.split) * size_t(tilesOf(z, s)) * size_t(kBM * s.ctas * s.accs) * size_t(s.bn) * 4 : 0; }
constexpr int kMaxSplit = 16;
constexpr size_t kMaxPartial = size_t(256) << 20;
// The tile that is expected to take least, and the parts into which k of the first product is cut (where `mayCut`): its tiles may be few and long.
// The gradient of x, [tokens, hidden], sums over twice the intermediate size: 2595 x 424 with k = 46560 has 12 tiles (all three gradients, us, whole /
// cut: 2595, 424, 23280 375 / 281; 16, 8192, 28672 530 / 511; 100, 1024, 2048 22.0 / 16.9).
inline Shape chooseShape(const Sizes* z, int n, int sms, int epi, bool mayCut) {
  Shape best{2, 2, 256, 1};
  double least = 1e30;
  auto consider = [&](Shape s) {
    const int units = sms / s.ctas;
    for (s.split = 1; s.split <= (mayCut ? kMaxSplit : 1); s.split *= 2) {
      const Sizes first{z[0].M, z[0].N, (z[0].K + s.split - 1) / s.split};
      if (s.split > 1 && (first.K < 4 * kBK || partialBytes(z[0], s) > kMaxPartial)) break;
      double cycles = 0, longest = 0;
      if (n == 1) {
        const int64_t tiles = tilesOf(z[0], s) * s.split, rest = tiles % units;
        double waves = double((tiles + units - 1) / units);
        if (s.accs == 2 && tiles > units && rest > 0 && 2 * rest <= units) waves -= 0.5;
        cycles = waves * tileCycles(first, s, epi);
      } else {
        double last = 0;
        for (int i = 0; i < n; ++i) {
          last = tileCycles(i ? z[i] : first, s, epi);
          longest = std::max(longest, last);
          cycles += double(tilesOf(z[i], s)) * (i ? 1 : s.split) * last / units;
        }
        cycles = std::max(cycles + 0.5 * last, longest);
      }
      if (s.accs == 1) cycles += 2000 + s.bn * 8.0;
      if (s.split > 1) cycles += 7000 + double(partialBytes(z[0], s)) / 3000;     // a launch, and the parts written and read
      if (cycles < least) { least = cycles; best = s; }
    }
  };
  consider({2, 2, 256, 1});
  consider({2, 2, 128, 1});
  consider({2, 1, 256, 1});
  consider({1, 1, 256, 1});
  consider({1, 1, 128, 1});
  if (epi != kGate) consider({1, 1, 64, 1});     // (64 columns of Z are 32 of h: half a staging tile)
  return best;
}

// Shares the tiles of a launch out over its pairs: group by group, the longest tiles first; pairs that got one tile fewer than others take more
// of the next group's. The last wave of all, if it fills at most half of the pairs, goes out as single accumulators.
inline void shareOut(Schedule& p, const Tiles* g, int groups, const Shape& s, int units, int epi) {
  int order[kMaxGroups] = {0, 1, 2};
  double cost[kMaxGroups] = {};
  for (int i = 0; i < groups; ++i) cost[i] = tileCycles(Sizes{g[i].M, g[i].N, (g[i].K + g[i].split - 1) / g[i].split}, s, epi);
  std::sort(order, order + groups, [&](int a, int b) { return cost[a] > cost[b]; });
  int lateFirst = 0, late = 0;                // pairs [lateFirst, lateFirst + late), wrapping around, end `ahead` cycles after the others
  double ahead = 0;
  auto add = [&](int group, int start, int count, int first, int pairs, int halves) {
    if (count > 0) p.seg[p.segments++] = Segment{group, start, count, first % units, pairs, halves};
  };
  p.segments = 0;
  for (int i = 0; i < groups; ++i) {
    const int group = order[i], tiles = g[group].tilesM * g[group].tilesN * g[group].split;
    int done = 0;
    if (late > 0) {
      const int each = int(ahead / cost[group] + 0.5);
      done = int(std::min<int64_t>(tiles, int64_t(each) * (units - late)));
      add(group, 0, done, lateFirst + late, units - late, 0);
    }
    const int left = tiles - done, whole = left / units * units, rest = left - whole;
    add(group, done, whole, lateFirst + late, units, 0);
    if (rest) {
      const bool halves = i == groups - 1 && s.accs == 2 && 2 * rest <= units && (whole || done || i > 0);
      add(group, done + whole, rest, lateFirst + late, halves ? 2 * rest : rest, halves);
      lateFirst = (lateFirst + late) % units; late = rest; ahead = cost[group];
    } else if (done && done % (units - late)) {
      const int some = done % (units - late);
      lateFirst = (lateFirst + late) % units; late = some; ahead = cost[group];
    } else if (left > 0 || done) {
      late = 0;
    }
  }
}

}  // namespace ffn
}  // namespace purlin
