// How the tiles of a pair launch of mb_ffn.cu are numbered, cut and dealt to its CTA
// pairs. Plain C++ as well as device code: the host fills a Deal, the roles of the
// kernel walk it (Items), and tests/c/ffn_deal.cpp replays it on the CPU.
#pragma once

#include <cstddef>
#include <cstdint>

#ifdef __CUDACC__
#define MB_HD __host__ __device__ __forceinline__
#else
#define MB_HD inline
#endif

namespace mb {
namespace ffn {

constexpr int kGroupLog2 = 4;  // row tiles of a group: 16 (see tile order in mb_ffn.cu)
constexpr int kMaxProblems = 4;
constexpr int kMaxPairs = 96;  // pairs a launch may have, for the size of its workspace
constexpr int kTileKb = 6;
constexpr int kLongDouble = 4;  // long tiles go in twos while one is at most this part of a pair's share

// Division of 0 <= x < 2^31 by a fixed d >= 1: floor(x m / 2^shift) with
// m = ceil(2^shift / d), shift = 31 + ceil(log2 d), exact since m d - 2^shift < 2^(shift - 31).
// The roles of a CTA find their next tile between two k-blocks: the compiler's
// divisions by run-time values cost more there than a k-block takes.
struct Div {
  uint32_t m;
  int shift;
  MB_HD int operator()(int x) const { return (int)(((uint64_t)(uint32_t)x * m) >> shift); }
};

inline Div make_div(int64_t d) {
  int log = 0;
  while (((int64_t)1 << log) < d) ++log;
  const int shift = 31 + log;
  return {(uint32_t)((((uint64_t)1 << shift) + (uint64_t)d - 1) / (uint64_t)d), shift};
}

// One problem of a pair launch: an output [M, N] (gated: N features) and up to two K
// segments accumulated into it. Operands and output name the launch's maps.
struct Problem {
  int M, N;
  int kb, nseg;      // 64-deep blocks of one segment; segments
  int a_mn;          // A is stored [K, M] (the form that takes either)
  int a[2], b[2];    // by segment; gated: b by CTA of the pair (gate, up)
  int o;             // backward: dg, du, h at o, o + 1, o + 2
  int mt, nt, tile0; // row and column tiles; its first tile's number
  // groups of rows of tiles (of pairs of them with pairing 2): their number of rows
  // (log2), the last one's, and the division by a group's tiles and by that last height
  int group_log2, height, tail_rows;
  Div by_group, by_tail;
};

// How a launch's tiles are dealt to its units (CTA pairs). With pairing 2 the tiles
// 2i and 2i + 1 are vertical neighbours, and a unit may take both as one item: they
// share B's loads. The first long_tiles tiles (of the problems with the longest
// contraction) go first: whole, in items of long_step, or each cut into `ways` pieces:
// n_long items in turn. Of the n_rest items after them (n_double double ones, then
// single tiles) the first `early` go to the units from `late_units` on, which had one
// long item less, and the others to all in turn.
struct Sched {
  int units, pairing, long_tiles, long_step, ways, n_long, n_rest, n_double, early, late_units;
};

// A launch's problems, those with the longer contraction first, and their dealing.
struct Deal {
  Problem p[kMaxProblems];
  int nprob;
  Sched sched;
};

// Tiles go in twos (one load of B for both: 96 instead of 128 KB of operands) where the
// contraction is long enough to cover that both epilogues end together, and there are
// rounds enough: in k-blocks and rounds of tiles. Measured against single tiles, one call
// among idle ones: 4096 tokens, d 4096, f 11008: gate and up 478 -> 467 us, backward 2000
// -> 1945; but the backward of 2048 tokens, d 2048, f 5504 (8 rounds) 285 -> 292, of 1024
// tokens, d 4096 (16 k-blocks) 549 -> 559. Back to back, at the power limit, the gradients'
// two limits matter less: 4 rounds instead of 16 gives 305 -> 310 and, for 8192 tokens,
// d 1024, f 4096, 509 -> 492; 8 k-blocks instead of 32, of 1024 tokens, 621 -> 639; 2048
// tokens, d 4096, f 11008 take 1180 whichever way. The backward projection's epilogue is
// too long for it (417 -> 472 thousand cycles).
constexpr int kTwosKb = 64, kTwosRounds = 2, kTwosKbGrads = 32, kTwosRoundsGrads = 16;
// When a pair launch cuts its last round: pieces of at least kMinPieceKb k-blocks, at
// most kMaxWays of them, for a gain of at least kMinSavedKb k-blocks' time, which covers
// the partials and the join. In us, for a gain of 24, 16 and 8, and without cuts:
//   gated, 1021 tokens, d 2048, f 5504     37.0   39.5   39.5   36.9
//   backward of the same                  181    190    191    182
//   forward, 256, 4096, 11008              78.7   78.2   78.9  109
//   backward of the same                  244    244    245    240
//   forward, 600, 4096, 11008             191    193    191    186
//   forward, 777, 1024, 2816               31.0   31.0   34.8   34.5
//   backward of the same                   64.5   64.5   70.9   64.7
//   backward, 300, 1024, 4096              52.5   52.5   55.1   52.5
//   backward, 1500, 1536, 4096            150    155    155    149
constexpr int kMinPieceKb = 4, kMaxWays = 4, kMinSavedKb = 24;

// One piece of work: k-blocks [k0, k1) of `count` tiles from row tile bm on, column
// tile bn, of a problem; `piece` of a cut tile, else -1.
struct Item {
  int tile, count, prob, bm, bn, k0, k1, piece;
};

// Tile -> problem and place: groups of 16 row tiles, row tiles fastest inside a
// group. False for the tile below an odd number of row tiles.
MB_HD bool place_tile(const Deal& g, Item& it) {
  it.prob = 0;
  for (int i = 1; i < kMaxProblems; ++i)
    if (i < g.nprob && it.tile >= g.p[i].tile0) it.prob = i;
  const Problem& p = g.p[it.prob];
  const bool twos = g.sched.pairing == 2;
  const int t = it.tile - p.tile0;
  const int cell = twos ? t >> 1 : t;
  const int group = p.by_group(cell), first = group << p.group_log2;
  const int in = cell - first * p.nt;
  int row;
  if (p.height - first >= 1 << p.group_log2) {
    row = in & ((1 << p.group_log2) - 1);
    it.bn = in >> p.group_log2;
  } else {
    it.bn = p.by_tail(in);
    row = in - it.bn * p.tail_rows;
  }
  row += first;
  it.bm = twos ? 2 * row + (t & 1) : row;
  it.k0 = 0;
  it.k1 = p.kb * p.nseg;
  it.piece = -1;
  if (it.bm + it.count > p.mt) it.count = p.mt - it.bm;
  return it.count > 0;
}

struct Items {
  int unit, next_long, next_early, next_rest;
  MB_HD Items(const Sched& s, int u)
      : unit(u), next_long(u), next_early(u >= s.late_units ? u - s.late_units : s.early), next_rest(s.early + u) {}
  MB_HD bool next(const Deal& g, Item& it) {
    const Sched& s = g.sched;
    while (true) {
      if (next_long < s.n_long) {
        int piece = 0;
        it.tile = next_long * s.long_step;
        if (s.ways > 1) {
          it.tile = next_long / s.ways;
          piece = next_long - it.tile * s.ways;
        }
        it.count = s.long_step;
        next_long += s.units;
        if (!place_tile(g, it)) continue;
        if (s.ways > 1) {
          const int kb = it.k1;
          it.piece = piece;
          it.k0 = (int)((int64_t)kb * piece / s.ways);
          it.k1 = (int)((int64_t)kb * (piece + 1) / s.ways);
        }
        return true;
      }
      int j;
      if (next_early < s.early) {
        j = next_early;
        next_early += s.units - s.late_units;
      } else {
        j = next_rest;
        if (j >= s.n_rest) return false;
        next_rest += s.units;
      }
      it.count = j < s.n_double ? 2 : 1;
      it.tile = s.long_tiles + j + (j < s.n_double ? j : s.n_double);
      if (place_tile(g, it)) return true;
    }
  }
};

// `tiles` tiles of kb k-blocks, all alike, over at most `most` pairs: full rounds of
// whole tiles (double ones with pairing 2), and the last round's tiles cut when that
// saves enough.
inline Sched deal_one(int tiles, int kb, int most, int pairing) {
  Sched s{};
  s.units = tiles < most ? tiles : most;
  s.pairing = pairing;
  s.long_step = s.ways = 1;
  int rest = tiles % most;
  int ways = rest ? most / rest : 1;
  if (ways > kMaxWays) ways = kMaxWays;
  if (ways > kb / kMinPieceKb) ways = kb / kMinPieceKb;
  if (rest && pairing == 2 && (rest & 1)) ++rest;  // what follows starts on a pair
  if (ways >= 2 && rest * ways <= most && kb - kb / ways >= kMinSavedKb) {
    s.long_tiles = rest;
    s.ways = ways;
    s.n_long = rest * ways;
    s.units = tiles > most ? most : s.n_long;
  }
  const int whole = tiles - s.long_tiles;
  s.n_double = pairing == 2 ? whole / (2 * most) * most : 0;
  s.n_rest = whole - s.n_double;
  return s;
}

// `first` tiles of long_kb k-blocks and `rest` tiles of kb: the long ones first, cut
// when one of them is more than a pair's share of the whole, the others so that the
// pairs end together. A tile costs about kTileKb k-blocks' time beside its own
// (filling the ring, storing).
inline Sched deal_two(int first, int64_t long_kb, int rest, int kb, int most, int pairing) {
  const int64_t cost = kb + kTileKb;
  const int64_t share = (first * (long_kb + kTileKb) + rest * cost + most - 1) / most;
  Sched s{};
  s.pairing = pairing;
  s.long_tiles = first;
  s.ways = s.long_step = 1;
  if (long_kb > share) {
    int ways = (int)((long_kb + share - 1) / share);
    if (ways > kMaxWays) ways = kMaxWays;
    if (ways > most / first) ways = most / first;
    if (ways > long_kb / kMinPieceKb) ways = (int)(long_kb / kMinPieceKb);
    if (ways > 1) s.ways = ways;
  } else if (pairing == 2 && kLongDouble * long_kb <= share) {
    s.long_step = 2;
  }
  s.n_long = first / s.long_step * s.ways;
  // double tiles but for about the last two rounds
  if (pairing == 2 && rest > 4 * most) s.n_double = (rest - 2 * most) / 2;
  s.n_rest = rest - s.n_double;
  s.units = s.n_long + s.n_rest < most ? s.n_long + s.n_rest : most;
  s.late_units = s.n_long % s.units;
  if (s.late_units > 0) {
    // items that make up for a long one
    const int64_t one = s.n_double > 0 ? 2 * cost : cost;
    const int64_t lead = (s.long_step * long_kb / s.ways + kTileKb + one / 2) / one;
    const int64_t early = (lead > 0 ? lead : 1) * (s.units - s.late_units);
    const int most_early = s.n_double > 0 ? s.n_double : rest;
    s.early = (int)(early < most_early ? early : most_early);
  }
  return s;
}

// Numbers the tiles of g's problems (mt, nt, kb and nseg are set; by falling
// contraction) and deals them over at most `most` units. `twos`: the kernel has a form
// for double tiles.
inline void deal_tiles(Deal& g, bool twos, int most) {
  const int n = g.nprob;
  const auto depth = [&](int i) { return g.p[i].kb * g.p[i].nseg; };
  int64_t tiles = 0;
  for (int i = 0; i < n; ++i) tiles += (int64_t)g.p[i].mt * g.p[i].nt;
  twos = twos && tiles >= (n > 1 ? kTwosRoundsGrads : kTwosRounds) * most &&
         depth(n - 1) >= (n > 1 ? kTwosKbGrads : kTwosKb);
  const int pairing = twos ? 2 : 1;
  int total = 0, first = 0;  // first: tiles of the longest contraction
  for (int i = 0; i < n; ++i) {
    Problem& p = g.p[i];
    p.tile0 = total;
    p.group_log2 = pairing == 2 ? kGroupLog2 - 1 : kGroupLog2;
    p.height = (p.mt + pairing - 1) / pairing;
    p.tail_rows = p.height & ((1 << p.group_log2) - 1);
    p.by_group = make_div(p.nt << p.group_log2);
    p.by_tail = make_div(p.tail_rows > 0 ? p.tail_rows : 1);
    total += p.height * pairing * p.nt;
    if (depth(i) == depth(0)) first = total;
  }
  g.sched = first == total ? deal_one(first, depth(0), most, pairing)
                           : deal_two(first, depth(0), total - first, depth(n - 1), most, pairing);
}

}  // namespace ffn
}  // namespace mb
