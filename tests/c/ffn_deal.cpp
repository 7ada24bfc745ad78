// Replays the dealing of pair launches (morph_b200/csrc/mb_ffn_deal.cuh) on the CPU.
// A line of input per launch: twos, pairs, number of problems, then mt, nt, kb and nseg
// of each; a line of output: 1 if every k-block of every tile is dealt exactly once and
// the pieces fit the workspace, the busiest unit's load and the even share of all, in
// k-blocks (a tile or piece costs kTileKb beside its own), and the cut tiles' pieces.
#include <cstdio>
#include <vector>

#include "mb_ffn_deal.cuh"

using namespace mb::ffn;

int main() {
  int twos, most, n;
  while (std::scanf("%d %d %d", &twos, &most, &n) == 3) {
    Deal g{};
    g.nprob = n;
    std::vector<std::vector<int>> done(n);  // k-blocks dealt, by tile
    for (int i = 0; i < n; ++i) {
      Problem& p = g.p[i];
      if (std::scanf("%d %d %d %d", &p.mt, &p.nt, &p.kb, &p.nseg) != 4) return 1;
      done[i].assign((size_t)p.mt * p.nt, 0);
    }
    deal_tiles(g, twos != 0, most);
    bool ok = g.sched.units <= most;
    long busiest = 0, all = 0, pieces = 0;
    std::vector<std::vector<int>> cut(g.sched.long_tiles);  // first k-blocks of the pieces
    for (int u = 0; u < g.sched.units; ++u) {
      long load = 0;
      Item it{};
      for (Items work(g.sched, u); work.next(g, it);) {
        for (int m = 0; m < it.count; ++m) {
          const Problem& p = g.p[it.prob];
          if (it.prob >= n || it.bm + m >= p.mt || it.bn >= p.nt || it.k0 < 0 || it.k0 >= it.k1 || it.k1 > p.kb * p.nseg) {
            ok = false;
            break;
          }
          done[it.prob][(size_t)(it.bm + m) * p.nt + it.bn] += it.k1 - it.k0;
          load += it.k1 - it.k0 + kTileKb;
        }
        if (it.piece >= 0) {
          ++pieces;
          ok = ok && it.count == 1 && it.tile < g.sched.long_tiles && it.piece < g.sched.ways &&
               it.tile * g.sched.ways + it.piece < kMaxPairs;
          if (ok) cut[it.tile].push_back(it.k0);
        }
      }
      busiest = load > busiest ? load : busiest;
      all += load;
    }
    for (int i = 0; i < n; ++i)
      for (int k : done[i]) ok = ok && k == g.p[i].kb * g.p[i].nseg;
    for (auto& starts : cut)  // a tile's pieces begin at different k-blocks: none is dealt twice
      for (size_t i = 0; i < starts.size(); ++i)
        for (size_t j = 0; j < i; ++j) ok = ok && starts[i] != starts[j];
    std::printf("%d %ld %ld %ld\n", ok ? 1 : 0, busiest, (all + most - 1) / most, pieces);
  }
  return 0;
}
