// The partition of moe_experts_kernel, walked through on the host for every CTA of a
// grid.  Arguments: grid D H chosen.  Prints "ok", or what is wrong with the plan.
#include <algorithm>
#include <cstdio>
#include <cstdlib>
#include <map>
#include <set>
#include <vector>

#define __device__
#define __forceinline__ inline
using std::min;
static struct { int x; } blockIdx, gridDim;
#include "dx_moe_plan.cuh"

struct Sizes {
  int kb_d, nt_h, kb_h, nt_d;
};

// A CTA's part of a tile, in the order it comes to them.
struct Part {
  int tile, u0, u1;  // units of the tile: [u0, u1)
  int slot;
  bool alone;
};

static int fail(const char* what, int phase, int cta, int tile) {
  printf("%s: phase %d, CTA %d, tile %d\n", what, phase + 1, cta, tile);
  return 1;
}

int main(int argc, char** argv) {
  if (argc != 5) return 2;
  const int grid = atoi(argv[1]), D = atoi(argv[2]), H = atoi(argv[3]), chosen = atoi(argv[4]);
  const Sizes s{(D + 63) / 64, (H + 127) / 128, (H + 63) / 64, (D + 255) / 256};
  gridDim.x = grid;
  for (int ph = 0; ph < 2; ++ph) {
    std::vector<std::vector<Part>> parts(grid);
    std::map<int, std::vector<char>> seen;
    std::map<int, std::set<int>> sharers;
    dx::MoePhase f{};
    for (int g = 0; g < grid; ++g) {
      blockIdx.x = g;
      f = dx::moe_phase(s, chosen, ph != 0);
      dx::MoeRun r;
      for (int u = 0; f.run(u, r); u += r.len) {
        const int expert = ph != 0 ? r.a : r.tile / f.nt;
        if (r.a != expert || r.tile < 0 || r.tile >= f.tiles || r.len < 1 || r.kb0 + r.len > f.kb)
          return fail("bad run", ph, g, r.tile);
        const int at = (ph != 0 ? r.a * f.kb : 0) + r.kb0;
        auto& mine = parts[g];
        if (!mine.empty() && mine.back().tile == r.tile) {
          if (mine.back().u1 != at) return fail("a tile in pieces", ph, g, r.tile);
          mine.back().u1 = at + r.len;
        } else {
          mine.push_back({r.tile, at, at + r.len, 0, false});
        }
        sharers[r.tile].insert(g);
        auto& units = seen[r.tile];
        units.resize(f.per_tile);
        for (int i = at; i < at + r.len; ++i)
          if (units[i]++) return fail("a unit twice", ph, g, r.tile);
      }
      for (Part& p : parts[g]) {
        p.alone = p.u0 == 0 && p.u1 == f.per_tile;
        p.slot = f.slot(p.tile, p.alone);
        if (p.slot < 0 || p.slot >= dx::kMoeSlots) return fail("bad slot", ph, g, p.tile);
      }
    }
    for (int t = 0; t < f.tiles; ++t) {
      if (!seen.count(t)) return fail("a tile left out", ph, -1, t);
      for (char c : seen[t])
        if (c != 1) return fail("a unit left out", ph, -1, t);
      // Where the others look for a shared tile's sums.
      const auto& who = sharers[t];
      if (who.size() == 1) continue;
      int next = *who.begin();
      for (int g : who) {
        if (g != next++) return fail("sharers that are not neighbours", ph, g, t);
        for (const Part& p : parts[g])
          if (p.tile == t) {
            const int want = g == *who.begin() ? f.slot_of(g, t) : 0;
            if (p.slot != want) return fail("sums looked for in another slot", ph, g, t);
            if (g != *who.begin() && f.begin(g) / f.per_tile != t - f.whole)
              return fail("a later sharer that does not start inside the tile", ph, g, t);
          }
      }
    }
    // A slot that others read keeps its sums to the end of the phase.  (Phase 1 writes a
    // tile that a CTA has alone straight to h.)
    for (int g = 0; g < grid; ++g) {
      std::set<int> read;
      for (const Part& p : parts[g]) {
        if (ph == 0 && p.alone) continue;
        if (read.count(p.slot)) return fail("sums overwritten that others may still read", ph, g, p.tile);
        if (sharers[p.tile].size() > 1) read.insert(p.slot);
      }
    }
  }
  printf("ok\n");
  return 0;
}
