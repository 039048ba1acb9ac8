// dx_moe_plan.cuh — how the two phases of moe_experts_kernel are dealt out over its
// CTAs.  Integer arithmetic only: with stand-ins for __device__, blockIdx and gridDim
// it also compiles for the host (tests/c_runtime/moe_plan.cpp).
#pragma once

namespace dx {

constexpr int kMoeSlots = 3;         // partial sums that a CTA can hold (MoePhase::slot)
constexpr int kMoeWholeBlocks = 10;  // (moe_phase)

// A run of K blocks that one accumulator collects: of one tile (phase 1), or of
// one tile and one expert (phase 2).
struct MoeRun {
  int tile, a, kb0, len;  // a: index into the chosen experts
};

// One phase's work of one CTA.  The `tiles - whole` tiles that do not make a full
// wave of the grid are dealt out first, as units of one K block, evenly and
// contiguously (a CTA gets parts of at most a few tiles); then come full waves of
// whole tiles, whose epilogues need nobody else.  So the exchange of partial sums
// runs beside the streaming of whole tiles, where a phase has any (phase 1 of
// 8 tokens, 64 experts of 2048 x 1024: 336 tiles on 148 CTAs).
struct MoePhase {
  int tiles, whole, per_tile;  // tiles [0, whole) are whole; units of a tile
  int each, more;              // split units of a CTA; the first `more` CTAs have one more
  int nt, kb;                  // phase 1: tiles of an expert; K blocks of an expert's product
  int u0, u1;                  // this CTA's units
  bool second;

  __device__ __forceinline__ int begin(int g) const { return g * each + min(g, more); }
  __device__ __forceinline__ int cta_of(int u) const {
    const int front = more * (each + 1);
    return u < front ? u / (each + 1) : more + (u - front) / each;
  }
  // The work item at position i of this CTA's list (its units, then the units of
  // its whole tiles): tile, expert index and K block.
  __device__ __forceinline__ int count() const {
    const int mine = whole > static_cast<int>(blockIdx.x)
                         ? (whole - 1 - static_cast<int>(blockIdx.x)) / static_cast<int>(gridDim.x) + 1
                         : 0;
    return u1 - u0 + mine * per_tile;
  }
  __device__ __forceinline__ void item(int i, int& tile, int& a, int& kb_) const {
    int r;
    if (i < u1 - u0) {
      const int u = u0 + i;
      tile = u / per_tile;
      r = u - tile * per_tile;
      tile += whole;
    } else {
      i -= u1 - u0;
      const int w = i / per_tile;
      r = i - w * per_tile;
      tile = static_cast<int>(blockIdx.x) + w * static_cast<int>(gridDim.x);
    }
    if (second) {
      a = r / kb;
      kb_ = r - a * kb;
    } else {
      a = tile / nt;
      kb_ = r;
    }
  }
  // Where this CTA leaves its sums of a tile: the first tile of its units, a later one,
  // or one that it has alone.  Other CTAs read the first two when they have counted
  // everyone in, and nothing tells this CTA when they are done: a slot that they read
  // is not written again in the phase (whole tiles come after the split ones).
  __device__ __forceinline__ int slot(int tile, bool alone) const {
    if (alone) return kMoeSlots - 1;
    return u0 / per_tile + whole == tile ? 0 : 1;
  }
  // The same of the split tile's first CTA (the others start inside it: slot 0).
  __device__ __forceinline__ int slot_of(int first, int tile) const {
    return begin(first) / per_tile == tile - whole ? 0 : 1;
  }
  __device__ __forceinline__ bool run(int i, MoeRun& r) const {
    if (i >= count()) return false;
    item(i, r.tile, r.a, r.kb0);
    r.len = kb - r.kb0;
    if (i < u1 - u0) r.len = min(r.len, u1 - u0 - i);
    return true;
  }
};

template <typename Params>
__device__ __forceinline__ MoePhase moe_phase(const Params& p, int chosen, bool second) {
  MoePhase f;
  const int grid = static_cast<int>(gridDim.x), g = static_cast<int>(blockIdx.x);
  f.second = second;
  f.kb = second ? p.kb_h : p.kb_d;
  f.nt = p.nt_h;
  f.per_tile = second ? chosen * p.kb_h : p.kb_d;
  f.tiles = second ? p.nt_d : chosen * p.nt_h;
  f.whole = f.tiles / grid * grid;
  // Fewer tiles than CTAs, and short ones: joining partial sums costs more than the K
  // blocks it saves the CTAs that have a tile (20 tokens, 2 of 60 experts of 1024 x 512:
  // 32.4 us whole, 35.1 split; 1 token, 1 of 8 of 2048 x 4096: 42.6 and 27.1).  Phase 2's
  // tiles are not short: each takes the K blocks of every chosen expert, and they are
  // few (D / 256), so whole ones would leave most CTAs without work.
  if (!second && f.whole == 0 && f.per_tile - f.tiles * f.per_tile / grid <= kMoeWholeBlocks)
    f.whole = f.tiles;
  const int units = (f.tiles - f.whole) * f.per_tile;
  f.each = units / grid;
  f.more = units - f.each * grid;
  f.u0 = f.begin(g);
  f.u1 = f.begin(g + 1);
  return f;
}

}  // namespace dx
