// What the products grouped by expert share (grouped.hip).
#pragma once
#include "packed.h"

namespace hi2x {

enum { GROUPED_LINEAR = 0, GROUPED_GRAD_X = 1, GROUPED_GRAD_W = 2 };

struct GroupedArgs {
  const void *x, *dy, *w;
  void* out;
  const int64_t *rows, *offs;
  int64_t ldx, ldy, x_rows, slots;
  int64_t ldw;  // of w's rows; an expert's are n of them
  int64_t experts, n, k;
  bool past = false;  // results go past the caches
  bool f32_out = false;  // of 16-bit operands (the tokens' gradient of each slot, to be added up)
};

// Expert e's slots, empty where the ranges are not as they should be.
__device__ __forceinline__ void slot_range(const GroupedArgs& g, int e, int64_t& a, int64_t& b) {
  a = g.offs[e];
  b = g.offs[e + 1];
  a = a < 0 ? 0 : (a > g.slots ? g.slots : a);
  b = b < a ? a : (b > g.slots ? g.slots : b);
}

// A row tile: slots [first, first + live) of expert e, or of none (e < 0: zeros).
struct RowTile {
  int64_t first;
  int32_t live, e;
};
struct Plan {
  int64_t count;
  int64_t reserved;
  RowTile tile[1];
};

// Row tiles of T slots at most: every range's last may be partial.
inline int64_t most_tiles(const GroupedArgs& g, int T) {
  return g.slots / T + (g.slots < g.experts ? g.slots : g.experts) + 2;
}
inline int64_t plan_bytes(const GroupedArgs& g, int T) {
  return align256(sizeof(Plan) + most_tiles(g, T) * sizeof(RowTile));
}

// The row tiles of T slots, expert after expert, then those of the slots behind the last range and
// before the first.
int launch_plan(const GroupedArgs& g, int T, Plan* plan, hipStream_t s, const char* name);

// The tile of a plan's row tiles (y) x nx columns (xt) that workgroup `block` of 8 ceil(tiles / 8)
// takes.  Workgroups go to the eight XCDs in turn, and each XCD takes an eighth of the tiles, which are in
// order of four row tiles at a time, column tile after column tile, so that rows and weights come to
// its L2 once.
__device__ __forceinline__ bool plan_tile(const Plan* p, uint32_t nx, uint32_t block, RowTile& w,
                                          uint32_t& xt, uint32_t& y) {
  const uint32_t count = (uint32_t)p->count, all = count * nx, per = (all + 7) / 8;
  const uint32_t j = block >> 3, at = (block & 7) * per + j;
  if (j >= per || at >= all) return false;
  // (what comes out of a division is in a vector register, and would keep what follows there)
  const uint32_t band = __builtin_amdgcn_readfirstlane(at / (4 * nx));
  const uint32_t rest = at - band * (4 * nx);
  const uint32_t deep = count - 4 * band < 4 ? count - 4 * band : 4;
  xt = __builtin_amdgcn_readfirstlane(rest / deep);
  y = 4 * band + rest - xt * deep;
  w = p->tile[y];
  return true;
}

// What a resource that offsets of 32 bits reach may span: an offset past it by this much again is
// past it still.
constexpr uint32_t GROUPED_SPAN = 0x7f000000u;

// The product in tiles of 16-bit operands that lie so, or of float32 ones with x within reach, and
// the workspace that it takes for its plan.
int64_t grouped_plan_bytes(const GroupedArgs& g, int what, int dtype);
int grouped_tiles(const GroupedArgs& g, int what, int dtype, char* plan, hipStream_t s,
                  const char* name);

// The side of the tiles that 16-bit operands take, and the ranges that their contraction is cut into.
int grouped_tile_side(const GroupedArgs& g, int what, int64_t& splits);

// The product of a few slots of 16 bits, whatever its operands' alignment, without a workspace.  Up
// to 32 slots (8 experts of 1024 x 2048, a slot each, weights in the last cache: 7.7 us, in tiles 23.5; 64
// slots of 64 of them 62 us and 45), and more where the weights would have to be copied for the tiles.
inline bool few_slots(const GroupedArgs& g, int dtype, bool w_fits) {
  return dtype != 0 && g.experts <= 512 && g.slots <= (w_fits ? 32 : 256);
}
int grouped_few(const GroupedArgs& g, int dtype, hipStream_t s, const char* name);

int grouped_f32(const GroupedArgs& g, int what, char* plan, hipStream_t s, const char* name);

}  // namespace hi2x
