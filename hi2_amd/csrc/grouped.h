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
  int64_t experts, n, k;
  uint32_t* offsets;  // of the slots' rows in x, for grad_w in tiles
};

// Expert e's slots, empty where the ranges are not as they should be.
__device__ __forceinline__ void slot_range(const GroupedArgs& g, int e, int64_t& a, int64_t& b) {
  a = g.offs[e];
  b = g.offs[e + 1];
  a = a < 0 ? 0 : (a > g.slots ? g.slots : a);
  b = b < a ? a : (b > g.slots ? g.slots : b);
}

// A tile's rows: those of expert e from `first` up to its range's end, of no expert (zeros), or
// none.
constexpr int WORK_ZEROS = -1, WORK_NONE = -2;
struct GroupedWork {
  int e;
  int64_t first, end;
};

// The want-th tile of `tile` rows, expert after expert; then those of the slots behind the last
// range and before the first.  Called by all lanes of a wave together.
__device__ __forceinline__ GroupedWork find_rows(const GroupedArgs& g, int tile, int64_t want) {
  GroupedWork w{WORK_NONE, 0, 0};
  const int lane = threadIdx.x & 63;
  const int experts = (int)g.experts;
  int64_t before = 0;
  for (int e0 = 0; e0 < experts + 2; e0 += 64) {
    const int e = e0 + lane;
    int64_t a = 0, b = 0;
    if (e < experts) {
      slot_range(g, e, a, b);
    } else if (e == experts) {
      a = g.offs[experts];
      a = a < 0 ? 0 : (a > g.slots ? g.slots : a);
      b = g.slots;
    } else if (e == experts + 1) {
      b = g.offs[0];
      b = b < 0 ? 0 : (b > g.slots ? g.slots : b);
    }
    const int n = (int)((b - a + tile - 1) / tile);
    int inc = n;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int o = __shfl_up(inc, d);
      if (lane >= d) inc += o;
    }
    const int64_t upto = before + inc;
    const unsigned long long hit = __ballot(want < upto && want >= upto - n);
    if (hit) {
      const int l = __builtin_ctzll(hit);
      const int64_t base = before + __shfl(inc, l) - __shfl(n, l);
      w.e = e0 + l < experts ? e0 + l : WORK_ZEROS;
      w.first = __shfl(a, l) + (want - base) * tile;
      w.end = __shfl(b, l);
      return w;
    }
    before += __shfl(inc, 63);
  }
  return w;
}

// What a resource that offsets of 32 bits reach may span: an offset past it by this much again is
// past it still.
constexpr uint32_t GROUPED_SPAN = 0x7f000000u;

// The product in tiles (16 bits; rows and weights at multiples of 16 bytes, n and k of 8).
// grad_w with rows: g.offsets, room for grouped_offsets(slots) of them.
constexpr int64_t grouped_offsets(int64_t slots) { return slots + 256; }
int grouped_tiles(const GroupedArgs& g, int what, int dtype, hipStream_t s, const char* name);

}  // namespace hi2x
