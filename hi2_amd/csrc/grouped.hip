// Products grouped by expert with ragged sizes, and their gradients: out = x[rows] w^T over the
// routed slots, dx = dy w and dw = dy^T x[rows].  This file: the entries, and what surrounds the
// products (grouped_tile.hip, grouped_f32.hip).
#include "grouped.h"

namespace hi2x {
namespace {

int64_t size_of(int dtype) { return dtype == 0 ? 4 : 2; }

// Threads over rows of `pieces`: 1 << shift along a row, 256 >> shift rows a workgroup.
struct Spread {
  uint32_t across;  // workgroups along a row
  int shift;
};
int64_t spread(int64_t rows, int64_t pieces, Spread& g) {
  g.shift = 8;
  while (g.shift > 0 && (1ll << (g.shift - 1)) >= pieces) --g.shift;
  g.across = (uint32_t)((pieces + (1ll << g.shift) - 1) >> g.shift);
  return g.across * ((rows + (256 >> g.shift) - 1) / (256 >> g.shift));
}
__device__ __forceinline__ void spread_at(const Spread& g, int64_t& row, int64_t& piece) {
  const uint32_t band = blockIdx.x / g.across, x = blockIdx.x - band * g.across;
  row = (int64_t)band * (256 >> g.shift) + (threadIdx.x >> g.shift);
  piece = ((int64_t)x << g.shift) + (threadIdx.x & ((1 << g.shift) - 1));
}

// ---- a token's sum over its slots -------------------------------------------------------------
// dx[t] = the rows of t's slots added in their order, V values a thread (4, 16 bytes of a row; 1 where rows
// do not begin at multiples of 16 bytes), up to four rows on their way at a time.  A slot outside gives
// NaN.  Rows are float32 whatever dx's type: rounded to 16 bits before they are added they would cost
// half the traffic and 1.4 times the error.  HBM bounds it: part is read once (16384 tokens of eight slots
// of 2048 208 us, 5.5 TB/s).
template <int DT, int V>
__global__ __launch_bounds__(256) void sum_slots_kernel(const float* part, int64_t slots, int64_t k,
                                                        const int64_t* slots_of, int64_t t,
                                                        int top_k, Spread by, void* out) {
  int64_t token, c;
  spread_at(by, token, c);
  c *= V;
  if (token >= t || c >= k) return;
  const int64_t* of = slots_of + token * top_k;
  float acc[V];
#pragma unroll
  for (int i = 0; i < V; ++i) acc[i] = 0.0f;
  constexpr int UN = 4;
  for (int j0 = 0; j0 < top_k; j0 += UN) {
    int64_t s[UN];
    f32x4v w[UN];
#pragma unroll
    for (int u = 0; u < UN; ++u) s[u] = of[j0 + u < top_k ? j0 + u : top_k - 1];
#pragma unroll
    for (int u = 0; u < UN; ++u) {
      const int64_t r = (uint64_t)s[u] < (uint64_t)slots ? s[u] : 0;
      w[u] = f32x4v{0.0f, 0.0f, 0.0f, 0.0f};
      if (slots == 0) continue;  // (no row to read in the place of one outside)
      if constexpr (V == 1)
        w[u][0] = part[r * k + c];
      else
        w[u] = *reinterpret_cast<const f32x4v*>(part + r * k + c);
    }
#pragma unroll
    for (int u = 0; u < UN; ++u) {
      if (j0 + u >= top_k) break;
      const bool in = (uint64_t)s[u] < (uint64_t)slots;
#pragma unroll
      for (int i = 0; i < V; ++i) acc[i] += in ? w[u][i] : __builtin_nanf("");
    }
  }
  if constexpr (V == 4 && DT != 0) {
    u32x2 w;
#pragma unroll
    for (int i = 0; i < 2; ++i)
      w[i] = DT == 1 ? (uint32_t)f16_bits(acc[2 * i]) | (uint32_t)f16_bits(acc[2 * i + 1]) << 16
                     : (uint32_t)bf16_bits(acc[2 * i]) | (uint32_t)bf16_bits(acc[2 * i + 1]) << 16;
    *reinterpret_cast<u32x2*>(static_cast<uint16_t*>(out) + token * k + c) = w;
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) store_from_f32(out, token * k + c + i, DT, acc[i]);
  }
}

template <int DT>
int sum_slots(const void* part, int64_t slots, int64_t k, const int64_t* slots_of, int64_t t,
              int64_t top_k, void* out, hipStream_t s) {
  const bool wide = k % 4 == 0 && ((uintptr_t)out & 15) == 0;
  const float* p = static_cast<const float*>(part);
  Spread by;
  const int64_t count = spread(t, wide ? k / 4 : k, by);
  HI2X_REQUIRE(count < (1ll << 31), "grouped_grad_x: too many results");
  if (wide)
    sum_slots_kernel<DT, 4><<<(unsigned)count, 256, 0, s>>>(p, slots, k, slots_of, t, (int)top_k, by,
                                                            out);
  else
    sum_slots_kernel<DT, 1><<<(unsigned)count, 256, 0, s>>>(p, slots, k, slots_of, t, (int)top_k, by,
                                                            out);
  return launch_status("grouped_grad_x");
}

// ---- operands that do not lie as the tiles take them -------------------------------------------
// Rows of `cols` 16-bit or 32-bit values copied to rows at multiples of 16 bytes, zeros behind them;
// with `index` the rows that it names (one outside: NaN), with `offs` those of experts that have
// slots, `per` rows each.  A thread writes 16 bytes, which it reads as words of 4: of 16-bit rows
// that begin between two words five of them, shifted.  (The fifth ends no further than the word
// that the row's last value is in.)
typedef uint32_t u32x4w __attribute__((ext_vector_type(4), aligned(4)));
template <class W>
__global__ __launch_bounds__(256) void copy_rows_kernel(const W* from, int64_t ld, int64_t rows,
                                                        int64_t cols, const int64_t* index,
                                                        int64_t from_rows, const int64_t* offs,
                                                        int64_t per, W nan, W* to, int64_t ld_to,
                                                        Spread by) {
  constexpr int V = 16 / sizeof(W);
  int64_t row, c;
  spread_at(by, row, c);
  c *= V;
  if (row >= rows || c >= ld_to) return;
  if (offs) {
    const int64_t e = row / per;
    if (offs[e + 1] <= offs[e]) return;
  }
  const int64_t r = index ? index[row] : row;
  const bool in = (uint64_t)r < (uint64_t)from_rows;
  const W* const at = from + r * ld + c;
  union {
    W v[V];
    u32x4 w;
  };
  if (in && c + V <= cols) {
    const uint32_t odd = sizeof(W) == 2 ? (uint32_t)((uintptr_t)at & 2) : 0;
    const char* base = reinterpret_cast<const char*>(at) - odd;
    w = *reinterpret_cast<const u32x4w*>(base);
    if (odd) {
      const uint32_t last = *reinterpret_cast<const uint32_t*>(base + 16);
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = w[i] >> 16 | (i < 3 ? w[i + 1] : last) << 16;
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = c + i < cols ? (in ? at[i] : nan) : (W)0;
  }
  *reinterpret_cast<u32x4*>(to + row * ld_to + c) = w;
}

int copy_rows(const void* from, int64_t ld, int64_t rows, int64_t cols, const int64_t* index,
              int64_t from_rows, const int64_t* offs, int64_t per, int dtype, void* to,
              int64_t ld_to, hipStream_t s, const char* what) {
  Spread by;
  const int64_t count = spread(rows, ld_to / (dtype == 0 ? 4 : 8), by);
  HI2X_REQUIRE(count < (1ll << 31), "%s: too many elements", what);
  if (count == 0) return HI2X_OK;
  if (dtype == 0)
    copy_rows_kernel<uint32_t><<<(unsigned)count, 256, 0, s>>>(
        static_cast<const uint32_t*>(from), ld, rows, cols, index, from_rows, offs, per,
        0x7fc00000u, static_cast<uint32_t*>(to), ld_to, by);
  else
    copy_rows_kernel<uint16_t><<<(unsigned)count, 256, 0, s>>>(
        static_cast<const uint16_t*>(from), ld, rows, cols, index, from_rows, offs, per,
        (uint16_t)(dtype == 1 ? 0x7e00 : 0x7fc0), static_cast<uint16_t*>(to), ld_to, by);
  return launch_status(what);
}

// ---- a product's workspace ----------------------------------------------------------------------
struct Space {
  int64_t part = 0, x = 0, dy = 0, w = 0, plan = 0, bytes = 0;
  bool has_part = false, has_x = false, has_dy = false, has_w = false;
  bool gather = false;  // the copy of x is in the slots' order
  int64_t ldx = 0, ldy = 0, ldw = 0;
};

int64_t pad8(int64_t n) { return (n + 7) / 8 * 8; }

// Which operands are copied, and where in the workspace what lies.  16-bit rows begin at multiples
// of 16 bytes, and those that run along the contraction end there (or in zeros).  Of x the rows are
// copied, or where these are beyond the reach of an index's offsets the slots'.
Space lay_out(const GroupedArgs& g, int what, int dtype, bool summed, bool x_fits, bool dy_fits,
              bool w_fits) {
  Space m;
  if (what == GROUPED_LINEAR && few_slots(g, dtype, w_fits)) return m;
  auto take = [&](int64_t n) {
    const int64_t a = m.bytes;
    m.bytes += align256(n);
    return a;
  };
  const int64_t size = size_of(dtype);
  GroupedArgs p = g;
  if (summed) m.has_part = true, m.part = take(g.slots * g.k * 4);
  if (what != GROUPED_GRAD_X) {
    const bool copied = dtype != 0 && (!x_fits || (what == GROUPED_LINEAR && g.k % 8));
    m.ldx = copied ? pad8(g.k) : g.ldx;
    m.gather = g.rows && g.x_rows * m.ldx * size > (int64_t)GROUPED_SPAN;
    if (m.gather) m.ldx = pad8(g.k), p.rows = nullptr;
    m.has_x = copied || m.gather;
    if (m.has_x) m.x = take((m.gather ? g.slots : g.x_rows) * m.ldx * size);
  }
  if (what != GROUPED_LINEAR && dtype != 0 &&
      (!dy_fits || (what == GROUPED_GRAD_X && g.n % 8)))
    m.has_dy = true, m.ldy = pad8(g.n), m.dy = take(g.slots * m.ldy * size);
  if (what != GROUPED_GRAD_W && dtype != 0 && !w_fits)
    m.has_w = true, m.ldw = pad8(g.k), m.w = take(g.experts * g.n * m.ldw * size);
  m.plan = take(grouped_plan_bytes(p, what, dtype));
  return m;
}

// How far the next row is does not count where there is one, but the tiles find by it where the rows end.
void one_row(GroupedArgs& g) {
  if (g.x_rows <= 1) g.ldx = g.k;
  if (g.slots <= 1) g.ldy = g.n;
}

bool lies_well(const void* p, int64_t ld) { return ((uintptr_t)p & 15) == 0 && ld % 8 == 0; }

int check_grouped(const GroupedArgs& g, int dtype, const char* what) {
  HI2X_REQUIRE(dtype >= 0 && dtype <= 2, "%s: dtype %d", what, dtype);
  HI2X_REQUIRE(g.experts >= 1 && g.experts <= 7000, "%s: %lld experts", what,
               (long long)g.experts);
  HI2X_REQUIRE(g.n >= 1 && g.k >= 1 && g.n < (1ll << 20) && g.k < (1ll << 20),
               "%s: weights of %lld x %lld", what, (long long)g.n, (long long)g.k);
  HI2X_REQUIRE(g.slots >= 0 && g.slots < (1ll << 31) && g.x_rows >= 0 && g.x_rows < (1ll << 31),
               "%s: bad rows", what);
  HI2X_REQUIRE((g.x_rows <= 1 || g.ldx < (1 << 21)) && (g.slots <= 1 || g.ldy < (1 << 21)),
               "%s: rows more than 2^21 elements apart", what);
  return HI2X_OK;
}

// The product, its operands copied first where they do not lie as it takes them.
int run(GroupedArgs g, int what, int dtype, bool summed, void* ws, int64_t ws_bytes, Workspace& w,
        void** part, hipStream_t s, const char* name) {
  one_row(g);
  // workgroups of the smallest tiles, whole rounds of them
  const int T = dtype ? 128 : 64;
  const int64_t nx = ((what == GROUPED_LINEAR ? g.n : g.k) + T - 1) / T + 3;
  const int64_t ny = what == GROUPED_GRAD_W ? g.experts * ((g.n + T - 1) / T + 1)
                                            : most_tiles(g, T) + 8;
  HI2X_REQUIRE(nx * ny < (1ll << 31), "%s: too many results", name);
  if (what == GROUPED_LINEAR && few_slots(g, dtype, lies_well(g.w, g.ldw)))
    return grouped_few(g, dtype, s, name);
  const Space m = lay_out(g, what, dtype, summed, lies_well(g.x, g.ldx), lies_well(g.dy, g.ldy),
                          lies_well(g.w, g.ldw));
  if (int rc = take_workspace(w, ws, ws_bytes, (size_t)m.bytes, s, name)) return rc;
  if (summed) g.out = *part = w.p + m.part, g.f32_out = true;
  if (m.has_x) {
    if (int rc = copy_rows(g.x, g.ldx, m.gather ? g.slots : g.x_rows, g.k,
                           m.gather ? g.rows : nullptr, g.x_rows, nullptr, 0, dtype, w.p + m.x,
                           m.ldx, s, name))
      return rc;
    g.x = w.p + m.x;
    g.ldx = m.ldx;
    if (m.gather) g.rows = nullptr, g.x_rows = g.slots;
  }
  if (m.has_dy) {
    if (int rc = copy_rows(g.dy, g.ldy, g.slots, g.n, nullptr, g.slots, nullptr, 0, dtype,
                           w.p + m.dy, m.ldy, s, name))
      return rc;
    g.dy = w.p + m.dy;
    g.ldy = m.ldy;
  }
  if (m.has_w) {
    if (int rc = copy_rows(g.w, g.ldw, g.experts * g.n, g.k, nullptr, g.experts * g.n, g.offs, g.n,
                           dtype, w.p + m.w, m.ldw, s, name))
      return rc;
    g.w = w.p + m.w;
    g.ldw = m.ldw;
  }
  return dtype == 0 ? grouped_f32(g, what, w.p + m.plan, s, name)
                    : grouped_tiles(g, what, dtype, w.p + m.plan, s, name);
}

}  // namespace
}  // namespace hi2x

using namespace hi2x;

extern "C" int64_t hi2x_grouped_workspace_bytes(int what, int dtype, int64_t tokens, int64_t ldx,
                                                int64_t experts, int64_t n, int64_t k,
                                                int64_t slots, int indexed, int first_aligned,
                                                int second_aligned) {
  GroupedArgs g{};
  g.experts = experts, g.n = n, g.k = k, g.slots = slots, g.x_rows = tokens, g.ldx = ldx;
  if (what == GROUPED_GRAD_W && slots == 0) g.x_rows = 0;  // (as in the call)
  if (what < 0 || what > 2 || check_grouped(g, dtype, "grouped_workspace_bytes")) return -1;
  const int64_t given = 0;  // (only whether there are rows counts)
  if (indexed && what != GROUPED_GRAD_X) g.rows = &given;
  one_row(g);
  const int x_aligned = what == GROUPED_LINEAR ? first_aligned : second_aligned;
  return lay_out(g, what, dtype, indexed && what == GROUPED_GRAD_X,
                 x_aligned && (tokens > 1 || k % 8 == 0), first_aligned && (slots > 1 || n % 8 == 0),
                 second_aligned)
      .bytes;
}

extern "C" int64_t hi2x_grouped_form(int what, int dtype, int64_t experts, int64_t n, int64_t k,
                                     int64_t slots, int64_t* splits) {
  GroupedArgs g{};
  g.experts = experts, g.n = n, g.k = k, g.slots = slots, g.x_rows = slots;
  if (what < 0 || what > 2 || check_grouped(g, dtype, "grouped_form")) return -1;
  int64_t ranges = 1, side = 64;
  if (what == GROUPED_LINEAR && few_slots(g, dtype, k % 8 == 0))
    side = 16;
  else if (dtype != 0)
    side = grouped_tile_side(g, what, ranges);
  if (splits) *splits = ranges;
  return side;
}

extern "C" int hi2x_grouped_linear(const void* x, int dtype, int64_t ldx, int64_t x_rows,
                                   const void* w, int64_t experts, int64_t n, int64_t k,
                                   const int64_t* rows, const int64_t* offs, int64_t slots,
                                   void* out, void* ws, int64_t ws_bytes, void* stream) {
  clear_error();
  GroupedArgs g{};
  g.x = x, g.ldx = ldx, g.x_rows = x_rows, g.w = w, g.ldw = k;
  g.experts = experts, g.n = n, g.k = k, g.rows = rows, g.offs = offs, g.slots = slots, g.out = out;
  if (int rc = check_grouped(g, dtype, "grouped_linear")) return rc;
  HI2X_REQUIRE(rows || x_rows == slots || slots == 0, "grouped_linear: %lld rows for %lld slots",
               (long long)x_rows, (long long)slots);
  HI2X_REQUIRE(x_rows <= 1 || ldx >= k, "grouped_linear: rows of x overlap");
  if (slots == 0) return HI2X_OK;
  HI2X_REQUIRE((x || x_rows == 0) && w && offs && out, "grouped_linear: null buffer");
  Workspace space;
  return run(g, GROUPED_LINEAR, dtype, false, ws, ws_bytes, space, nullptr, as_stream(stream),
             "grouped_linear");
}

extern "C" int hi2x_grouped_grad_x(const void* dy, int dtype, int64_t ldy, const void* w,
                                   int64_t experts, int64_t n, int64_t k, const int64_t* offs,
                                   int64_t slots, const int64_t* slots_of, int64_t t,
                                   int64_t top_k, void* dx, void* ws, int64_t ws_bytes,
                                   void* stream) {
  clear_error();
  GroupedArgs g{};
  g.dy = dy, g.ldy = ldy, g.w = w, g.ldw = k, g.experts = experts, g.n = n, g.k = k;
  g.offs = offs, g.slots = slots, g.out = dx, g.x_rows = slots_of ? t : slots;
  if (int rc = check_grouped(g, dtype, "grouped_grad_x")) return rc;
  HI2X_REQUIRE(!slots_of || (t >= 0 && top_k >= 1 && top_k < (1 << 20)),
               "grouped_grad_x: bad routing");
  HI2X_REQUIRE(slots <= 1 || ldy >= n, "grouped_grad_x: rows of dy overlap");
  if (slots_of ? t == 0 : slots == 0) return HI2X_OK;
  HI2X_REQUIRE((dy || slots == 0) && w && offs && dx, "grouped_grad_x: null buffer");
  const hipStream_t s = as_stream(stream);
  Workspace space;
  void* part = dx;
  if (slots)
    if (int rc = run(g, GROUPED_GRAD_X, dtype, slots_of != nullptr, ws, ws_bytes, space, &part, s,
                     "grouped_grad_x"))
      return rc;
  if (!slots_of) return HI2X_OK;
  return dtype == 0   ? sum_slots<0>(part, slots, k, slots_of, t, top_k, dx, s)
         : dtype == 1 ? sum_slots<1>(part, slots, k, slots_of, t, top_k, dx, s)
                      : sum_slots<2>(part, slots, k, slots_of, t, top_k, dx, s);
}

extern "C" int hi2x_grouped_grad_w(const void* dy, int dtype, int64_t ldy, const void* x,
                                   int64_t ldx, int64_t x_rows, int64_t experts, int64_t n,
                                   int64_t k, const int64_t* rows, const int64_t* offs,
                                   int64_t slots, void* dw, void* ws, int64_t ws_bytes,
                                   void* stream) {
  clear_error();
  GroupedArgs g{};
  g.dy = dy, g.ldy = ldy, g.x = x, g.ldx = ldx, g.x_rows = x_rows;
  g.experts = experts, g.n = n, g.k = k, g.rows = rows, g.offs = offs, g.slots = slots;
  g.out = dw;
  if (int rc = check_grouped(g, dtype, "grouped_grad_w")) return rc;
  // (where there are no slots, rows may be NULL as the address of an empty array is)
  HI2X_REQUIRE(rows || x_rows == slots || slots == 0, "grouped_grad_w: %lld rows for %lld slots",
               (long long)x_rows, (long long)slots);
  HI2X_REQUIRE((x_rows <= 1 || ldx >= k) && (slots <= 1 || ldy >= n),
               "grouped_grad_w: rows overlap");
  HI2X_REQUIRE(((x || x_rows == 0) && dy || slots == 0) && offs && dw,
               "grouped_grad_w: null buffer");
  if (slots == 0) g.x_rows = 0, g.rows = nullptr;  // no row of x is read
  Workspace space;
  return run(g, GROUPED_GRAD_W, dtype, false, ws, ws_bytes, space, nullptr, as_stream(stream),
             "grouped_grad_w");
}
