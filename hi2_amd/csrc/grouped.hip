// Products grouped by expert with ragged sizes, and their gradients: out = x[rows] w^T over the
// routed slots, dx = dy w and dw = dy^T x[rows].
#include "grouped.h"

#include "mfma_gemm.h"

namespace hi2x {
namespace {

// ---- any type, any alignment: float32 MFMA ----------------------------------------------------
// A workgroup's tile of 64 x 64 results, 32 of the contraction at a time through LDS, where
// values are float32 (16-bit ones exactly); the sum of each result is a chain of FMAs.
constexpr int FT = 64;

template <int DT, bool ALONG>
struct TileLoader {
  float v[8];
  // Element (i, c) of the operand: ALONG, neighbours in c are neighbours in memory, else in i.
  template <class At>
  __device__ __forceinline__ void load(At at) {
    const int tid = threadIdx.x;
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int i = ALONG ? (tid >> 5) + 8 * u : tid & 63;
      const int c = ALONG ? tid & 31 : (tid >> 6) + 4 * u;
      v[u] = at(i, c);
    }
  }
  __device__ __forceinline__ void store(float (*S)[MG_RP]) const {
    const int tid = threadIdx.x;
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int i = ALONG ? (tid >> 5) + 8 * u : tid & 63;
      const int c = ALONG ? tid & 31 : (tid >> 6) + 4 * u;
      S[i][(c & 1) * MG_KP + (c >> 1)] = v[u];
    }
  }
};

template <int DT, int WHAT>
__global__ __launch_bounds__(256) void grouped_any_kernel(GroupedArgs g, uint32_t nx) {
  __shared__ __attribute__((aligned(16))) MgSmemT<FT> sm;
  __shared__ int64_t src[2][FT];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const uint32_t work = blockIdx.x / nx, xt = blockIdx.x - work * nx;
  int e;
  int64_t first, end, r0, rows_out;
  if constexpr (WHAT == GROUPED_GRAD_W) {
    const uint32_t ny = (uint32_t)((g.n + FT - 1) / FT);
    e = (int)(work / ny);
    r0 = (int64_t)(work - e * ny) * FT;
    rows_out = g.n;
    slot_range(g, e, first, end);
  } else {
    const GroupedWork w = find_rows(g, FT, work);
    if (w.e == WORK_NONE) return;
    e = w.e;
    r0 = first = w.first;
    end = rows_out = w.end;
  }
  const int64_t c0 = (int64_t)xt * FT;
  const int64_t cols = WHAT == GROUPED_LINEAR ? g.n : g.k;
  const int64_t len = WHAT == GROUPED_LINEAR ? g.k : (WHAT == GROUPED_GRAD_X ? g.n : end - first);
  f32x16 acc[1][1];
  mg_zero(acc);
  // row of x of slot first + i; -1: none, -2: outside
  auto row_of = [&](int64_t slot) -> int64_t {
    if (slot >= end) return -1;
    if (!g.rows) return slot;
    const int64_t r = g.rows[slot];
    return r >= 0 && r < g.x_rows ? r : -2;
  };
  auto x_at = [&](int64_t r, int64_t c) -> float {
    if (r < 0) return r == -1 ? 0.0f : __builtin_nanf("");
    return c < g.k ? load_as_f32(g.x, r * g.ldx + c, DT) : 0.0f;
  };
  auto w_at = [&](int64_t n, int64_t k) -> float {
    return n < g.n && k < g.k ? load_as_f32(g.w, ((int64_t)e * g.n + n) * g.k + k, DT) : 0.0f;
  };
  auto dy_at = [&](int64_t slot, int64_t n) -> float {
    return slot < end && n < g.n ? load_as_f32(g.dy, slot * g.ldy + n, DT) : 0.0f;
  };
  const int nch = e < 0 ? 0 : (int)((len + MG_KC - 1) / MG_KC);
  if (WHAT == GROUPED_LINEAR) {
    if (tid < FT) src[0][tid] = row_of(first + tid);
    __syncthreads();
  }
  for (int ch = 0; ch < nch; ++ch) {
    const int64_t k0 = (int64_t)ch * MG_KC;
    if (WHAT == GROUPED_GRAD_W) {
      if (tid < MG_KC) src[ch & 1][tid] = row_of(first + k0 + tid);
      __syncthreads();
    }
    TileLoader<DT, WHAT != GROUPED_GRAD_W> a;
    TileLoader<DT, WHAT == GROUPED_LINEAR> b;
    if constexpr (WHAT == GROUPED_LINEAR) {
      a.load([&](int i, int c) { return x_at(src[0][i], k0 + c); });
      b.load([&](int i, int c) { return w_at(c0 + i, k0 + c); });
    } else if constexpr (WHAT == GROUPED_GRAD_X) {
      a.load([&](int i, int c) { return dy_at(r0 + i, k0 + c); });
      b.load([&](int i, int c) { return w_at(k0 + c, c0 + i); });
    } else {
      a.load([&](int i, int c) { return dy_at(first + k0 + c, r0 + i); });
      b.load([&](int i, int c) { return x_at(src[ch & 1][c], c0 + i); });
    }
    __syncthreads();  // the chunk before has been read
    a.store(sm.A[0]);
    b.store(sm.B[0]);
    __syncthreads();
    mg_chunk<1>(acc, sm.A[0], sm.B[0], wave >> 1, wave & 1, lane >> 5, lane & 31);
  }
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    const int64_t r = r0 + mg_row<FT>(0, j), c = c0 + mg_col<FT>(0);
    if (r < rows_out && c < cols)
      store_from_f32(g.out, (WHAT == GROUPED_GRAD_W ? (int64_t)e * g.n + r : r) * cols + c, DT,
                     acc[0][0][j]);
  }
}

// dx[t] = the sum of its slots' rows, in their order; a wave (or more) on a token.
template <int DT>
__global__ __launch_bounds__(256) void sum_slots_kernel(const void* part, int64_t slots, int64_t k,
                                                        const int64_t* slots_of, int64_t t,
                                                        int top_k, void* out) {
  const int64_t token = blockIdx.x;
  const int64_t* of = slots_of + token * top_k;
  for (int64_t c = threadIdx.x; c < k; c += 256) {
    float acc = 0.0f;
    for (int j = 0; j < top_k; ++j) {
      const int64_t s = of[j];
      acc += s >= 0 && s < slots ? load_as_f32(part, s * k + c, DT) : __builtin_nanf("");
    }
    store_from_f32(out, token * k + c, DT, acc);
  }
}

template <int WHAT>
int launch_any(const GroupedArgs& g, int dtype, hipStream_t s, const char* what) {
  const int64_t cols = WHAT == GROUPED_LINEAR ? g.n : g.k;
  const int64_t nx = (cols + FT - 1) / FT;
  const int64_t ny = WHAT == GROUPED_GRAD_W ? g.experts * ((g.n + FT - 1) / FT)
                                            : g.slots / FT + g.experts + 2;
  HI2X_REQUIRE(nx < (1ll << 31) && ny < (1ll << 31) && nx * ny < (1ll << 31),
               "%s: too many results", what);
  const unsigned grid = (unsigned)(nx * ny);
  if (dtype == 0)
    grouped_any_kernel<0, WHAT><<<grid, 256, 0, s>>>(g, (uint32_t)nx);
  else if (dtype == 1)
    grouped_any_kernel<1, WHAT><<<grid, 256, 0, s>>>(g, (uint32_t)nx);
  else
    grouped_any_kernel<2, WHAT><<<grid, 256, 0, s>>>(g, (uint32_t)nx);
  return launch_status(what);
}

int check_grouped(const GroupedArgs& g, int dtype, const char* what) {
  HI2X_REQUIRE(dtype >= 0 && dtype <= 2, "%s: dtype %d", what, dtype);
  HI2X_REQUIRE(g.experts >= 1 && g.experts <= 7000, "%s: %lld experts", what,
               (long long)g.experts);
  HI2X_REQUIRE(g.n >= 1 && g.k >= 1 && g.n < (1ll << 20) && g.k < (1ll << 20),
               "%s: weights of %lld x %lld", what, (long long)g.n, (long long)g.k);
  HI2X_REQUIRE(g.slots >= 0 && g.slots < (1ll << 31) && g.x_rows >= 0 && g.x_rows < (1ll << 31),
               "%s: bad rows", what);
  return HI2X_OK;
}

int64_t size_of(int dtype) { return dtype == 0 ? 4 : 2; }

// Whether the product goes in tiles of 16-bit values: pieces of 16 bytes are whole.
bool in_tiles(const GroupedArgs& g, int what, int dtype) {
  auto whole = [](const void* p, int64_t ld) { return ((uintptr_t)p & 15) == 0 && ld % 8 == 0; };
  if (dtype == 0 || g.n % 8 || g.k % 8) return false;
  if (what != GROUPED_GRAD_W && !whole(g.w, g.k)) return false;
  if (what != GROUPED_LINEAR && (!whole(g.dy, g.ldy) || g.ldy >= (1 << 21))) return false;
  if (what != GROUPED_GRAD_X &&
      (!whole(g.x, g.ldx) || g.ldx >= (1 << 21) ||
       (g.rows && g.x_rows * g.ldx * 2 > (int64_t)GROUPED_SPAN)))
    return false;
  return true;
}

template <int WHAT>
int launch_product(const GroupedArgs& g, int dtype, hipStream_t s, const char* what) {
  return in_tiles(g, WHAT, dtype) ? grouped_tiles(g, WHAT, dtype, s, what)
                                  : launch_any<WHAT>(g, dtype, s, what);
}

}  // namespace
}  // namespace hi2x

using namespace hi2x;

extern "C" int64_t hi2x_grouped_workspace_bytes(int what, int dtype, int64_t tokens,
                                                int64_t experts, int64_t n, int64_t k,
                                                int64_t slots, int indexed, int first_aligned,
                                                int second_aligned) {
  GroupedArgs g{};
  g.experts = experts, g.n = n, g.k = k, g.slots = slots, g.x_rows = tokens;
  if (what < 0 || what > 2 || check_grouped(g, dtype, "grouped_workspace_bytes")) return -1;
  if (what == GROUPED_GRAD_X && indexed) return align256(slots * k * size_of(dtype));
  if (what == GROUPED_GRAD_W && indexed && dtype) return align256(grouped_offsets(slots) * 4);
  (void)first_aligned, (void)second_aligned;
  return 0;
}

extern "C" int hi2x_grouped_linear(const void* x, int dtype, int64_t ldx, int64_t x_rows,
                                   const void* w, int64_t experts, int64_t n, int64_t k,
                                   const int64_t* rows, const int64_t* offs, int64_t slots,
                                   void* out, void* ws, int64_t ws_bytes, void* stream) {
  clear_error();
  GroupedArgs g{};
  g.x = x, g.ldx = ldx, g.x_rows = x_rows, g.w = w, g.experts = experts, g.n = n, g.k = k;
  g.rows = rows, g.offs = offs, g.slots = slots, g.out = out;
  if (int rc = check_grouped(g, dtype, "grouped_linear")) return rc;
  HI2X_REQUIRE(rows || x_rows == slots, "grouped_linear: %lld rows for %lld slots",
               (long long)x_rows, (long long)slots);
  HI2X_REQUIRE(x_rows <= 1 || ldx >= k, "grouped_linear: rows of x overlap");
  if (slots == 0) return HI2X_OK;
  HI2X_REQUIRE((x || x_rows == 0) && w && offs && out, "grouped_linear: null buffer");
  return launch_product<GROUPED_LINEAR>(g, dtype, as_stream(stream), "grouped_linear");
}

extern "C" int hi2x_grouped_grad_x(const void* dy, int dtype, int64_t ldy, const void* w,
                                   int64_t experts, int64_t n, int64_t k, const int64_t* offs,
                                   int64_t slots, const int64_t* slots_of, int64_t t,
                                   int64_t top_k, void* dx, void* ws, int64_t ws_bytes,
                                   void* stream) {
  clear_error();
  GroupedArgs g{};
  g.dy = dy, g.ldy = ldy, g.w = w, g.experts = experts, g.n = n, g.k = k;
  g.offs = offs, g.slots = slots, g.out = dx, g.x_rows = slots_of ? t : slots;
  if (int rc = check_grouped(g, dtype, "grouped_grad_x")) return rc;
  HI2X_REQUIRE(!slots_of || (t >= 0 && top_k >= 1 && top_k < (1 << 20)),
               "grouped_grad_x: bad routing");
  HI2X_REQUIRE(slots <= 1 || ldy >= n, "grouped_grad_x: rows of dy overlap");
  if (slots_of ? t == 0 : slots == 0) return HI2X_OK;
  HI2X_REQUIRE((dy || slots == 0) && w && offs && dx, "grouped_grad_x: null buffer");
  const hipStream_t s = as_stream(stream);
  if (!slots_of) return launch_product<GROUPED_GRAD_X>(g, dtype, s, "grouped_grad_x");
  Workspace part;
  const size_t need = (size_t)align256(slots * k * size_of(dtype));
  if (int rc = take_workspace(part, ws, ws_bytes, need, s, "grouped_grad_x")) return rc;
  g.out = part.p;
  if (slots)
    if (int rc = launch_product<GROUPED_GRAD_X>(g, dtype, s, "grouped_grad_x")) return rc;
  if (dtype == 0)
    sum_slots_kernel<0><<<(unsigned)t, 256, 0, s>>>(part.p, slots, k, slots_of, t, (int)top_k, dx);
  else if (dtype == 1)
    sum_slots_kernel<1><<<(unsigned)t, 256, 0, s>>>(part.p, slots, k, slots_of, t, (int)top_k, dx);
  else
    sum_slots_kernel<2><<<(unsigned)t, 256, 0, s>>>(part.p, slots, k, slots_of, t, (int)top_k, dx);
  return launch_status("grouped_grad_x");
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
  HI2X_REQUIRE(rows || x_rows == slots, "grouped_grad_w: %lld rows for %lld slots",
               (long long)x_rows, (long long)slots);
  HI2X_REQUIRE((x_rows <= 1 || ldx >= k) && (slots <= 1 || ldy >= n),
               "grouped_grad_w: rows overlap");
  HI2X_REQUIRE(((x || x_rows == 0) && dy || slots == 0) && offs && dw,
               "grouped_grad_w: null buffer");
  const hipStream_t s = as_stream(stream);
  Workspace offsets;
  if (rows && in_tiles(g, GROUPED_GRAD_W, dtype)) {
    const size_t need = (size_t)align256(grouped_offsets(slots) * 4);
    if (int rc = take_workspace(offsets, ws, ws_bytes, need, s, "grouped_grad_w")) return rc;
    g.offsets = reinterpret_cast<uint32_t*>(offsets.p);
  }
  return launch_product<GROUPED_GRAD_W>(g, dtype, s, "grouped_grad_w");
}
