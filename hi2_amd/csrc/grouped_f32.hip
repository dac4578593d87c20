// Products grouped by expert in float32: tiles of 64 x 64 on the float32 matrix unit.
#include "grouped.h"

namespace hi2x {
namespace {

// A workgroup's tile of 64 x 64 results, 32 of the contraction at a time through two LDS buffers:
// while one is multiplied the next two chunks are on their way into registers.  A wave has 16 rows and
// two fragments of 16 columns, and leaves out fragments and steps in which nothing lives, so that short
// ranges and odd sizes cost what they hold (60 experts of 520 x 1001, 3108 slots: 63 us, and 209 to 218
// with both gradients; 256 threads a tile and one chunk ahead took 229 where this took 212).  Lanes take
// neighbours in memory, along the contraction or across it, one value each, so rows may begin anywhere.
// Offsets are 32 bits from a chunk's or a tile's first row.
constexpr int FT = 64, KC = 32;
constexpr int THREADS = 512, EACH = FT * KC / THREADS;  // values of an operand's chunk a thread
constexpr int PITCH = KC + 4;  // floats of a row in LDS
struct Buffers {
  float a[2][FT][PITCH], b[2][FT][PITCH];
};
constexpr uint32_t DEAD = 0x80000000u, SPAN = GROUPED_SPAN;

__device__ __forceinline__ float load_f32(__amdgpu_buffer_rsrc_t rs, uint32_t off) {
  return __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rs, (int)off, 0, 0));
}

// Neighbours along the contraction: lane c = tid % 32 of rows tid / 32 + 16 u.
struct AlongLoader {
  __amdgpu_buffer_rsrc_t rs;
  uint32_t row[EACH];
  int len;
  static __device__ __forceinline__ int row_of(int u) { return (threadIdx.x >> 5) + 16 * u; }
  __device__ __forceinline__ void load(int k0, float (&v)[EACH]) const {
    const uint32_t c = k0 + (threadIdx.x & 31);
    const uint32_t at = c < (uint32_t)len ? 4 * c : SPAN;
#pragma unroll
    for (int u = 0; u < EACH; ++u) v[u] = load_f32(rs, row[u] + at);
  }
  static __device__ __forceinline__ void store(float (*S)[PITCH], const float (&v)[EACH]) {
#pragma unroll
    for (int u = 0; u < EACH; ++u) S[row_of(u)][threadIdx.x & 31] = v[u];
  }
};

// Neighbours across it: lane i = tid % 64 of the contraction's rows tid / 64 + 8 u.
struct AcrossLoader {
  const char* base;  // of the tile's columns
  int64_t pitch;     // bytes
  int len;
  uint32_t col;      // this lane's column, dead past the last
  static __device__ __forceinline__ int row_of(int u) { return (threadIdx.x >> 6) + 8 * u; }
  __device__ __forceinline__ void load(int k0, float (&v)[EACH]) const {
    const int left = len - k0 < KC ? len - k0 : KC;
    const __amdgpu_buffer_rsrc_t rs =
        rsrc(base + (int64_t)k0 * pitch, (left - 1) * pitch + FT * 4);
#pragma unroll
    for (int u = 0; u < EACH; ++u)
      v[u] = load_f32(rs, row_of(u) < left ? (uint32_t)(row_of(u) * pitch) + col : DEAD);
  }
  static __device__ __forceinline__ void store(float (*S)[PITCH], const float (&v)[EACH]) {
#pragma unroll
    for (int u = 0; u < EACH; ++u) S[threadIdx.x & 63][row_of(u)] = v[u];
  }
};

// The same of rows that an index names.
struct IndexedLoader : AcrossLoader {
  const int64_t* index;
  __amdgpu_buffer_rsrc_t all;
  int64_t x_rows;
  __device__ __forceinline__ void load(int k0, float (&v)[EACH]) const {
    int64_t r[EACH];
#pragma unroll
    for (int u = 0; u < EACH; ++u) {
      const int j = k0 + row_of(u);
      r[u] = index[j < len ? j : len - 1];
    }
#pragma unroll
    for (int u = 0; u < EACH; ++u) {
      const bool live = k0 + row_of(u) < len, in = (uint64_t)r[u] < (uint64_t)x_rows;
      v[u] = load_f32(all, live && in ? (uint32_t)(r[u] * pitch) + col : DEAD);
      if (live && !in) v[u] = __builtin_nanf("");
    }
  }
};

// A chunk's products for F fragments of columns: all operands are read before the first product, and
// neighbouring products are of different sums.
template <int F>
__device__ __forceinline__ void chunk_products(f32x4v (&acc)[2], const float* xs, const float* ys,
                                               int left) {
  f32x4v x[KC / 16], y[KC / 16][F];
#pragma unroll
  for (int h = 0; h < KC / 16; ++h) {
    x[h] = *reinterpret_cast<const f32x4v*>(xs + 16 * h);
#pragma unroll
    for (int f = 0; f < F; ++f)
      y[h][f] = *reinterpret_cast<const f32x4v*>(ys + 16 * f * PITCH + 16 * h);
  }
#pragma unroll
  for (int h = 0; h < KC / 16; ++h) {
    if (16 * h >= left) break;
#pragma unroll
    for (int s = 0; s < 4; ++s)
#pragma unroll
      for (int f = 0; f < F; ++f)
        acc[f] = __builtin_amdgcn_mfma_f32_16x16x4f32(x[h][s], y[h][f][s], acc[f], 0, 0, 0);
  }
}

// acc += A B^T over `len` of the contraction, for `rows` x `cols` results that live.  Of 16 values of
// the contraction lane group q = lane / 16 has 4 q .. 4 q + 3, one to each of four steps.  A running
// sum takes 256 of them and is added to the others': 6408 products in one were off by 1.4e-6 of the norm,
// so by 2.9e-7, for the 4 to 5 % that eight more registers a lane cost.
template <class A, class B>
__device__ __forceinline__ void f32_loop(f32x4v (&acc)[2], Buffers& sm, A& a, B& b, int len,
                                         int rows, int cols) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int i = lane & 15, q = lane >> 4;
  const int nch = (len + KC - 1) / KC;
  const int wr = 16 * (wave & 3), wc = 32 * (wave >> 2);
  const int frags = wr < rows ? (cols - wc + 15) / 16 : 0;
  float va[2][EACH], vb[2][EACH];
  a.load(0, va[0]);
  b.load(0, vb[0]);
  if (nch > 1) {
    a.load(KC, va[1]);
    b.load(KC, vb[1]);
  }
  a.store(sm.a[0], va[0]);
  b.store(sm.b[0], vb[0]);
  __syncthreads();
  // chunk ch in its buffer, the next in the other set of registers, the one behind it asked for
  auto chunk = [&](int ch, int buf, float (&fa)[EACH], float (&fb)[EACH],
                   const float (&na)[EACH], const float (&nb)[EACH]) {
    if (ch + 2 < nch) {
      a.load((ch + 2) * KC, fa);
      b.load((ch + 2) * KC, fb);
    }
    const int left = len - ch * KC;
    const float* xs = &sm.a[buf][wr + i][4 * q];
    const float* ys = &sm.b[buf][wc + i][4 * q];
    if (frags >= 2)
      chunk_products<2>(acc, xs, ys, left);
    else if (frags == 1)
      chunk_products<1>(acc, xs, ys, left);
    __builtin_amdgcn_sched_barrier(0);
    if (ch + 1 < nch) {  // (the other buffer was last read before the barrier)
      a.store(sm.a[buf ^ 1], na);
      b.store(sm.b[buf ^ 1], nb);
    }
    __syncthreads();
  };
  constexpr int BLOCK = 256 / KC;
  f32x4v total[2] = {acc[0], acc[1]};
  for (int first = 0; first < nch; first += BLOCK) {
    acc[0] = acc[1] = f32x4v{0.0f, 0.0f, 0.0f, 0.0f};
    const int end = nch - first < BLOCK ? nch : first + BLOCK;
    for (int ch = first; ch < end; ch += 2) {
      chunk(ch, 0, va[0], vb[0], va[1], vb[1]);
      if (ch + 1 < nch) chunk(ch + 1, 1, va[1], vb[1], va[0], vb[0]);
    }
    total[0] += acc[0], total[1] += acc[1];
  }
  acc[0] = total[0], acc[1] = total[1];
}

template <int WHAT, bool INDEXED>
__global__ __launch_bounds__(THREADS) void grouped_f32_kernel(GroupedArgs g, uint32_t nx,
                                                          uint32_t ny, const Plan* plan) {
  __shared__ __attribute__((aligned(16))) Buffers sm;
  const int n = (int)g.n, k = (int)g.k;
  float* const out = static_cast<float*>(g.out);
  f32x4v acc[2];
#pragma unroll
  for (int f = 0; f < 2; ++f) acc[f] = f32x4v{0.0f, 0.0f, 0.0f, 0.0f};
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int row0 = 16 * (wave & 3) + 4 * (lane >> 4), col0 = 32 * (wave >> 2) + (lane & 15);
  int64_t to;  // of the tile's first result
  int rows, cols, width;
  uint32_t bad = 0;  // rows of NaN among this lane's four
  if constexpr (WHAT == GROUPED_GRAD_W) {
    const uint32_t tiles = nx * ny;
    const int e = (int)(blockIdx.x / tiles), t = (int)(blockIdx.x - e * tiles);
    const int r0 = t / (int)nx * FT, c0 = t % (int)nx * FT;
    int64_t first, end;
    slot_range(g, e, first, end);
    const int len = (int)(end - first);
    rows = n - r0 < FT ? n - r0 : FT;
    cols = k - c0 < FT ? k - c0 : FT;
    width = k;
    to = ((int64_t)e * n + r0) * k + c0;
    if (len > 0) {
      const int i = threadIdx.x & 63;
      AcrossLoader a;
      a.base = static_cast<const char*>(g.dy) + (first * g.ldy + r0) * 4;
      a.pitch = g.ldy * 4;
      a.len = len;
      a.col = i < rows ? 4 * i : DEAD;
      auto finish = [&](auto& b) {
        b.pitch = g.ldx * 4;
        b.len = len;
        b.col = i < cols ? 4 * i : DEAD;
        f32_loop(acc, sm, a, b, len, rows, cols);
      };
      if constexpr (INDEXED) {
        IndexedLoader b;
        b.index = g.rows + first;
        b.x_rows = g.x_rows;
        b.all = rsrc(static_cast<const char*>(g.x) + c0 * 4,
                     g.x_rows > 0 ? ((g.x_rows - 1) * g.ldx + cols) * 4 : 0);
        finish(b);
      } else {
        AcrossLoader b;
        b.base = static_cast<const char*>(g.x) + (first * g.ldx + c0) * 4;
        finish(b);
      }
    }
  } else {
    RowTile w;
    uint32_t xt, y;
    if (!plan_tile(plan, nx, blockIdx.x, w, xt, y)) return;
    width = WHAT == GROUPED_LINEAR ? n : k;
    const int c0 = (int)xt * FT;
    rows = w.live;
    cols = width - c0 < FT ? width - c0 : FT;
    to = w.first * width + c0;
    if (w.e >= 0) {
      AlongLoader a;
      a.len = WHAT == GROUPED_LINEAR ? k : n;
      if constexpr (WHAT == GROUPED_LINEAR && INDEXED) {
        a.rs = rsrc(g.x, g.x_rows > 0 ? ((g.x_rows - 1) * g.ldx + k) * 4 : 0);
        auto row = [&](int t, bool& in) {
          const uint64_t r = t < w.live ? (uint64_t)g.rows[w.first + t] : 0;
          in = t >= w.live || r < (uint64_t)g.x_rows;
          return t < w.live && in ? (uint32_t)(r * g.ldx * 4) : DEAD;
        };
        bool in;
#pragma unroll
        for (int u = 0; u < EACH; ++u) a.row[u] = row(a.row_of(u), in);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          row(row0 + j, in);
          bad |= in ? 0u : 1u << j;
        }
      } else {
        const int64_t ld = WHAT == GROUPED_LINEAR ? g.ldx : g.ldy;
        a.rs = rsrc(static_cast<const char*>(WHAT == GROUPED_LINEAR ? g.x : g.dy) +
                        w.first * ld * 4,
                    ((w.live - 1) * ld + a.len) * 4);
#pragma unroll
        for (int u = 0; u < EACH; ++u)
          a.row[u] = a.row_of(u) < w.live ? (uint32_t)(a.row_of(u) * ld * 4) : DEAD;
      }
      const char* we = static_cast<const char*>(g.w) + (int64_t)w.e * n * g.ldw * 4;
      if constexpr (WHAT == GROUPED_LINEAR) {
        AlongLoader b;
        b.len = k;
        b.rs = rsrc(we + c0 * g.ldw * 4, ((cols - 1) * g.ldw + k) * 4);
#pragma unroll
        for (int u = 0; u < EACH; ++u)
          b.row[u] = b.row_of(u) < cols ? (uint32_t)(b.row_of(u) * g.ldw * 4) : DEAD;
        f32_loop(acc, sm, a, b, k, rows, cols);
      } else {
        AcrossLoader b;
        b.base = we + c0 * 4;
        b.pitch = g.ldw * 4;
        b.len = n;
        b.col = (int)(threadIdx.x & 63) < cols ? 4 * (threadIdx.x & 63) : DEAD;
        f32_loop(acc, sm, a, b, n, rows, cols);
      }
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int f = 0; f < 2; ++f) {
      const int r = row0 + j, c = col0 + 16 * f;
      if (r < rows && c < cols)
        out[to + (int64_t)r * width + c] = bad >> j & 1 ? __builtin_nanf("") : acc[f][j];
    }
}

template <int WHAT, bool INDEXED>
int launch(const GroupedArgs& g, char* plan, hipStream_t s, const char* name) {
  const int64_t nx = ((WHAT == GROUPED_LINEAR ? g.n : g.k) + FT - 1) / FT;
  const int64_t ny = WHAT == GROUPED_GRAD_W ? (g.n + FT - 1) / FT : most_tiles(g, FT);
  const int64_t count = WHAT == GROUPED_GRAD_W ? nx * ny * g.experts : (nx * ny + 7) / 8 * 8;
  Plan* const p = reinterpret_cast<Plan*>(plan);
  if constexpr (WHAT != GROUPED_GRAD_W) {
    if (int rc = launch_plan(g, FT, p, s, name)) return rc;
  }
  grouped_f32_kernel<WHAT, INDEXED>
      <<<(unsigned)count, THREADS, 0, s>>>(g, (uint32_t)nx, (uint32_t)ny, p);
  return launch_status(name);
}

}  // namespace

int grouped_f32(const GroupedArgs& g, int what, char* plan, hipStream_t s, const char* name) {
  if (what == GROUPED_GRAD_X) return launch<GROUPED_GRAD_X, false>(g, plan, s, name);
  if (what == GROUPED_LINEAR)
    return g.rows ? launch<GROUPED_LINEAR, true>(g, plan, s, name)
                  : launch<GROUPED_LINEAR, false>(g, plan, s, name);
  return g.rows ? launch<GROUPED_GRAD_W, true>(g, plan, s, name)
                : launch<GROUPED_GRAD_W, false>(g, plan, s, name);
}

}  // namespace hi2x
