// Products grouped by expert in float32: tiles of 64 x 64 on the float32 matrix unit.
#include "grouped.h"
#include "mfma_gemm.h"

namespace hi2x {
namespace {

// A workgroup's tile of 64 x 64 results, 32 of the contraction at a time through two LDS buffers:
// while one is multiplied the next chunk is on its way into registers.  A result is one chain of
// FMAs.  Lanes take neighbours in memory, along the contraction or across it, one value each, so
// rows may begin anywhere.  Offsets are 32 bits from a chunk's or a tile's first row.
constexpr int FT = 64;
constexpr uint32_t DEAD = 0x80000000u, SPAN = GROUPED_SPAN;

__device__ __forceinline__ float load_f32(__amdgpu_buffer_rsrc_t rs, uint32_t off) {
  return __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rs, (int)off, 0, 0));
}

// Neighbours along the contraction: lane c = tid % 32 of rows tid / 32 + 8 u.
struct AlongLoader {
  __amdgpu_buffer_rsrc_t rs;
  uint32_t row[8];
  int len;
  float v[8];
  static __device__ __forceinline__ int row_of(int u) { return (threadIdx.x >> 5) + 8 * u; }
  __device__ __forceinline__ void load(int k0) {
    const uint32_t c = k0 + (threadIdx.x & 31);
    const uint32_t at = c < (uint32_t)len ? 4 * c : SPAN;
#pragma unroll
    for (int u = 0; u < 8; ++u) v[u] = load_f32(rs, row[u] + at);
  }
  __device__ __forceinline__ void store(float (*S)[MG_RP]) const {
    const int c = threadIdx.x & 31;
#pragma unroll
    for (int u = 0; u < 8; ++u) S[row_of(u)][(c & 1) * MG_KP + (c >> 1)] = v[u];
  }
};

// Neighbours across it: lane i = tid % 64 of the contraction's rows tid / 64 + 4 u.
struct AcrossLoader {
  const char* base;  // of the tile's columns
  int64_t pitch;     // bytes
  int len;
  uint32_t col;      // this lane's column, dead past the last
  float v[8];
  static __device__ __forceinline__ int row_of(int u) { return (threadIdx.x >> 6) + 4 * u; }
  __device__ __forceinline__ void load(int k0) {
    const int left = len - k0 < MG_KC ? len - k0 : MG_KC;
    const __amdgpu_buffer_rsrc_t rs =
        rsrc(base + (int64_t)k0 * pitch, (left - 1) * pitch + FT * 4);
#pragma unroll
    for (int u = 0; u < 8; ++u)
      v[u] = load_f32(rs, row_of(u) < left ? (uint32_t)(row_of(u) * pitch) + col : DEAD);
  }
  __device__ __forceinline__ void store(float (*S)[MG_RP]) const {
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int c = row_of(u);
      S[threadIdx.x & 63][(c & 1) * MG_KP + (c >> 1)] = v[u];
    }
  }
};

// The same of rows that an index names.
struct IndexedLoader : AcrossLoader {
  const int64_t* index;
  __amdgpu_buffer_rsrc_t all;
  int64_t x_rows;
  __device__ __forceinline__ void load(int k0) {
    int64_t r[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int j = k0 + row_of(u);
      r[u] = index[j < len ? j : len - 1];
    }
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const bool live = k0 + row_of(u) < len, in = (uint64_t)r[u] < (uint64_t)x_rows;
      v[u] = load_f32(all, live && in ? (uint32_t)(r[u] * pitch) + col : DEAD);
      if (live && !in) v[u] = __builtin_nanf("");
    }
  }
};

template <class A, class B>
__device__ __forceinline__ void f32_loop(f32x16 (&acc)[1][1], MgSmemT<FT>& sm, A& a, B& b,
                                         int len) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int nch = (len + MG_KC - 1) / MG_KC;
  a.load(0);
  b.load(0);
  a.store(sm.A[0]);
  b.store(sm.B[0]);
  __syncthreads();
  for (int ch = 0; ch < nch; ++ch) {
    const int buf = ch & 1;
    const bool more = ch + 1 < nch;
    if (more) {
      a.load((ch + 1) * MG_KC);
      b.load((ch + 1) * MG_KC);
    }
    mg_chunk<1>(acc, sm.A[buf], sm.B[buf], wave >> 1, wave & 1, lane >> 5, lane & 31);
    __builtin_amdgcn_sched_barrier(0);
    if (more) {  // (the other buffer was last read before the barrier)
      a.store(sm.A[buf ^ 1]);
      b.store(sm.B[buf ^ 1]);
    }
    __syncthreads();
  }
}

template <int WHAT, bool INDEXED>
__global__ __launch_bounds__(256) void grouped_f32_kernel(GroupedArgs g, uint32_t nx,
                                                          uint32_t ny, const Plan* plan) {
  __shared__ __attribute__((aligned(16))) MgSmemT<FT> sm;
  const int n = (int)g.n, k = (int)g.k;
  float* const out = static_cast<float*>(g.out);
  f32x16 acc[1][1];
  mg_zero(acc);
  int64_t to;  // of the tile's first result
  int rows, cols, width;
  uint32_t bad = 0;  // rows of NaN, by accumulator register
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
        f32_loop(acc, sm, a, b, len);
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
    uint32_t xt;
    if (!plan_tile(plan, nx, blockIdx.x, w, xt)) return;
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
        for (int u = 0; u < 8; ++u) a.row[u] = row(a.row_of(u), in);
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          row(mg_row<FT>(0, j), in);
          bad |= in ? 0u : 1u << j;
        }
      } else {
        const int64_t ld = WHAT == GROUPED_LINEAR ? g.ldx : g.ldy;
        a.rs = rsrc(static_cast<const char*>(WHAT == GROUPED_LINEAR ? g.x : g.dy) +
                        w.first * ld * 4,
                    ((w.live - 1) * ld + a.len) * 4);
#pragma unroll
        for (int u = 0; u < 8; ++u)
          a.row[u] = a.row_of(u) < w.live ? (uint32_t)(a.row_of(u) * ld * 4) : DEAD;
      }
      const char* we = static_cast<const char*>(g.w) + (int64_t)w.e * n * g.ldw * 4;
      if constexpr (WHAT == GROUPED_LINEAR) {
        AlongLoader b;
        b.len = k;
        b.rs = rsrc(we + c0 * g.ldw * 4, ((cols - 1) * g.ldw + k) * 4);
#pragma unroll
        for (int u = 0; u < 8; ++u)
          b.row[u] = b.row_of(u) < cols ? (uint32_t)(b.row_of(u) * g.ldw * 4) : DEAD;
        f32_loop(acc, sm, a, b, k);
      } else {
        AcrossLoader b;
        b.base = we + c0 * 4;
        b.pitch = g.ldw * 4;
        b.len = n;
        b.col = (int)(threadIdx.x & 63) < cols ? 4 * (threadIdx.x & 63) : DEAD;
        f32_loop(acc, sm, a, b, n);
      }
    }
  }
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    const int r = mg_row<FT>(0, j), c = mg_col<FT>(0);
    if (r < rows && c < cols)
      out[to + (int64_t)r * width + c] = bad >> j & 1 ? __builtin_nanf("") : acc[0][0][j];
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
      <<<(unsigned)count, 256, 0, s>>>(g, (uint32_t)nx, (uint32_t)ny, p);
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
