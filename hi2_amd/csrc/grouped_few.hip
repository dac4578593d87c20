// The grouped product of a few slots in 16 bits: single tokens and small batches of them.  Bound by
// reading the experts' weights once: 8 slots of 8 of 64 experts of 1024 x 2048 8 to 10 us with the weights
// (33.6 MB) in the last cache, 16 us (2.1 TB/s) from memory, where a launch is over before the loads that
// wait for the slot's expert reach the memory's rate.
#include "grouped.h"

namespace hi2x {
namespace {

typedef __bf16 b16x8 __attribute__((ext_vector_type(8)));
typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));

constexpr int ROWS = 16;  // of w, and slots at most, of a workgroup
constexpr int UN = 8;     // steps of 32 columns of a wave in flight

// Columns k .. k + 7 of a row of `len`, zeros behind it.
template <bool WHOLE>
__device__ __forceinline__ u16x8 piece(const uint16_t* row, int k, int len) {
  if (k + 8 <= len) {
    u16x8 v;
    if constexpr (WHOLE)
      v = *reinterpret_cast<const u16x8*>(row + k);
    else
      __builtin_memcpy(&v, row + k, 16);
    return v;
  }
  u16x8 v = {0, 0, 0, 0, 0, 0, 0, 0};
  if constexpr (!WHOLE) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (k + i < len) v[i] = row[k + i];
  }
  return v;
}

template <int DT>
__device__ __forceinline__ f32x4v step_product(const u16x8& a, const u16x8& b, const f32x4v& c) {
  if constexpr (DT == 1)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h16x8, a),
                                                  __builtin_bit_cast(h16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b16x8, a),
                                                   __builtin_bit_cast(b16x8, b), c, 0, 0, 0);
}

// A workgroup to 16 rows of w (blockIdx.x) and one slot (blockIdx.y), which is the first of up to
// 16 of its expert's, or else goes to another workgroup.  The four waves take the columns' steps in
// turn, 256 bytes of a row at a time together, and their sums meet in LDS.  WHOLE: rows of x and w
// begin and end at multiples of 16 bytes.
template <int DT, bool WHOLE>
__global__ __launch_bounds__(256) void grouped_few_kernel(GroupedArgs g) {
  __shared__ __attribute__((aligned(16))) f32x4v sums[3][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t slot = blockIdx.y;
  const int n = (int)g.n, k = (int)g.k, r0 = (int)blockIdx.x * ROWS;
  uint16_t* const out = static_cast<uint16_t*>(g.out);
  int e = -1;
  int64_t first = 0, end = 0;
  for (int e0 = 0; e0 < (int)g.experts && e < 0; e0 += 64) {
    int64_t a = 0, b = 0;
    if (e0 + lane < (int)g.experts) slot_range(g, e0 + lane, a, b);
    const unsigned long long hit = __ballot(a <= slot && slot < b);
    if (hit) {
      const int l = __builtin_ctzll(hit);
      e = e0 + l;
      first = __shfl(a, l);
      end = __shfl(b, l);
    }
  }
  if (e < 0) {
    if (threadIdx.x < ROWS && r0 + (int)threadIdx.x < n) out[slot * n + r0 + threadIdx.x] = 0;
    return;
  }
  if ((slot - first) % ROWS) return;
  e = __builtin_amdgcn_readfirstlane(e);
  const int live = __builtin_amdgcn_readfirstlane((int)(end - slot < ROWS ? end - slot : ROWS));
  const int i = lane & 15, q = lane >> 4;
  // this lane's row of w and of x; those that are not there read another's, and are not stored
  const int wr = r0 + i < n ? r0 + i : n - 1;
  const uint16_t* const w = static_cast<const uint16_t*>(g.w) + ((int64_t)e * n + wr) * k;
  const int64_t s = slot + (i < live ? i : 0);
  int64_t r = g.rows ? g.rows[s] : s;
  const bool in = (uint64_t)r < (uint64_t)g.x_rows;
  if (!in) r = 0;
  const uint16_t* const x = static_cast<const uint16_t*>(g.x) + r * g.ldx;
  const int reach = g.x_rows > 0 ? k : 0;  // (no rows of x: nothing to read)
  f32x4v acc = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int k0 = 32 * wave + 8 * q; k0 < k + 8 * q; k0 += 128 * UN) {
    u16x8 a[UN], b[UN];
#pragma unroll
    for (int u = 0; u < UN; ++u) a[u] = piece<WHOLE>(w, k0 + 128 * u, k);
#pragma unroll
    for (int u = 0; u < UN; ++u) b[u] = piece<WHOLE>(x, k0 + 128 * u, reach);
#pragma unroll
    for (int u = 0; u < UN; ++u) acc = step_product<DT>(a[u], b[u], acc);
  }
  if (wave) sums[wave - 1][lane] = acc;
  __syncthreads();
  if (wave) return;
#pragma unroll
  for (int u = 0; u < 3; ++u) acc += sums[u][lane];
  if (i >= live) return;
  uint16_t* const to = out + s * n + r0 + 4 * q;
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (r0 + 4 * q + j < n) store_from_f32(to, j, DT, in ? acc[j] : __builtin_nanf(""));
}

}  // namespace

int grouped_few(const GroupedArgs& g, int dtype, hipStream_t s, const char* name) {
  const bool whole = g.k % 8 == 0 && g.ldx % 8 == 0 &&
                     (((uintptr_t)g.x | (uintptr_t)g.w) & 15) == 0;
  const dim3 grid((unsigned)((g.n + ROWS - 1) / ROWS), (unsigned)g.slots);
#define HI2X_FEW(DT)                                  \
  if (whole)                                          \
    grouped_few_kernel<DT, true><<<grid, 256, 0, s>>>(g); \
  else                                                \
    grouped_few_kernel<DT, false><<<grid, 256, 0, s>>>(g)
  if (dtype == 1) {
    HI2X_FEW(1);
  } else {
    HI2X_FEW(2);
  }
#undef HI2X_FEW
  return launch_status(name);
}

}  // namespace hi2x
