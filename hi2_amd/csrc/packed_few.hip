// Products of few rows by packed tensors: single tokens, small batches of them, and the
// experts' products of a decode step.  Bound by reading the packed weights once.
//
// A workgroup of 8 waves takes FR fragments (16 FR rows of the tensor) and up to 16 MF
// activation rows; the columns are split over the waves by chunks of 128, and the partial
// sums meet in LDS, so nothing is joined across workgroups.  A wave keeps D chunks of codes
// in flight (one 16-byte load a lane holds a fragment's whole chunk at 4 bits).
#include "packed.h"

namespace hi2x {
namespace {

constexpr int FW = 8;  // waves

struct FewArgs {
  GemmArgs g;
  // fused: the activations as they are, transformed here
  const void* x;
  int dtype;
  int64_t ldx, x_rows;
  const uint8_t* had;
  const uint16_t* cs;
  int per_expert;  // had and cs hold one transform per expert
  int npl;         // fp16 planes of the transformed activations
  int mt;          // activation rows of a workgroup
};

// The transform of a wave's own columns (chunks w, w + 8, ...) into LDS, one 16-column group
// of one row per lane and pass.  As in the separate pass (activations_kernel) each row is
// scaled by a power of two, here by the largest value among the wave's columns.  Row r of
// chunk i lies at (i R + r) 256 with its 16-byte pieces p at p ^ (r % 16); R = mt npl, the
// second plane's rows behind the first's.
__device__ __forceinline__ void few_transform(const FewArgs& a, int e, int64_t first, int live,
                                              int w, int nc, char* xl, uint32_t* mx,
                                              float* unscale) {
  const int lane = threadIdx.x & 63;
  const int k = (int)a.g.w.k;
  const int R = a.mt * a.npl;
  const uint8_t* had = a.had + (a.per_expert ? (int64_t)e * (k / 16) : 0);
  const uint16_t* cs = a.cs ? a.cs + (a.per_expert ? (int64_t)e * k : 0) : nullptr;
  const int total = nc * 8 * live;
  const int passes = (total + 63) / 64;
  if (lane < 16) mx[lane] = 0;
  float v[16];
  auto load = [&](int p, int& row, int& i, int& g) {
    const int j = p * 64 + lane;
    row = j / (nc * 8);
    const int rest = j - row * (nc * 8);
    i = rest >> 3;
    g = 8 * (w + FW * i) + (rest & 7);  // group of 16 columns
    const bool in = j < total;
    const int64_t src = in ? (a.g.src ? a.g.src[first + row] : first + row) : -1;
    if (src < 0 || src >= a.x_rows || 16 * g >= k) {
#pragma unroll
      for (int t = 0; t < 16; ++t) v[t] = 0.0f;
      return in;
    }
    load16(a.x, src * a.ldx + 16 * g, a.dtype, v);
    if (cs) {
#pragma unroll
      for (int t = 0; t < 16; ++t) v[t] = v[t] / f16_from_bits(cs[16 * g + t]);
    }
    return in;
  };
  int row, i, g;
  bool in = false;
  for (int p = 0; p < passes; ++p) {
    in = load(p, row, i, g);
    float m = 0.0f;
#pragma unroll
    for (int t = 0; t < 16; ++t) {
      const float b = fabsf(v[t]);
      m = fmaxf(m, b < __builtin_inff() ? b : 0.0f);
    }
    if (in && m > 0.0f) atomicMax(&mx[row], __float_as_uint(m));
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup", "local");  // the wave's own values
  if (lane < 16) {
    const float m = __uint_as_float(mx[lane]);
    int ex = 0;
    if (m > 0.0f) (void)frexpf(m, &ex);
    const int s = 13 - ex > 126 ? 126 : (13 - ex < -126 ? -126 : 13 - ex);
    mx[lane] = (uint32_t)s;
    bool bad = false;
    if (lane < live && a.g.src) {
      const int64_t src = a.g.src[first + lane];
      bad = src < 0 || src >= a.x_rows;
    }
    unscale[lane] = bad ? __builtin_nanf("") : ldexpf(1.0f, -s);
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup", "local");
  for (int p = 0; p < passes; ++p) {
    if (passes > 1) in = load(p, row, i, g);
    if (!in) continue;
    const float sc = ldexpf(1.0f, (int)mx[row]);
#pragma unroll
    for (int t = 0; t < 16; ++t) v[t] *= sc;
    if (16 * g < k && had[g]) {
#pragma unroll
      for (int d = 1; d < 16; d <<= 1)
#pragma unroll
        for (int t = 0; t < 16; ++t)
          if (!(t & d)) {
            const float x = v[t], y = v[t | d];
            v[t] = x + y;
            v[t | d] = x - y;
          }
#pragma unroll
      for (int t = 0; t < 16; ++t) v[t] *= 0.25f;
    }
    uint32_t h[8], l[8];
#pragma unroll
    for (int t = 0; t < 8; ++t) {
      const uint16_t x = f16_bits(v[2 * t]), y = f16_bits(v[2 * t + 1]);
      h[t] = (uint32_t)x | (uint32_t)y << 16;
      l[t] = (uint32_t)f16_bits(v[2 * t] - f16_from_bits(x)) |
             (uint32_t)f16_bits(v[2 * t + 1] - f16_from_bits(y)) << 16;
    }
    const int p0 = 2 * (g & 7);
    {
      char* d = xl + (i * R + row) * 256;
      *reinterpret_cast<u32x4*>(d + 16 * (p0 ^ (row & 15))) = u32x4{h[0], h[1], h[2], h[3]};
      *reinterpret_cast<u32x4*>(d + 16 * ((p0 + 1) ^ (row & 15))) = u32x4{h[4], h[5], h[6], h[7]};
    }
    if (a.npl == 2) {
      const int r = a.mt + row;
      char* d = xl + (i * R + r) * 256;
      *reinterpret_cast<u32x4*>(d + 16 * (p0 ^ (r & 15))) = u32x4{l[0], l[1], l[2], l[3]};
      *reinterpret_cast<u32x4*>(d + 16 * ((p0 + 1) ^ (r & 15))) = u32x4{l[4], l[5], l[6], l[7]};
    }
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup", "local");
}

template <int BITS, bool B16, int FR, int MF, bool FUSED>
__device__ __forceinline__ void few_loop(const FewArgs& a, const Tile& tile, int e, int64_t first,
                                         int live, char* xl, uint32_t* mx, float* unscale,
                                         f32x4v (&acc)[FR][MF]) {
  constexpr int D = FUSED ? (FR == 1 ? 4 : 2) : (FR * MF <= 2 ? 3 : 2);  // chunks in flight
  const GemmArgs& g = a.g;
  const int tid = threadIdx.x, lane = tid & 63, q = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int nch = (int)(g.w.kp / PK_CHUNK);
  const int nc = w < nch ? (nch - w + FW - 1) / FW : 0;
  const int64_t nblk = g.w.kp / tile.sg.block;
  const uint32_t cfrag = (uint32_t)nch * (256 * BITS), pfrag = (uint32_t)nblk * 64;
  const __amdgpu_buffer_rsrc_t cr =
      rsrc(static_cast<const char*>(g.w.codes) + tile.sg.codes + (int64_t)tile.first * cfrag,
           (int64_t)tile.count * cfrag);
  const __amdgpu_buffer_rsrc_t pr =
      rsrc(static_cast<const char*>(g.w.params) + tile.sg.params + (int64_t)tile.first * pfrag,
           (int64_t)tile.count * pfrag);
  const int bsh = tile.sg.block == 64 ? 6 : (tile.sg.block == 32 ? 5 : 4);
  const uint32_t poff = 64 * ((32 * q) >> bsh) + 4 * (lane & 15);
  uint32_t cw[D][FR][BITS], pw[D][FR][2];
  auto fetch = [&](int d, int i) {
    const int c = w + FW * i;
#pragma unroll
    for (int f = 0; f < FR; ++f) {
      load_codes<BITS>(cr, lane, f * cfrag + (uint32_t)c * (256 * BITS), cw[d][f]);
      const uint32_t so = f * pfrag + ((uint32_t)(c * PK_CHUNK) >> bsh) * 64;
      pw[d][f][0] = __builtin_amdgcn_raw_buffer_load_b32(pr, (int)poff, (int)so, 0);
      pw[d][f][1] = B16 ? __builtin_amdgcn_raw_buffer_load_b32(pr, (int)poff + 64, (int)so, 0) : 0u;
    }
  };
#pragma unroll
  for (int d = 0; d < D; ++d)
    if (d < nc) fetch(d, d);
  // where this lane's activation rows are
  const int col = lane & 15;
  const char* xrow = nullptr;
  int xr = 0, R = 0;
  uint32_t xoff[MF];
  __amdgpu_buffer_rsrc_t xs;
  int64_t plane = 0;
  if constexpr (FUSED) {
    few_transform(a, e, first, live, w, nc, xl, mx, unscale);
    R = a.mt * a.npl;
    xr = a.npl == 2 ? ((col & 7) < live ? (col >> 3) * a.mt + (col & 7) : 0)
                    : (col < live ? col : 0);
    xrow = xl + xr * 256;
  } else {
    const uint32_t pitch = (uint32_t)g.x.kp * 2;
    const int64_t row0 = g.src ? 0 : first;
    plane = g.x.rows * (int64_t)pitch;
    xs = rsrc(reinterpret_cast<const char*>(g.x.planes) + row0 * pitch,
              (g.x.rows - row0) * pitch);
#pragma unroll
    for (int m = 0; m < MF; ++m) {
      int64_t r = 16 * m + col < live ? 16 * m + col : 0;
      if (g.src) {
        r = g.src[first + r];
        if (r < 0 || r >= g.x.rows) r = 0;
      }
      xoff[m] = (uint32_t)r * pitch + 64 * q;
    }
  }
  const int npl = FUSED ? 1 : g.x.nplanes;
  for (int i0 = 0; i0 < nc; i0 += D) {
#pragma unroll
    for (int d = 0; d < D; ++d) {
      const int i = i0 + d;
      if (i < nc) {
        for (int pl = 0; pl < npl; ++pl) {
          h16x8 b[4][MF];
#pragma unroll
          for (int s = 0; s < 4; ++s)
#pragma unroll
            for (int m = 0; m < MF; ++m) {
              if constexpr (FUSED)
                b[s][m] = *reinterpret_cast<const h16x8*>(xrow + i * R * 256 +
                                                          16 * ((4 * q + s) ^ (xr & 15)));
              else
                b[s][m] = __builtin_bit_cast(
                    h16x8, __builtin_amdgcn_raw_buffer_load_b128(
                               pl ? rsrc(reinterpret_cast<const char*>(g.x.planes) + plane +
                                             (g.src ? 0 : first) * (int64_t)(g.x.kp * 2),
                                         (g.x.rows - (g.src ? 0 : first)) * (int64_t)(g.x.kp * 2))
                                  : xs,
                               (int)xoff[m] + 16 * s, (w + FW * i) * 256, 0));
            }
#pragma unroll
          for (int s = 0; s < 4; ++s)
#pragma unroll
            for (int f = 0; f < FR; ++f) {
              const h16x2 ls =
                  __builtin_bit_cast(h16x2, B16 && s >= 2 ? pw[d][f][1] : pw[d][f][0]);
              const h16x8 av =
                  decode_step<BITS>(cw[d][f], s, (h16x2){ls[0], ls[0]}, (h16x2){ls[1], ls[1]});
#pragma unroll
              for (int m = 0; m < MF; ++m)
                acc[f][m] = __builtin_amdgcn_mfma_f32_16x16x32_f16(av, b[s][m], acc[f][m], 0, 0, 0);
            }
        }
        if (i + D < nc) fetch(d, i + D);
      }
    }
  }
  if constexpr (FUSED) {
    const float u = unscale[a.npl == 2 ? col & 7 : col];
#pragma unroll
    for (int f = 0; f < FR; ++f)
#pragma unroll
      for (int t = 0; t < 4; ++t) acc[f][0][t] *= nc ? u : 1.0f;
  }
}

template <int FR, int MF, bool FUSED>
__global__ __launch_bounds__(64 * FW) void packed_few_kernel(FewArgs a) {
  extern __shared__ char lds[];
  __shared__ uint32_t mx[FW][16];
  __shared__ float unscale[FW][16];
  const GemmArgs& g = a.g;
  const PkWork wk = find_work(g.offs, (int)g.w.experts, g.slots, a.mt, blockIdx.y);
  const int e = __builtin_amdgcn_readfirstlane(wk.e);
  if (e < 0) return;
  Tile tile;
  if (!find_tile(g.w, e, blockIdx.x, FR, tile)) return;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int64_t first = __builtin_amdgcn_readfirstlane((int)wk.first);  // slots < 2^31
  const int64_t left = __builtin_amdgcn_readfirstlane((int)wk.end) - first;
  const int live = (int)(left < a.mt ? left : a.mt);
  f32x4v acc[FR][MF];
#pragma unroll
  for (int f = 0; f < FR; ++f)
#pragma unroll
    for (int m = 0; m < MF; ++m) acc[f][m] = f32x4v{0.0f, 0.0f, 0.0f, 0.0f};
  const int nch = (int)(g.w.kp / PK_CHUNK);
  char* xl = lds + (size_t)w * ((nch + FW - 1) / FW) * a.mt * a.npl * 256;
#define HI2X_FEW(BITS)                                                                     \
  if (tile.sg.block == 16)                                                                 \
    few_loop<BITS, true, FR, MF, FUSED>(a, tile, e, first, live, xl, mx[w], unscale[w], acc); \
  else                                                                                     \
    few_loop<BITS, false, FR, MF, FUSED>(a, tile, e, first, live, xl, mx[w], unscale[w], acc);
  switch (tile.sg.nbits) {
    case 2:
      HI2X_FEW(2)
      break;
    case 4:
      HI2X_FEW(4)
      break;
    default:
      HI2X_FEW(8)
  }
#undef HI2X_FEW
  // the waves' partial sums: [fragment][row of activations][slot]
  float* red = reinterpret_cast<float*>(lds);
  __syncthreads();
#pragma unroll
  for (int f = 0; f < FR; ++f)
#pragma unroll
    for (int m = 0; m < MF; ++m)
      *reinterpret_cast<f32x4v*>(red + ((w * FR + f) * MF + m) * 256 + (lane & 15) * 16 +
                                 4 * (lane >> 4)) = acc[f][m];
  __syncthreads();
  for (int o = tid; o < 256 * FR * MF; o += 64 * FW) {
    const int slot = o & 15, row = (o >> 4) & 15, m = (o >> 8) % MF, f = (o >> 8) / MF;
    const int t = 16 * m + row;
    if (t >= live || f >= tile.count) continue;
    const int n = g.w.rows[(int64_t)(tile.sg.frag0 + tile.first + f) * 16 + slot];
    if (n < 0) continue;
    float y = 0.0f;
#pragma unroll
    for (int v = 0; v < FW; ++v) {
      const float* p = red + ((v * FR + f) * MF + m) * 256 + slot;
      y += p[row * 16];
      if (FUSED && a.npl == 2) y += p[(row + 8) * 16];
    }
    const int64_t at = first + t;
    if (!FUSED) {
      const int64_t r = g.src ? g.src[at] : at;
      y *= r >= 0 && r < g.x.rows ? g.x.scale[r] : __builtin_nanf("");
    }
    const float bias = g.epi.bias ? load_as_f32(g.epi.bias, n, g.epi.dt_bias) : 0.0f;
    finish(g.epi, y, bias, at, n);
  }
}

template <int FR, int MF, bool FUSED>
int launch(const FewArgs& a, hipStream_t s) {
  const hi2x_packed& w = a.g.w;
  const int64_t nch = w.kp / PK_CHUNK;
  const size_t x = FUSED ? (size_t)FW * ((nch + FW - 1) / FW) * a.mt * a.npl * 256 : 0;
  const size_t red = (size_t)FW * FR * MF * 1024;
  const size_t dyn = x > red ? x : red;
  // a segment's last tile may be partly filled
  const int64_t nx = FR == 1 ? w.max_frags : w.max_frags / FR + PK_SEGS;
  const int64_t part = a.g.offs ? (w.experts < a.g.slots ? w.experts : a.g.slots) : 1;
  const int64_t ny = a.g.offs ? a.g.slots / a.mt + part : (a.g.slots + a.mt - 1) / a.mt;
  HI2X_REQUIRE(nx < (1ll << 31) && ny <= 65535, "packed_linear: %lld rows are too many",
               (long long)a.g.slots);
  if (dyn > 32768)
    HI2X_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(packed_few_kernel<FR, MF, FUSED>),
                                 hipFuncAttributeMaxDynamicSharedMemorySize, (int)dyn));
  packed_few_kernel<FR, MF, FUSED><<<dim3((unsigned)nx, (unsigned)ny), 64 * FW, dyn, s>>>(a);
  return launch_status("packed_linear");
}

}  // namespace

// Activation rows a workgroup can transform for itself: their planes in 64 KB of LDS (two
// workgroups a CU), both planes' rows in one MFMA operand of 16.
int64_t few_rows(int64_t k, int npl) {
  const int64_t nch = (k + PK_CHUNK - 1) / PK_CHUNK;
  const int64_t row = (nch + FW - 1) / FW * FW * 256 * npl;
  const int64_t fit = 65536 / row;
  return fit < 16 / npl ? fit : 16 / npl;
}

int packed_few(const GemmArgs& g, hipStream_t s) {
  FewArgs a{};
  a.g = g;
  a.npl = g.x.nplanes;
  if (g.slots <= 16 || (g.offs && g.slots <= 16 * g.w.experts)) {
    a.mt = 16;
    return g.w.max_frags >= 1024 ? launch<4, 1, false>(a, s)
                                 : (g.w.max_frags >= 512 ? launch<2, 1, false>(a, s)
                                                         : launch<1, 1, false>(a, s));
  }
  if (g.slots <= 32) {
    a.mt = 32;
    return g.w.max_frags >= 512 ? launch<2, 2, false>(a, s) : launch<1, 2, false>(a, s);
  }
  a.mt = 64;
  return g.w.max_frags >= 512 ? launch<2, 4, false>(a, s) : launch<1, 4, false>(a, s);
}

}  // namespace hi2x

using namespace hi2x;

extern "C" int64_t hi2x_packed_few_rows(int64_t k, int nplanes) {
  if (k < 16 || k % 16 || nplanes < 1 || nplanes > 2) return -1;
  return few_rows(k, nplanes);
}

extern "C" int hi2x_packed_linear_few(const hi2x_packed* w, const void* x, int dtype, int64_t ldx,
                                      int64_t x_rows, int nplanes, const uint8_t* had,
                                      const uint16_t* col_scale, int per_expert,
                                      const int64_t* src, const int64_t* offs, int64_t slots,
                                      const hi2x_epilogue* epi, void* stream) {
  clear_error();
  HI2X_REQUIRE(w && epi, "packed_linear_few: null argument");
  if (int rc = check_packed(w, "packed_linear_few")) return rc;
  if (int rc = check_product(w, src, offs, slots, x_rows, epi, "packed_linear_few")) return rc;
  if (int rc = check_x(x, dtype, ldx, x_rows, w->k, "packed_linear_few")) return rc;
  HI2X_REQUIRE(nplanes == 1 || nplanes == 2, "packed_linear_few: %d planes", nplanes);
  const int64_t mt = few_rows(w->k, nplanes);
  HI2X_REQUIRE(mt >= 1, "packed_linear_few: %lld columns do not fit", (long long)w->k);
  if (slots == 0) return HI2X_OK;
  HI2X_REQUIRE(had, "packed_linear_few: null flags");
  FewArgs a{};
  a.g = GemmArgs{*w, hi2x_activations{}, src, offs, slots, *epi};
  a.x = x;
  a.dtype = dtype;
  a.ldx = ldx;
  a.x_rows = x_rows;
  a.had = had;
  a.cs = col_scale;
  a.per_expert = per_expert;
  a.npl = nplanes;
  a.mt = (int)mt;
  const hipStream_t s = as_stream(stream);
  return w->max_frags >= 1024 ? launch<2, 1, true>(a, s) : launch<1, 1, true>(a, s);
}
