// Products of few rows by packed tensors: single tokens, small batches of them, and the
// experts' products of a decode step.  Bound by reading the packed weights once.
//
// A workgroup of 8 waves takes FR fragments (16 FR rows of the tensor) and up to MT
// activation rows; the columns are split over the waves by chunks of 128, and the partial
// sums meet in LDS, so nothing is joined across workgroups.  A wave keeps UN chunks of codes
// in flight (one 16-byte load a lane holds a fragment's whole chunk at 4 bits).  The loops
// stay rolled: unrolled, the code of a short call outgrows the instruction cache.
#include "packed.h"

namespace hi2x {
namespace {

struct FewArgs {
  GemmPair two;  // blockIdx.z picks
  RawRows x;     // activations that are transformed here
};

// activations: transformed, or as they are (16 bits, 32 bits, act(x) * x2 of 32 bits)
enum { GIVEN = 0, RAW16 = 1, RAW32 = 2, GLU32 = 3 };

// One pass of the transform: the wave's next CP = 8 / MP chunks of up to MP rows (a power of
// two), a 16-column group of one row per lane.  As in the separate pass (activations_kernel)
// a row is scaled by a power of two, here by its largest value among the pass's columns; the
// products of a pass are summed apart and unscaled.  Row r of chunk i lies in LDS at
// (i R + r) 256 with its 16-byte pieces p at p ^ (r % 16); R = MP npl, the second plane's
// rows behind the first's.
template <int MODE, int MP, int FW>
struct FewPass {
  static constexpr bool F32 = MODE != RAW16, GLU = MODE == GLU32;
  static constexpr int CP = 8 / MP, V = F32 ? 4 : 2;  // chunks; 16-byte pieces of a group
  u32x4 raw[V], up[GLU ? V : 1];

  __device__ __forceinline__ static int group(int w, int i0) {  // of 16 columns
    const int r = threadIdx.x & (64 / MP - 1);
    return 8 * (w + FW * (i0 + (r >> 3))) + (r & 7);
  }

  // `src`: the lane's row of the activations, negative for none
  __device__ __forceinline__ void load(const FewArgs& a, int k, int64_t src, int w, int i0) {
    const int g = group(w, i0);
#pragma unroll
    for (int v = 0; v < V; ++v) raw[v] = up[GLU ? v : 0] = u32x4{0u, 0u, 0u, 0u};
    if (src >= 0 && 16 * g < k) {
      const u32x4* from = reinterpret_cast<const u32x4*>(
          static_cast<const char*>(a.x.x) + (src * a.x.ldx + 16 * g) * (F32 ? 4 : 2));
#pragma unroll
      for (int v = 0; v < V; ++v) raw[v] = from[v];
      if constexpr (GLU) {
        from = reinterpret_cast<const u32x4*>(a.x.x2 + src * a.x.ldx + 16 * g);
#pragma unroll
        for (int v = 0; v < V; ++v) up[v] = from[v];
      }
    }
  }

  // Returns the factor that unscales the lane's row.
  __device__ __forceinline__ float store(const FewArgs& a, int k, const uint8_t* had,
                                         const uint16_t* cs, int w, int i0, char* xl) const {
    const int lane = threadIdx.x & 63, g = group(w, i0);
    const bool in = 16 * g < k;
    float v[16];
    if constexpr (F32) {
#pragma unroll
      for (int t = 0; t < 16; ++t) v[t] = __uint_as_float(raw[t >> 2][t & 3]);
      if constexpr (GLU) {
#pragma unroll
        for (int t = 0; t < 16; ++t) {
          v[t] = activate(v[t], a.x.act) * __uint_as_float(up[t >> 2][t & 3]);
          __builtin_amdgcn_sched_barrier(0);  // one after the other: few registers
        }
      }
    } else if (a.x.dtype == 1) {
#pragma unroll
      for (int t = 0; t < 16; ++t)
        v[t] = f16_from_bits((uint16_t)(raw[t >> 3][(t >> 1) & 3] >> (16 * (t & 1))));
    } else {
#pragma unroll
      for (int t = 0; t < 8; ++t) {
        const uint32_t u = raw[t >> 2][t & 3];
        v[2 * t] = __uint_as_float(u << 16);
        v[2 * t + 1] = __uint_as_float(u & 0xffff0000u);
      }
    }
    if (cs && in) {
#pragma unroll
      for (int t = 0; t < 16; ++t) {
        v[t] = v[t] / f16_from_bits(cs[16 * g + t]);
        if (t & 1) __builtin_amdgcn_sched_barrier(0);  // two at a time: few registers
      }
    }
    float m = 0.0f;
#pragma unroll
    for (int t = 0; t < 16; ++t) m = fmaxf(m, fabsf(v[t]));  // NaN is passed over
    if (m == __builtin_inff()) {
      m = 0.0f;
#pragma unroll
      for (int t = 0; t < 16; ++t) {
        const float b = fabsf(v[t]);
        m = fmaxf(m, b < __builtin_inff() ? b : 0.0f);
      }
    }
    uint32_t mb = __float_as_uint(m);  // the order of non-negative floats
    if constexpr (MP <= 4) {
      mb = row_umax(mb);
#pragma unroll
      for (int d = 16; d < 64 / MP; d <<= 1) {
        const uint32_t o = __shfl_xor(mb, d);
        mb = o > mb ? o : mb;
      }
    } else {
#pragma unroll
      for (int d = 1; d < 64 / MP; d <<= 1) {
        const uint32_t o = __shfl_xor(mb, d);
        mb = o > mb ? o : mb;
      }
    }
    int ex = 0;
    if (mb) (void)frexpf(__uint_as_float(mb), &ex);
    const int s = 13 - ex > 126 ? 126 : (13 - ex < -126 ? -126 : 13 - ex);
    const float sc = ldexpf(1.0f, s);
#pragma unroll
    for (int t = 0; t < 16; ++t) v[t] *= sc;
    if (in && had[g]) {
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
    const int R = MP * a.x.npl, p0 = 2 * (g & 7);
    const int r = lane / (64 / MP), chunk = (lane & (64 / MP - 1)) >> 3;
    uint32_t h[8];
#pragma unroll
    for (int t = 0; t < 8; ++t)
      h[t] = (uint32_t)f16_bits(v[2 * t]) | (uint32_t)f16_bits(v[2 * t + 1]) << 16;
    char* d = xl + (chunk * R + r) * 256;
    *reinterpret_cast<u32x4*>(d + 16 * (p0 ^ r)) = u32x4{h[0], h[1], h[2], h[3]};
    *reinterpret_cast<u32x4*>(d + 16 * ((p0 + 1) ^ r)) = u32x4{h[4], h[5], h[6], h[7]};
    if (a.x.npl == 2) {
      const int r2 = MP + r;
#pragma unroll
      for (int t = 0; t < 8; ++t)
        h[t] = rest_bits(v[2 * t], h[t]) | rest_bits(v[2 * t + 1], h[t] >> 16) << 16;
      d = xl + (chunk * R + r2) * 256;
      *reinterpret_cast<u32x4*>(d + 16 * (p0 ^ r2)) = u32x4{h[0], h[1], h[2], h[3]};
      *reinterpret_cast<u32x4*>(d + 16 * ((p0 + 1) ^ r2)) = u32x4{h[4], h[5], h[6], h[7]};
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup", "local");  // read by this wave only
    return ldexpf(1.0f, -s);
  }
};

// MT: activation rows of the workgroup; as they are, a power of two up to 8, transformed, 16.
// A step is one chunk and plane; the codes (and transformed activations) of UN
// steps are fetched while the UN before them are multiplied.
template <int BITS, int FR, int MT, int MODE, int FW>
__device__ __forceinline__ void few_loop(const FewArgs& a, const GemmArgs& g, const Tile& tile,
                                         int e, int64_t first, int live,
                                         FewPass<MODE == GIVEN ? RAW16 : MODE,
                                                 MODE == GIVEN ? 1 : MT, FW> pass,
                                         int64_t src, char* xl,
                                         f32x4v (&acc)[FR][MODE == GIVEN ? MT / 16 : 1]) {
  constexpr bool RAW = MODE != GIVEN;
  constexpr int MF = RAW ? 1 : MT / 16, MP = RAW ? MT : 1;
  constexpr int CP = 8 / MP;
  // what the registers hold: 128 with eight waves, of which a CU takes two workgroups
  constexpr int RU = BITS == 8 ? 1 : (MODE != RAW16 || FW == 8 ? 2 : 4);
  constexpr int UN = RAW ? (CP < RU ? CP : RU) : (FR == 1 && BITS < 8 ? 2 : 1);
  constexpr bool AHEAD = RAW || BITS < 8 || FR == 1;
  const int k = (int)g.w.k;
  const int tid = threadIdx.x, lane = tid & 63, q = lane >> 4, col = lane & 15;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int nch = (int)(g.w.kp / PK_CHUNK);
  const int nc = w < nch ? (nch - w + FW - 1) / FW : 0;
  const int psh = RAW ? 0 : g.x.nplanes - 1;
  const int steps = nc << psh;
  const int64_t nblk = g.w.kp / tile.block;
  const uint32_t cfrag = (uint32_t)nch * (256 * BITS), pfrag = (uint32_t)nblk * 64;
  const __amdgpu_buffer_rsrc_t cr =
      rsrc(static_cast<const char*>(g.w.codes) + tile.codes + (int64_t)tile.first * cfrag,
           (int64_t)tile.count * cfrag);
  const __amdgpu_buffer_rsrc_t pr =
      rsrc(static_cast<const char*>(g.w.params) + tile.params + (int64_t)tile.first * pfrag,
           (int64_t)tile.count * pfrag);
  const int bsh = tile.block == 64 ? 6 : (tile.block == 32 ? 5 : 4);
  const uint32_t poff = 64 * ((32 * q) >> bsh) + 4 * (lane & 15);
  const uint32_t poff2 = poff + (tile.block == 16 ? 64 : 0);  // of columns 16..31
  const uint32_t magic = decode_magic();
  struct Group {
    uint32_t cw[UN][FR][BITS], pw[UN][FR][2];
    h16x8 b[RAW ? 1 : UN][4][MF];
  };
  Group cur, nxt;
  uint32_t xoff[MF];
  __amdgpu_buffer_rsrc_t xs;
  if constexpr (!RAW) {
    const uint32_t pitch = (uint32_t)g.x.kp * 2 * g.x.nplanes;
    const int64_t row0 = g.src ? 0 : first;
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
  auto fetch = [&](int s0, Group& to) {
#pragma unroll
    for (int u = 0; u < UN; ++u) {
      if (s0 + u >= steps) continue;
      const int c = w + FW * ((s0 + u) >> psh);
#pragma unroll
      for (int f = 0; f < FR; ++f) {
        load_codes<BITS>(cr, lane, f * cfrag + (uint32_t)c * (256 * BITS), to.cw[u][f]);
        const uint32_t so = f * pfrag + ((uint32_t)(c * PK_CHUNK) >> bsh) * 64;
        to.pw[u][f][0] = __builtin_amdgcn_raw_buffer_load_b32(pr, (int)poff, (int)so, 0);
        to.pw[u][f][1] = __builtin_amdgcn_raw_buffer_load_b32(pr, (int)poff2, (int)so, 0);
      }
      if constexpr (!RAW) {
        const int at = ((c << psh) + ((s0 + u) & psh)) * 256;
#pragma unroll
        for (int s = 0; s < 4; ++s)
#pragma unroll
          for (int m = 0; m < MF; ++m)
            to.b[u][s][m] = __builtin_bit_cast(
                h16x8, __builtin_amdgcn_raw_buffer_load_b128(xs, (int)xoff[m] + 16 * s, at, 0));
      }
    }
  };
  // raw: the row this lane's operand column reads, and which lane transforms it
  int R = 0, xr = 0, from = 0;
  float unscale = 1.0f;
  const uint8_t* had = nullptr;
  const uint16_t* cs = nullptr;
  f32x4v part[FR];
  if constexpr (RAW) {
    had = g.w.had + (g.w.per_expert ? (int64_t)e * (g.w.k / 16) : 0);
    cs = g.w.col_scale;
    if (cs && g.w.per_expert) cs += (int64_t)e * g.w.k;
    R = MP * a.x.npl;
    const int t = a.x.npl == 2 ? col & 7 : col, plane = a.x.npl == 2 ? col >> 3 : 0;
    xr = t < MP ? plane * MP + t : 0;
    from = t < MP ? t * (64 / MP) : 0;
  }
  if constexpr (AHEAD) fetch(0, nxt);
  for (int s0 = 0; s0 < steps; s0 += UN) {
    if constexpr (AHEAD)
      cur = nxt;
    else
      fetch(s0, cur);
    if constexpr (RAW) {
      if (s0 % CP == 0) {
        fetch(s0 + UN, nxt);
        unscale = pass.store(a, k, had, cs, w, s0, xl);
        if (s0 + CP < steps) pass.load(a, k, src, w, s0 + CP);
        unscale = __shfl(src < 0 ? __builtin_nanf("") : unscale, from);
#pragma unroll
        for (int f = 0; f < FR; ++f) part[f] = f32x4v{0.0f, 0.0f, 0.0f, 0.0f};
      } else {
        fetch(s0 + UN, nxt);
      }
    } else if constexpr (AHEAD) {
      fetch(s0 + UN, nxt);
    }
#pragma unroll
    for (int u = 0; u < UN; ++u) {
      if (s0 + u >= steps) break;
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        h16x8 x;
        if constexpr (RAW)
          x = *reinterpret_cast<const h16x8*>(xl + (((s0 + u) % CP) * R + xr) * 256 +
                                              16 * ((4 * q + s) ^ xr));
#pragma unroll
        for (int f = 0; f < FR; ++f) {
          const h16x2 ls = __builtin_bit_cast(h16x2, cur.pw[u][f][s >> 1]);
          const h16x8 av = decode_step<BITS>(cur.cw[u][f], s, (h16x2){ls[0], ls[0]},
                                             (h16x2){ls[1], ls[1]}, magic);
          if constexpr (RAW) {
            part[f] = __builtin_amdgcn_mfma_f32_16x16x32_f16(av, x, part[f], 0, 0, 0);
          } else {
#pragma unroll
            for (int m = 0; m < MF; ++m)
              acc[f][m] = __builtin_amdgcn_mfma_f32_16x16x32_f16(av, cur.b[u][s][m], acc[f][m],
                                                                 0, 0, 0);
          }
        }
      }
    }
    if constexpr (RAW) {
      if (s0 % CP + UN >= CP || s0 + UN >= steps) {
#pragma unroll
        for (int f = 0; f < FR; ++f)
#pragma unroll
          for (int t = 0; t < 4; ++t)
            acc[f][0][t] = __builtin_fmaf(part[f][t], unscale, acc[f][0][t]);
      }
    }
  }
}

template <int FR, int MT, int MODE, int FW>
__global__ __launch_bounds__(64 * FW,
                             MODE == GIVEN ? 4 : (MODE != RAW16 ? 2 : (FW == 8 ? 4 : 3)))
void packed_few_kernel(FewArgs a) {
  constexpr bool RAW = MODE != GIVEN;
  constexpr int MF = RAW ? 1 : MT / 16;
  constexpr int XW = RAW ? 4096 : 0;         // bytes of transformed rows of a wave
  constexpr int RED = FW * FR * MF * 1024;   // the partial sums
  __shared__ __attribute__((aligned(16))) char lds[FW * XW > RED ? FW * XW : RED];
  const GemmArgs& g = a.two.g[blockIdx.z];
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  int e = 0, live = 1;
  int64_t first = blockIdx.y;  // tiles of one row: the tile is its slot
  if constexpr (MT > 1) {      // (one tensor)
    first *= MT;
    live = (int)(g.slots - first < MT ? g.slots - first : MT);
  }
  // the rows to transform come first, behind nothing but their index
  FewPass<RAW ? MODE : RAW16, RAW ? MT : 1, FW> pass;
  int64_t src = -1;
  if constexpr (RAW) {
    const int row = lane / (64 / MT);
    if (row < live) {
      src = g.src ? g.src[first + row] : first + row;
      if (src >= a.x.rows) src = -1;
    }
    pass.load(a, (int)g.w.k, src, w, 0);
  }
  if (MT == 1 && g.offs) {  // the expert: as many as end at or before the slot come before it
    for (int e0 = 0; e0 < (int)g.w.experts; e0 += 64) {
      const bool before = e0 + lane < (int)g.w.experts && g.offs[e0 + lane + 1] <= first;
      e += __builtin_popcountll(__ballot(before));
    }
    if (e >= (int)g.w.experts) return;  // (ranges that end before the last slot)
  }
  Tile tile;
  if (!find_tile(g.w, e, blockIdx.x, FR, tile)) return;
  // what the epilogue needs of this thread's first output is on its way meanwhile
  const hi2x_epilogue& E = g.epi;
  int n = -1, t = 0;
  float bias = 0.0f, mul = 1.0f, res = 0.0f;
  auto operands = [&](int o) {
    const int f = (o >> 8) / MF;
    t = 16 * ((o >> 8) % MF) + ((o >> 4) & 15);
    n = t < live && f < tile.count ? g.w.rows[(int64_t)(tile.frag + f) * 16 + (o & 15)] : -1;
    if (n < 0) return;
    if (E.bias) bias = load_as_f32(E.bias, n, E.dt_bias);
    if (E.mul) mul = load_as_f32(E.mul, (first + t) * E.ld_mul + n, E.dt_mul);
    if (E.residual) res = load_as_f32(E.residual, (first + t) * E.ld_residual + n, E.dt_residual);
  };
  if (tid < 256 * FR * MF) operands(tid);
  f32x4v acc[FR][MF];
#pragma unroll
  for (int f = 0; f < FR; ++f)
#pragma unroll
    for (int m = 0; m < MF; ++m) acc[f][m] = f32x4v{0.0f, 0.0f, 0.0f, 0.0f};
  char* xl = lds + w * XW;
  switch (tile.nbits) {
    case 2:
      few_loop<2, FR, MT, MODE, FW>(a, g, tile, e, first, live, pass, src, xl, acc);
      break;
    case 4:
      few_loop<4, FR, MT, MODE, FW>(a, g, tile, e, first, live, pass, src, xl, acc);
      break;
    default:
      few_loop<8, FR, MT, MODE, FW>(a, g, tile, e, first, live, pass, src, xl, acc);
  }
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
    if (o != tid) operands(o);
    if (n < 0) continue;
    float y = 0.0f;
#pragma unroll
    for (int v = 0; v < FW; ++v) {
      const float* p = red + v * (FR * MF * 256) + o;
      y += p[0];
      if (RAW && a.x.npl == 2) y += p[128];  // the second plane's, 8 rows on
    }
    const int64_t at = first + t;
    if (!RAW) {
      const int64_t r = g.src ? g.src[at] : at;
      y *= r >= 0 && r < g.x.rows ? g.x.scale[r] : __builtin_nanf("");
    }
    y = activate(y + bias, E.act);
    if (E.mul) y = y * mul;
    if (E.residual) y = y + res;
    store_from_f32(E.out, at * E.ld_out + n, E.dt_out, y);
  }
}

template <int FR, int MT, int MODE, int FW>
int launch(const FewArgs& a, int count, hipStream_t s) {
  const GemmArgs& g = a.two.g[0];
  const hi2x_packed& w = g.w;
  // a segment's last tile may be partly filled
  int64_t nx = w.max_frags;
  if (count > 1 && a.two.g[1].w.max_frags > nx) nx = a.two.g[1].w.max_frags;
  if (FR > 1) nx = nx / FR + PK_SEGS;
  const int64_t ny = (g.slots + MT - 1) / MT;
  HI2X_REQUIRE(nx < (1ll << 31) && ny <= 65535, "packed_linear: %lld rows are too many",
               (long long)g.slots);
  packed_few_kernel<FR, MT, MODE, FW>
      <<<dim3((unsigned)nx, (unsigned)ny, (unsigned)count), 64 * FW, 0, s>>>(a);
  return launch_status("packed_linear");
}

// One row (a tile of one of an expert's): the eight chunks of a pass keep all lanes of the
// transform busy, so a wave takes eight chunks where there are workgroups enough (2 a CU),
// and fewer where there are not: 4096 x 14336 16.8 us with eight waves and 18.2 with four,
// 14336 x 4096 16.7 and 13.3, the down projection of eight experts (2048 x 1024) 16.2 with
// four and 13.1 with one.
template <int MODE>
int launch_one(const FewArgs& a, int count, int64_t frags, hipStream_t s) {
  const int64_t nch = a.two.g[0].w.kp / PK_CHUNK;
  int waves = nch <= 8 ? 1 : (nch <= 16 ? 2 : (nch <= 32 ? 4 : 8));
  if (frags < 512 && waves < 8) waves *= 2;
  if (MODE != RAW16 && waves > 4) waves = 4;  // (more registers a wave)
  switch (waves) {
    case 1:
      return launch<1, 1, MODE, 1>(a, count, s);
    case 2:
      return launch<1, 1, MODE, 2>(a, count, s);
    case 4:
      return launch<1, 1, MODE, 4>(a, count, s);
    default:
      return launch<1, 1, MODE, MODE == RAW16 ? 8 : 4>(a, count, s);
  }
}

}  // namespace

int packed_few(const GemmArgs& g, hipStream_t s) {
  FewArgs a{};
  a.two = GemmPair{{g, g}};
  // More fragments a wave share their activation reads, while there are workgroups enough:
  // at 16 rows 28672 x 8192 takes 29.9 us with four, 37.6 with two and 61 with one, 8192 x
  // 8192 18.0 and 21.2, 4096 x 4096 11.6, 9.2 and 11.3, 1024 x 4096 8.4 with one and 10.4
  // with two.
  const int64_t frags = g.w.max_frags;
  return frags >= 512 ? launch<4, 16, GIVEN, 8>(a, 1, s)
                      : (frags >= 192 ? launch<2, 16, GIVEN, 8>(a, 1, s)
                                      : launch<1, 16, GIVEN, 8>(a, 1, s));
}

int packed_few_raw(const GemmPair& g, int count, const RawRows& x, hipStream_t s) {
  FewArgs a{};
  a.two = g;
  a.x = x;
  const GemmArgs& g0 = g.g[0];
  const int64_t live = !g0.offs ? 1 : (g0.slots < g0.w.experts ? g0.slots : g0.w.experts);
  const int64_t frags = g0.w.max_frags * count * live;
  if (g0.offs || g0.slots == 1)
    return x.x2 ? launch_one<GLU32>(a, count, frags, s)
                : (x.dtype == 0 ? launch_one<RAW32>(a, count, frags, s)
                                : launch_one<RAW16>(a, count, frags, s));
  // Eight waves shorten the walk along the columns, four transform the rows with half the
  // instructions, which counts where workgroups share a CU.
  const bool wide = frags < 512;
#define HI2X_RAW(MT)                                                                         \
  if (x.dtype == 0) return launch<1, MT, RAW32, 4>(a, count, s);                             \
  return wide ? launch<1, MT, RAW16, 8>(a, count, s) : launch<1, MT, RAW16, 4>(a, count, s);
  if (g0.slots <= 2) {
    HI2X_RAW(2)
  }
  if (g0.slots <= 4) {
    HI2X_RAW(4)
  }
  HI2X_RAW(8)
#undef HI2X_RAW
}

}  // namespace hi2x
