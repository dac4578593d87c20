// Products by packed tensors: out = act(T(x) Wq^T + bias) * mul + residual, for one tensor
// or for the experts of a projection over their routed slots.
#include "packed.h"

namespace hi2x {
namespace {

// 64 lanes x 16 bytes from global memory straight into LDS at `lds` (+ 16 lane).  As inline
// assembly: the compiler would otherwise take the asynchronous write for an alias of every
// later LDS read and wait for all loads in flight before each one.
__device__ __forceinline__ void dma16(__amdgpu_buffer_rsrc_t rs, uint32_t voff, uint32_t soff,
                                      void* lds) {
  const uint32_t la = __builtin_amdgcn_readfirstlane(
      (uint32_t)(size_t)(__attribute__((address_space(3))) void*)lds);
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
  asm volatile("s_mov_b32 m0, %0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
               :
               : "s"(la), "v"(voff), "s"(rs), "s"(soff)
               : "m0", "memory");
#pragma clang diagnostic pop
}

constexpr int waitcnt(int vm, int lgkm) {
  return (vm & 15) | ((vm >> 4) << 14) | (7 << 4) | (lgkm << 8);
}

// The main loop of one tile: 4 waves of NF fragments x 16 MF slots each, all reading the
// same activations from LDS.  A stage of 16 MF slots x 128 columns is 256 bytes a slot in
// 16 pieces; piece p of slot t lies at p ^ (t % 16), so that the 16 slots a fragment read
// touches at one piece fall on different banks.
template <int BITS, bool B16, int NF, int MF>
__device__ __forceinline__ void gemm_loop(const GemmArgs& g, const Tile& tile, char* lds,
                                          const char* xb, int64_t xbytes,
                                          const uint32_t (&xoff)[MF], f32x4v (&acc)[NF][MF]) {
  const int tid = threadIdx.x, lane = tid & 63;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int q = lane >> 4;
  const int nch = (int)(g.w.kp / PK_CHUNK);
  const int nst = nch * g.x.nplanes;
  constexpr int STAGE = 16 * MF * 256;
  // this wave's fragments: what lies past the tile's reads as zero and is never stored
  const int mine = tile.count - wv * NF < NF ? tile.count - wv * NF : NF;
  const int64_t nblk = g.w.kp / tile.sg.block;
  const uint32_t cfrag = (uint32_t)nch * (256 * BITS), pfrag = (uint32_t)nblk * 64;
  const int64_t f0 = tile.first + wv * NF;
  const __amdgpu_buffer_rsrc_t cr =
      rsrc(static_cast<const char*>(g.w.codes) + tile.sg.codes + f0 * cfrag,
           mine > 0 ? (int64_t)mine * cfrag : 0);
  const __amdgpu_buffer_rsrc_t pr =
      rsrc(static_cast<const char*>(g.w.params) + tile.sg.params + f0 * pfrag,
           mine > 0 ? (int64_t)mine * pfrag : 0);
  const int bsh = tile.sg.block == 64 ? 6 : (tile.sg.block == 32 ? 5 : 4);
  const uint32_t poff = 64 * ((32 * q) >> bsh) + 4 * (lane & 15);
  const int64_t plane = g.x.rows * g.x.kp * 2;
  auto stage = [&](int st) {
    const int pl = g.x.nplanes == 2 ? st & 1 : 0, c = g.x.nplanes == 2 ? st >> 1 : st;
    const __amdgpu_buffer_rsrc_t xr = rsrc(xb + pl * plane, xbytes);
    char* to = lds + (st & 1) * STAGE;
#pragma unroll
    for (int i = 0; i < MF; ++i) dma16(xr, xoff[i], (uint32_t)c * 256, to + (wv * MF + i) * 1024);
  };
  // The codes of the next stage are fetched a stage ahead; at 8 bits (32 registers a set)
  // a second set would spill, and the stage's own are fetched as it begins.
  constexpr bool AHEAD = BITS < 8;
  uint32_t cw[NF][BITS], pw[NF][2], cn[AHEAD ? NF : 1][BITS], pn[AHEAD ? NF : 1][2];
  auto fetch = [&](int c, int f, uint32_t (&cd)[BITS], uint32_t (&pd)[2]) {
    load_codes<BITS>(cr, lane, f * cfrag + (uint32_t)c * (256 * BITS), cd);
    const uint32_t so = f * pfrag + ((uint32_t)(c * PK_CHUNK) >> bsh) * 64;
    pd[0] = __builtin_amdgcn_raw_buffer_load_b32(pr, (int)poff, (int)so, 0);
    pd[1] = B16 ? __builtin_amdgcn_raw_buffer_load_b32(pr, (int)poff + 64, (int)so, 0) : 0u;
  };
  auto chunk = [&](int st) { return g.x.nplanes == 2 ? st >> 1 : st; };
  if constexpr (AHEAD) {
#pragma unroll
    for (int f = 0; f < NF; ++f) fetch(0, f, cn[f], pn[f]);
  }
  stage(0);
  const int t0 = lane & 15;
  for (int st = 0; st < nst; ++st) {
    // stage st and the codes have landed; behind the barrier nobody reads stage st - 1
    __builtin_amdgcn_s_waitcnt(waitcnt(0, 15));
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    __builtin_amdgcn_s_barrier();
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
#pragma unroll
    for (int f = 0; f < NF; ++f) {
      if constexpr (AHEAD) {
#pragma unroll
        for (int i = 0; i < BITS; ++i) cw[f][i] = cn[f][i];
        pw[f][0] = pn[f][0];
        pw[f][1] = pn[f][1];
        if (st + 1 < nst) fetch(chunk(st + 1), f, cn[f], pn[f]);
      } else {
        fetch(chunk(st), f, cw[f], pw[f]);
      }
    }
    if (st + 1 < nst) stage(st + 1);
    const char* xs = lds + (st & 1) * STAGE + t0 * 256;
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      h16x8 b[MF];
#pragma unroll
      for (int m = 0; m < MF; ++m)
        b[m] = *reinterpret_cast<const h16x8*>(xs + m * 4096 + 16 * (((4 * q) ^ t0) ^ s));
#pragma unroll
      for (int f = 0; f < NF; ++f) {
        const h16x2 ls = __builtin_bit_cast(h16x2, B16 && s >= 2 ? pw[f][1] : pw[f][0]);
        const h16x8 a = decode_step<BITS>(cw[f], s, (h16x2){ls[0], ls[0]}, (h16x2){ls[1], ls[1]});
#pragma unroll
        for (int m = 0; m < MF; ++m)
          acc[f][m] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b[m], acc[f][m], 0, 0, 0);
      }
    }
  }
}

// One workgroup: 64 NF slots of w's layout (one segment) x 16 MF activation rows.
template <int NF, int MF>
__global__ __launch_bounds__(256, 2) void packed_gemm_kernel(GemmArgs g) {
  constexpr int MT = 16 * MF;
  constexpr int XB = 2 * MT * 256;                   // two stages of activations
  constexpr int EH = XB / (64 * NF * 4) < MT ? XB / (64 * NF * 4) : MT;  // rows per store pass
  static_assert(EH >= 16 && EH % 16 == 0 && MT % EH == 0, "store passes");
  __shared__ __attribute__((aligned(1024))) char lds[XB];
  const PkWork wk = find_work(g.offs, (int)g.w.experts, g.slots, MT, blockIdx.y);
  const int e = __builtin_amdgcn_readfirstlane(wk.e);
  if (e < 0) return;
  Tile tile;
  if (!find_tile(g.w, e, blockIdx.x, 4 * NF, tile)) return;
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
  const int64_t first = __builtin_amdgcn_readfirstlane((int)wk.first);  // slots < 2^31
  const int64_t left = __builtin_amdgcn_readfirstlane((int)wk.end) - first;
  const int live = (int)(left < MT ? left : MT);
  // Where the rows this lane stages begin.  Rows past the end read zeros or another
  // tile's, and are not stored; indices outside the activations read row 0 (and come out as
  // NaN below).  Without src the resource begins at the tile's own rows.
  uint32_t xoff[MF];
  const uint32_t pitch = (uint32_t)g.x.kp * 2;
  const int64_t row0 = g.src ? 0 : first;
  const char* xb = reinterpret_cast<const char*>(g.x.planes) + row0 * pitch;
  const int64_t xbytes = (g.x.rows - row0) * pitch;
#pragma unroll
  for (int i = 0; i < MF; ++i) {
    const int t = 4 * (wv * MF + i) + (lane >> 4);
    int64_t r = t;
    if (g.src) {
      r = t < live ? g.src[first + t] : 0;
      if (r < 0 || r >= g.x.rows) r = 0;
    }
    xoff[i] = (uint32_t)r * pitch + 16 * ((lane & 15) ^ (t & 15));
  }
  f32x4v acc[NF][MF];
#pragma unroll
  for (int f = 0; f < NF; ++f)
#pragma unroll
    for (int m = 0; m < MF; ++m) acc[f][m] = f32x4v{0.0f, 0.0f, 0.0f, 0.0f};
  const bool b16 = tile.sg.block == 16;
  switch (tile.sg.nbits) {
    case 2:
      if (b16)
        gemm_loop<2, true, NF, MF>(g, tile, lds, xb, xbytes, xoff, acc);
      else
        gemm_loop<2, false, NF, MF>(g, tile, lds, xb, xbytes, xoff, acc);
      break;
    case 4:
      if (b16)
        gemm_loop<4, true, NF, MF>(g, tile, lds, xb, xbytes, xoff, acc);
      else
        gemm_loop<4, false, NF, MF>(g, tile, lds, xb, xbytes, xoff, acc);
      break;
    default:
      if (b16)
        gemm_loop<8, true, NF, MF>(g, tile, lds, xb, xbytes, xoff, acc);
      else
        gemm_loop<8, false, NF, MF>(g, tile, lds, xb, xbytes, xoff, acc);
  }
  // Store passes of EH rows through LDS: the accumulators hold 4 slots of one row each; a
  // pass then takes consecutive threads over consecutive slots.
  float* ep = reinterpret_cast<float*>(lds);
  constexpr int NS = 64 * NF;
  const hi2x_epilogue& E = g.epi;
#pragma unroll
  for (int p = 0; p < MT / EH; ++p) {
    __syncthreads();
#pragma unroll
    for (int m = 0; m < EH / 16; ++m)
#pragma unroll
      for (int f = 0; f < NF; ++f)
        *reinterpret_cast<f32x4v*>(ep + (16 * m + (lane & 15)) * NS + (wv * NF + f) * 16 +
                                   4 * (lane >> 4)) = acc[f][p * (EH / 16) + m];
    __syncthreads();
    constexpr int TPR = NS < 256 ? NS : 256;  // threads on one row
    const int slot = tid % TPR;
    const int n = slot < 16 * tile.count
                      ? g.w.rows[(int64_t)(tile.sg.frag0 + tile.first) * 16 + slot]
                      : -1;
    if (n >= 0) {
      const float bias = E.bias ? load_as_f32(E.bias, n, E.dt_bias) : 0.0f;
      for (int t = tid / TPR; t < EH && p * EH + t < live; t += 256 / TPR) {
        const int64_t o = first + p * EH + t;
        int64_t r = g.src ? g.src[o] : o;
        float sc = __builtin_nanf("");
        if (r >= 0 && r < g.x.rows) sc = g.x.scale[r];
        finish(E, ep[t * NS + slot] * sc, bias, o, n);
      }
    }
  }
}

template <int NF, int MF>
int launch_gemm(const GemmArgs& g, hipStream_t s) {
  constexpr int MT = 16 * MF;
  const int64_t nx = g.w.max_tiles[NF == 1 ? 0 : (NF == 2 ? 1 : 2)];
  // every expert can leave one tile partly filled
  const int64_t part = g.offs ? (g.w.experts < g.slots ? g.w.experts : g.slots) : 1;
  const int64_t ny = g.offs ? g.slots / MT + part : (g.slots + MT - 1) / MT;
  HI2X_REQUIRE(nx < (1ll << 31) && ny <= 65535, "packed_linear: %lld rows are too many",
               (long long)g.slots);
  packed_gemm_kernel<NF, MF><<<dim3((unsigned)nx, (unsigned)ny), 256, 0, s>>>(g);
  return launch_status("packed_linear");
}

}  // namespace
}  // namespace hi2x

using namespace hi2x;

extern "C" int hi2x_packed_linear(const hi2x_packed* w, const hi2x_activations* x,
                                  const int64_t* src, const int64_t* offs, int64_t slots,
                                  const hi2x_epilogue* epi, void* stream) {
  clear_error();
  HI2X_REQUIRE(w && x && epi, "packed_linear: null argument");
  if (int rc = check_packed(w, "packed_linear")) return rc;
  if (int rc = check_product(w, src, offs, slots, x->rows, epi, "packed_linear")) return rc;
  HI2X_REQUIRE(x->kp == w->kp, "packed_linear: activations of %lld padded columns, %lld needed",
               (long long)x->kp, (long long)w->kp);
  HI2X_REQUIRE(x->nplanes == 1 || x->nplanes == 2, "packed_linear: %d planes", x->nplanes);
  HI2X_REQUIRE(!src || x->rows * x->kp * 2 < (1ll << 32) - 1,
               "packed_linear: 4 GiB of activations or more cannot be taken by index");
  if (slots == 0) return HI2X_OK;
  HI2X_REQUIRE(x->rows > 0 && x->planes && x->scale, "packed_linear: null activations");
  const GemmArgs g{*w, *x, src, offs, slots, *epi};
  const hipStream_t s = as_stream(stream);
  if (slots <= 64 || (offs && slots <= 16 * w->experts)) return packed_few(g, s);
  return launch_gemm<4, 8>(g, s);
}
