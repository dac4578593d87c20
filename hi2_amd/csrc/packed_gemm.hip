// Products by packed tensors: out = act(T(x) Wq^T + bias) * mul + residual, for one tensor
// or for the experts of a projection over their routed slots.
#include "packed.h"

namespace hi2x {
namespace {

// 64 lanes x 16 bytes from global memory straight into LDS at byte `la` (+ 16 lane).  As
// inline assembly: the compiler would otherwise take the asynchronous write for an alias of
// every later LDS read and wait for all loads in flight before each one.  The hardware wants one
// wait state between the write of M0 and the load, which the compiler does not add in here.
__device__ __forceinline__ void dma16(__amdgpu_buffer_rsrc_t rs, uint32_t voff, uint32_t soff,
                                      uint32_t la) {
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
               :
               : "s"(la), "v"(voff), "s"(rs), "s"(soff)
               : "m0");
#pragma clang diagnostic pop
}

constexpr int waitcnt(int vm, int lgkm) {
  return (vm & 15) | ((vm >> 4) << 14) | (7 << 4) | (lgkm << 8);
}

// The main loop of one tile: 4 waves of NF fragments x 16 MF slots each (of the AF and AM that
// the accumulators hold), all reading the same activations from LDS.  A stage of 16 MF slots x
// 128 columns is 256 bytes a slot in 16 pieces; piece p of slot t lies at p ^ (t % 16), so that
// the 16 slots a fragment read touches at one piece fall on different banks.  The activations of
// the next stage are on their way while one is multiplied, and the matrix units are busy 52 % of
// the cycles (14336 x 4096, 4096 rows, 470 us, 1020 TFLOP/s); the rest is decoding (28 % of the
// issue slots) and waits.  A barrier in mid-stage with the decode a fragment further ahead took 3
// to 8 % longer.
template <int BITS, bool B16, int NF, int MF, int AF, int AM>
__device__ __forceinline__ void gemm_loop(const GemmArgs& g, const Tile& tile, char* lds,
                                          const char* xb, int64_t xbytes,
                                          const uint32_t (&xoff)[AM], int c0, int c1,
                                          f32x4v (&acc)[AF][AM]) {
  const int tid = threadIdx.x, lane = tid & 63;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int q = lane >> 4;
  const int nch = __builtin_amdgcn_readfirstlane((int)(g.w.kp / PK_CHUNK));
  const int psh = __builtin_amdgcn_readfirstlane(g.x.nplanes - 1);
  const int first = c0 << psh, nst = c1 << psh;  // a chunk's planes one after the other
  const uint32_t lbase = __builtin_amdgcn_readfirstlane(
      (uint32_t)(size_t)(__attribute__((address_space(3))) char*)lds + wv * (MF * 1024));
  constexpr int STAGE = 16 * MF * 256;
  // this wave's fragments: what lies past the tile's reads as zero and is never stored
  const int mine = tile.count - wv * NF < NF ? tile.count - wv * NF : NF;
  const int64_t nblk = g.w.kp / tile.block;
  const uint32_t cfrag = (uint32_t)nch * (256 * BITS), pfrag = (uint32_t)nblk * 64;
  const int64_t f0 = tile.first + wv * NF;
  const __amdgpu_buffer_rsrc_t cr =
      rsrc(static_cast<const char*>(g.w.codes) + tile.codes + f0 * cfrag,
           mine > 0 ? (int64_t)mine * cfrag : 0);
  const __amdgpu_buffer_rsrc_t pr =
      rsrc(static_cast<const char*>(g.w.params) + tile.params + f0 * pfrag,
           mine > 0 ? (int64_t)mine * pfrag : 0);
  const int bsh = tile.block == 64 ? 6 : (tile.block == 32 ? 5 : 4);
  const uint32_t poff = 64 * ((32 * q) >> bsh) + 4 * (lane & 15);
  const __amdgpu_buffer_rsrc_t xr = rsrc(xb, xbytes);
  auto stage = [&](int st) {
    const uint32_t to = lbase + (uint32_t)(st & 1) * STAGE;
#pragma unroll
    for (int i = 0; i < MF; ++i) dma16(xr, xoff[i], (uint32_t)st * 256, to + i * 1024);
  };
  // The codes of the next stage are fetched a stage ahead; at 8 bits (32 registers a set)
  // a second set would spill, and the stage's own are fetched as it begins.
  constexpr bool AHEAD = BITS < 8;
  struct Codes {
    uint32_t w[NF][BITS], p[NF][2];
  };
  const uint32_t magic = decode_magic();
  auto fetch = [&](int st, Codes& d) {
    const int c = st >> psh;
#pragma unroll
    for (int f = 0; f < NF; ++f) {
      load_codes<BITS>(cr, lane, f * cfrag + (uint32_t)c * (256 * BITS), d.w[f]);
      const uint32_t so = f * pfrag + ((uint32_t)(c * PK_CHUNK) >> bsh) * 64;
      d.p[f][0] = __builtin_amdgcn_raw_buffer_load_b32(pr, (int)poff, (int)so, 0);
      d.p[f][1] =
          B16 ? __builtin_amdgcn_raw_buffer_load_b32(pr, (int)poff + 64, (int)so, 0) : 0u;
    }
  };
  const int t0 = lane & 15;
  const char* xs = lds + t0 * 256;
  const uint32_t piece0 = 16 * ((4 * q) ^ t0);
  auto decode = [&](const Codes& d, int f, int s) {
    const h16x2 ls = __builtin_bit_cast(h16x2, B16 && s >= 2 ? d.p[f][1] : d.p[f][0]);
    return decode_step<BITS>(d.w[f], s, (h16x2){ls[0], ls[0]}, (h16x2){ls[1], ls[1]}, magic);
  };
  // A stage: the codes in `cur`, the next stage's into `nxt`.  What the last stage fetches
  // ahead is never used; it stays inside the resources.
  auto body = [&](int st, Codes& cur, Codes& nxt) {
    // stage st and the codes have landed; behind the barrier nobody reads stage st - 1
    __builtin_amdgcn_s_waitcnt(waitcnt(0, 15));
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    __builtin_amdgcn_s_barrier();
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    if constexpr (!AHEAD) fetch(st, cur);
    const char* x = xs + (st & 1) * STAGE;
    h16x8 b[MF];
#pragma unroll
    for (int m = 0; m < MF; ++m) b[m] = *reinterpret_cast<const h16x8*>(x + m * 4096 + piece0);
    if constexpr (AHEAD) fetch(st + 1, nxt);
    stage(st + 1);
    __builtin_amdgcn_sched_barrier(0);
    h16x8 a = decode(cur, 0, 0);
#pragma unroll
    for (int s = 0; s < 4; ++s) {
#pragma unroll
      for (int f = 0; f < NF; ++f) {
        // the next fragment's weights are decoded between this one's products, and behind
        // its last product of a step an activation register takes the next step's
        const bool more = f + 1 < NF || s + 1 < 4;
        h16x8 an = a;
        if (more) an = decode(cur, f + 1 < NF ? f + 1 : 0, f + 1 < NF ? s : s + 1);
#pragma unroll
        for (int m = 0; m < MF; ++m) {
          acc[f][m] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b[m], acc[f][m], 0, 0, 0);
          if (f == NF - 1 && s < 3)
            b[m] = *reinterpret_cast<const h16x8*>(x + m * 4096 + (piece0 ^ (16 * (s + 1))));
        }
        a = an;
      }
    }
  };
  Codes even, odd;
  if constexpr (AHEAD) fetch(first, even);
  stage(first);
  int st = first;
  for (; st + 1 < nst; st += 2) {
    body(st, even, odd);
    body(st + 1, odd, even);
  }
  if (st < nst) body(st, even, odd);
  // the last stage's transfers into LDS end before the store passes use it
  __builtin_amdgcn_s_waitcnt(waitcnt(0, 15));
}

// Rows u (at most `last`) of one column of an operand, all loads in flight before the first
// conversion: with the type's branch around each single load they would wait in turn (the
// 4096 x 14336 output times its factor: 640 us; so: 490 us).
template <int UN>
__device__ __forceinline__ void load_column(const void* p, int64_t at, int64_t ld, int64_t last,
                                            int dtype, float (&v)[UN]) {
  if (dtype == 0) {
    const float* f = static_cast<const float*>(p) + at;
#pragma unroll
    for (int u = 0; u < UN; ++u) v[u] = f[(u < last ? u : last) * ld];
  } else {
    const uint16_t* h = static_cast<const uint16_t*>(p) + at;
    uint16_t r[UN];
#pragma unroll
    for (int u = 0; u < UN; ++u) r[u] = h[(u < last ? u : last) * ld];
#pragma unroll
    for (int u = 0; u < UN; ++u)
      v[u] = dtype == 1 ? f16_from_bits(r[u]) : __uint_as_float((uint32_t)r[u] << 16);
  }
}

template <int UN>
__device__ __forceinline__ void store_column(void* p, int64_t at, int64_t ld, int64_t last,
                                             int dtype, const float (&v)[UN]) {
#pragma unroll
  for (int u = 0; u < UN; ++u)
    if (u <= last) store_from_f32(p, at + u * ld, dtype, v[u]);
}

// The store of a pass: `rows` rows (from row `o` of the output on) of NS slots, whose sums lie
// in LDS [row][PITCH].  Consecutive threads take consecutive slots, UN rows at a time so that
// their operands are loaded together.
template <int NS, int PITCH, int EH, int UN>
__device__ __forceinline__ void store_pass(const hi2x_epilogue& E, const float* ep,
                                           const float* xscale, int n, float bias, int64_t o0,
                                           int rows) {
  constexpr int TPR = NS < 256 ? NS : 256;  // threads on one row
  static_assert(EH % UN == 0, "whole batches");
  const int slot = threadIdx.x % TPR;
  if (n < 0) return;
  for (int t0 = threadIdx.x / TPR * UN; t0 < rows; t0 += 256 / TPR * UN) {
    const int64_t o = o0 + t0;
    const int64_t last = rows - 1 - t0;  // rows past the end repeat the last one's loads
    float y[UN], mu[UN], re[UN];
    if (E.mul) load_column(E.mul, o * E.ld_mul + n, E.ld_mul, last, E.dt_mul, mu);
    if (E.residual)
      load_column(E.residual, o * E.ld_residual + n, E.ld_residual, last, E.dt_residual, re);
#pragma unroll
    for (int u = 0; u < UN; ++u) y[u] = ep[(t0 + u) * PITCH + slot] * xscale[t0 + u] + bias;
    activate_all(y, E.act);
    if (E.mul) {
#pragma unroll
      for (int u = 0; u < UN; ++u) y[u] = y[u] * mu[u];
    }
    if (E.residual) {
#pragma unroll
      for (int u = 0; u < UN; ++u) y[u] = y[u] + re[u];
    }
    store_column(E.out, o * E.ld_out + n, E.ld_out, last, E.dt_out, y);
  }
}

// The store of a pass of a product with exponents: the slots as they lie, 8 to a thread and two
// threads to a fragment, from slot `at` of the output's rows on.  (The exponents cost the products
// of 64 experts at 16384 tokens 2 to 3 %; several rows of a thread at a time no less.)
template <int NS, int PITCH>
__device__ __forceinline__ void store_slots(const GemmArgs& g, const float* ep, int at, int slots,
                                            int64_t o0, int rows) {
  constexpr int TPR = NS / 8;
  const int slot = threadIdx.x % TPR * 8;
  if (slot >= slots) return;
  const hi2x_epilogue& E = g.epi;
  uint16_t* out = static_cast<uint16_t*>(E.out) + o0 * E.ld_out + at + slot;
  int8_t* exps = g.exps + o0 * g.ep + (at + slot) / 16;
  for (int t = threadIdx.x / TPR; t < rows; t += 256 / TPR) {
    const f32x4v* from = reinterpret_cast<const f32x4v*>(ep + t * PITCH + slot);
    const f32x4v a = from[0], b = from[1];
    float m = 0.0f;  // the largest finite one (NaN is passed over)
#pragma unroll
    for (int i = 0; i < 4; ++i) m = fmaxf(m, fmaxf(fabsf(a[i]), fabsf(b[i])));
    if (m == __builtin_inff()) {
      m = 0.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float x = fabsf(i < 4 ? a[i] : b[i - 4]);
        m = fmaxf(m, x < __builtin_inff() ? x : 0.0f);
      }
    }
    m = fmaxf(m, __int_as_float(dpp<0xB1>(__float_as_int(m))));
    // by the bits of m: 2^(e - 127) <= m < 2^(e - 126), and 2^c is a normal float
    const int c = m > 0.0f ? imax_((__float_as_int(m) >> 23) - 141, EXP_LEAST) : 0;
    const float scale = __int_as_float((127 - c) << 23);  // 2^-c
    u32x4 v;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float x = i < 2 ? a[2 * i] : b[2 * i - 4], y = i < 2 ? a[2 * i + 1] : b[2 * i - 3];
      v[i] = (uint32_t)f16_bits(x * scale) | (uint32_t)f16_bits(y * scale) << 16;
    }
    *reinterpret_cast<u32x4*>(out + t * E.ld_out) = v;
    if (!(slot & 8)) exps[t * g.ep] = (int8_t)c;
  }
}

// Row `t` of a tile's factor of scale: 0 past the end, NaN for an index outside.
__device__ __forceinline__ float row_scale(const GemmArgs& g, int64_t first, int t, int live) {
  if (t >= live) return 0.0f;
  const int64_t r = g.src ? g.src[first + t] : first + t;
  return r >= 0 && r < g.x.rows ? g.x.scale[r] : __builtin_nanf("");
}

// The work of a workgroup: its expert, tile of fragments and tile of activation rows.  Of
// several experts the grid is (tiles x tiles of rows) long: workgroups go to the eight XCDs
// in turn, so an XCD takes all tiles of four neighbouring row tiles one after the other, and
// the rows (and mostly the expert's weights) come to its L2 once.
template <int NF, int MF>
__device__ __forceinline__ bool find(const GemmArgs& g, int nx, Tile& tile, int64_t& first,
                                     int& live) {
  int x = blockIdx.x;
  int64_t y = blockIdx.y;
  if (g.offs) {
    const int xcd = x & 7, j = x >> 3, r = j / nx;
    x = j - r * nx;
    y = ((int64_t)(r >> 2) * 8 + xcd) * 4 + (r & 3);
  }
  const PkWork wk = find_work(g.offs, (int)g.w.experts, g.slots, 16 * MF, y);
  const int e = __builtin_amdgcn_readfirstlane(wk.e);
  if (e < 0) return false;
  if (!find_tile(g.w, e, x, 4 * NF, tile)) return false;
  first = __builtin_amdgcn_readfirstlane((int)wk.first);  // slots < 2^31
  const int64_t left = __builtin_amdgcn_readfirstlane((int)wk.end) - first;
  live = (int)(left < 16 * MF ? left : 16 * MF);
  return true;
}

__device__ __forceinline__ int slot_row(const GemmArgs& g, const Tile& tile, int slot) {
  return slot < 16 * tile.count
             ? g.w.rows[(int64_t)tile.frag * 16 + slot]
             : -1;
}

// The least of MOST, its half and its quarter that holds n.
template <int MOST>
__device__ __forceinline__ int share_of(int n) {
  if (MOST >= 4 && n <= MOST / 4) return MOST / 4;
  return MOST >= 2 && n <= MOST / 2 ? MOST / 2 : MOST;
}

// The loop for the tile's own nf fragments a wave and 16 mf rows: an expert's last rows and a
// class's last fragments fill a tile in part only, and most tiles of a small batch are such
// (64 experts, 8 choices: 64 tokens 127 us in whole tiles and 107 so, 2048 tokens 433 and
// 417).  (128 x 64 tiles share by rows alone: both would not fit their registers.)
template <int BITS, bool B16, int N, int M, int NF, int MF>
__device__ __forceinline__ void sized_loop(const GemmArgs& g, const Tile& tile, char* lds,
                                           const char* xb, int64_t xbytes,
                                           const uint32_t (&xoff)[MF], int nf, int mf, int c0,
                                           int c1, f32x4v (&acc)[NF][MF]) {
  if constexpr (NF != 2 && N > 1 && 4 * N > NF) {
    if (nf < N)
      return sized_loop<BITS, B16, N / 2, M>(g, tile, lds, xb, xbytes, xoff, nf, mf, c0, c1, acc);
  }
  if constexpr (M > 1 && 4 * M > MF) {
    if (mf < M)
      return sized_loop<BITS, B16, N, M / 2>(g, tile, lds, xb, xbytes, xoff, nf, mf, c0, c1, acc);
  }
  gemm_loop<BITS, B16, N, M>(g, tile, lds, xb, xbytes, xoff, c0, c1, acc);
}

// One workgroup: 64 NF slots of w's layout (one segment) x 16 MF activation rows, over all
// columns or (SPLIT) the blockIdx.z-th share of their chunks.  A split's sums go to `part` as
// the accumulators hold them.
template <int NF, int MF, bool SPLIT>
__global__ __launch_bounds__(256, NF == 4 ? 2 : 4)
void packed_gemm_kernel(GemmPair two, float* part, int per, int nx) {
  const GemmArgs& g = two.g[SPLIT ? 0 : blockIdx.z];
  constexpr int MT = 16 * MF, NS = 64 * NF;
  constexpr int XB = 2 * MT * 256;  // two stages of activations
  constexpr int PITCH = NS + 4;     // floats of one row in LDS: rows 4 banks apart
  // rows of a store pass: what two stages' room holds (and the pitch a little more)
  constexpr int EH = NS * 4 * MT <= XB ? MT : XB / (NS * 4);
  constexpr int LB = EH * PITCH * 4 > XB ? EH * PITCH * 4 : XB;
  static_assert(EH % 16 == 0 && MT % EH == 0, "store passes");
  __shared__ __attribute__((aligned(1024))) char lds[LB];
  __shared__ float xscale[MT];
  Tile tile;
  int64_t first;
  int live;
  if (!find<NF, MF>(g, nx, tile, first, live)) return;
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
  const int nf = SPLIT || NF == 2 ? NF : share_of<NF>((tile.count + 3) / 4);
  const int mf = SPLIT ? MF : share_of<MF>((live + 15) / 16);
  // Where the rows this lane stages begin.  Rows past the end read zeros or another
  // tile's, and are not stored; indices outside the activations read row 0 (and come out as
  // NaN below).  Without src the resource begins at the tile's own rows.
  uint32_t xoff[MF];
  const uint32_t pitch = (uint32_t)g.x.kp * 2 * g.x.nplanes;
  const int64_t row0 = g.src ? 0 : first;
  const char* xb = reinterpret_cast<const char*>(g.x.planes) + row0 * pitch;
  const int64_t xbytes = (g.x.rows - row0) * pitch;
#pragma unroll
  for (int i = 0; i < MF; ++i) {
    const int t = 4 * (wv * mf + i) + (lane >> 4);
    int64_t r = t;
    if (g.src) {
      r = t < live ? g.src[first + t] : 0;
      if (r < 0 || r >= g.x.rows) r = 0;
    }
    xoff[i] = (uint32_t)r * pitch + 16 * ((lane & 15) ^ (t & 15));
  }
  if (tid < MT) xscale[tid] = row_scale(g, first, tid, live);
  const int nch = (int)(g.w.kp / PK_CHUNK);
  const int c0 = SPLIT ? (int)blockIdx.z * per : 0;
  const int c1 = SPLIT && c0 + per < nch ? c0 + per : nch;
  f32x4v acc[NF][MF];
#pragma unroll
  for (int f = 0; f < NF; ++f)
#pragma unroll
    for (int m = 0; m < MF; ++m) acc[f][m] = f32x4v{0.0f, 0.0f, 0.0f, 0.0f};
#define HI2X_LOOP(BITS, B16)                                                                \
  if constexpr (SPLIT)                                                                    \
    gemm_loop<BITS, B16, NF, MF>(g, tile, lds, xb, xbytes, xoff, c0, c1, acc);            \
  else                                                                                    \
    sized_loop<BITS, B16, NF, MF>(g, tile, lds, xb, xbytes, xoff, nf, mf, c0, c1, acc);   \
  break;
  switch (2 * tile.nbits + (tile.block == 16)) {
    case 4:
      HI2X_LOOP(2, false)
    case 5:
      HI2X_LOOP(2, true)
    case 8:
      HI2X_LOOP(4, false)
    case 9:
      HI2X_LOOP(4, true)
    case 16:
      HI2X_LOOP(8, false)
    default:
      HI2X_LOOP(8, true)
  }
#undef HI2X_LOOP
  if constexpr (SPLIT) {
    float* to = part + ((((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * gridDim.z +
                         blockIdx.z) * MF * 4 * NF) * 256;
#pragma unroll
    for (int m = 0; m < MF; ++m)
#pragma unroll
      for (int f = 0; f < NF; ++f)
        *reinterpret_cast<f32x4v*>(to + ((m * 4 + wv) * NF + f) * 256 + 4 * lane) = acc[f][m];
    return;
  }
  float* ep = reinterpret_cast<float*>(lds);
  const int n = slot_row(g, tile, tid % (NS < 256 ? NS : 256));
  const float bias = g.epi.bias && n >= 0 ? load_as_f32(g.epi.bias, n, g.epi.dt_bias) : 0.0f;
#pragma unroll
  for (int p = 0; p < MT / EH; ++p) {
    if (p * EH >= live) break;
    __syncthreads();
#pragma unroll
    for (int m = 0; m < EH / 16; ++m)
#pragma unroll
      for (int f = 0; f < NF; ++f)
        if (f < nf)
          *reinterpret_cast<f32x4v*>(ep + (16 * m + (lane & 15)) * PITCH + (wv * nf + f) * 16 +
                                     4 * (lane >> 4)) = acc[f][p * (EH / 16) + m];
    __syncthreads();
    const int rows = live - p * EH < EH ? live - p * EH : EH;
    if (g.exps)
      store_slots<NS, PITCH>(g, ep, 16 * (tile.frag - tile.base), 16 * tile.count, first + p * EH,
                             rows);
    else
      store_pass<NS, PITCH, EH, 8>(g.epi, ep, xscale + p * EH, n, bias, first + p * EH, rows);
  }
}

// The splits' sums of 16 rows of a tile (blockIdx.z), added in their order, and the epilogue.
template <int NF, int MF>
__global__ __launch_bounds__(256) void packed_join_kernel(GemmArgs g, const float* part,
                                                          int splits) {
  constexpr int NS = 64 * NF, PITCH = NS + 4;
  __shared__ __attribute__((aligned(16))) float ep[16 * PITCH];
  __shared__ float xscale[16];
  Tile tile;
  int64_t first;
  int live;
  if (!find<NF, MF>(g, 1, tile, first, live)) return;
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6, m = blockIdx.z;
  const int rows = live - 16 * m < 16 ? live - 16 * m : 16;
  if (rows <= 0) return;
  const float* from = part + ((((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * splits) * MF * 4 *
                              NF) * 256;
  f32x4v sum[NF];
#pragma unroll
  for (int f = 0; f < NF; ++f) sum[f] = f32x4v{0.0f, 0.0f, 0.0f, 0.0f};
  for (int z = 0; z < splits; ++z)
#pragma unroll
    for (int f = 0; f < NF; ++f)
      sum[f] += *reinterpret_cast<const f32x4v*>(
          from + (((int64_t)z * MF + m) * 4 * NF + wv * NF + f) * 256 + 4 * lane);
#pragma unroll
  for (int f = 0; f < NF; ++f)
    *reinterpret_cast<f32x4v*>(ep + (lane & 15) * PITCH + (wv * NF + f) * 16 + 4 * (lane >> 4)) =
        sum[f];
  if (tid < 16) xscale[tid] = row_scale(g, first, 16 * m + tid, live);
  __syncthreads();
  const int n = slot_row(g, tile, tid % (NS < 256 ? NS : 256));
  const float bias = g.epi.bias && n >= 0 ? load_as_f32(g.epi.bias, n, g.epi.dt_bias) : 0.0f;
  store_pass<NS, PITCH, 16, NF == 2 ? 8 : 4>(g.epi, ep, xscale, n, bias, first + 16 * m, rows);
}

template <int NF, int MF>
int launch_gemm(const GemmPair& g, int count, float* part, int splits, int per, dim3 grid,
                int nx, hipStream_t s) {
  if (splits == 1) {
    grid.z = count;
    packed_gemm_kernel<NF, MF, false><<<grid, 256, 0, s>>>(g, nullptr, 0, nx);
  } else {
    grid.z = splits;
    packed_gemm_kernel<NF, MF, true><<<grid, 256, 0, s>>>(g, part, per, nx);
    grid.z = MF;
    packed_join_kernel<NF, MF><<<grid, 256, 0, s>>>(g.g[0], part, splits);
  }
  return launch_status("packed_linear");
}

// Which tiles a product takes: 64 nf slots x 16 mf rows, the chunks in `splits` shares of
// `per`.
struct GemmPlan {
  int nf, mf, splits, per;
  int64_t nx, ny;
  int64_t part_bytes() const {
    return splits == 1 ? 0 : nx * ny * splits * mf * nf * 4 * 1024;
  }
};

// Large tiles feed the matrix units best, but only where there are enough of them: 256 x 128
// (two workgroups a CU) reaches 1020 TFLOP/s at 14336 x 4096 and 4096 rows, but takes 2 us a
// chunk where a workgroup has its CU to itself.  The choice is the least of the estimates
//   5.5 us + chunks x (a + b x workgroups on a CU), for each round of them,
// and for splits the joining pass, 3.5 us + 0.45 us a share + the partial sums at 4.5 TB/s.
// a and b (us a chunk) are measured.  4096 x 4096 at 128 rows takes 70 us in 256 x 128 tiles,
// 19 in 128 x 64 or 64 x 64 ones with the columns in four shares; 4096 x 14336 at 1000 rows
// 232 us, 153 in 128 x 64 tiles and four shares.
GemmPlan plan_gemm(const hi2x_packed& w, int64_t slots, bool ranges, int npl) {
  struct Tiles {
    int nf, mf, cap;  // workgroups a CU holds
    double a, b;
  };
  static constexpr Tiles kTiles[3] = {{4, 8, 2, 0.6, 1.65}, {2, 4, 4, 0.25, 0.55},
                                      {1, 4, 4, 0.35, 0.28}};
  const int nch = (int)(w.kp / PK_CHUNK);
  GemmPlan best{};
  double least = 0.0;
  for (const Tiles& t : kTiles) {
    GemmPlan p{t.nf, t.mf, 1, nch, 0, 0};
    const int64_t mt = 16 * t.mf;
    p.nx = w.max_tiles[t.nf == 1 ? 0 : (t.nf == 2 ? 1 : 2)];
    // every expert can leave one tile partly filled
    const int64_t part = ranges ? (w.experts < slots ? w.experts : slots) : 1;
    p.ny = ranges ? slots / mt + part : (slots + mt - 1) / mt;
    const double tiles = (double)p.nx * (ranges ? (double)slots / mt + 0.5 * part : (double)p.ny);
    for (int s = 1; s <= 16; ++s) {
      if (s > 1 && (ranges || t.nf == 4 || nch < 2 * s)) break;
      p.per = (nch + s - 1) / s;
      p.splits = (nch + p.per - 1) / p.per;
      if (p.splits != s) continue;
      const double groups = tiles * s;
      const double whole = __builtin_floor(groups / (256.0 * t.cap));
      const double rest = groups - whole * 256.0 * t.cap;
      double us = whole * (t.a + t.b * t.cap);
      if (rest > 0) us += t.a + t.b * __builtin_ceil(rest / 256);
      us = 5.5 + us * p.per * npl;
      if (s > 1) us += 3.5 + 0.45 * s + groups * t.nf * t.mf * 4096 / 4.5e6;
      if (least == 0.0 || us < least) {
        least = us;
        best = p;
      }
    }
  }
  return best;
}

}  // namespace

// Rows of one launch without ranges: a grid holds 65535 tiles of them.  More go in parts.
constexpr int64_t MOST_ROWS = 65535 * 64;

int64_t packed_part_bytes(const hi2x_packed& w, int64_t slots, bool ranges, int npl) {
  if (few_rows_product(slots, ranges)) return 0;
  if (!ranges && slots > MOST_ROWS) {
    const int64_t a = packed_part_bytes(w, MOST_ROWS, ranges, npl);
    const int64_t b = packed_part_bytes(w, (slots - 1) % MOST_ROWS + 1, ranges, npl);
    return a > b ? a : b;
  }
  return plan_gemm(w, slots, ranges, npl).part_bytes();
}

namespace {
// Rows [first, first + n) of a product without ranges.
GemmArgs part_of(GemmArgs g, int64_t first, int64_t n) {
  auto at = [&](const void* p, int64_t ld, int dtype) {
    return p ? static_cast<const char*>(p) + first * ld * (dtype == 0 ? 4 : 2) : nullptr;
  };
  hi2x_epilogue& e = g.epi;
  e.mul = at(e.mul, e.ld_mul, e.dt_mul);
  e.residual = at(e.residual, e.ld_residual, e.dt_residual);
  e.out = const_cast<char*>(at(e.out, e.ld_out, e.dt_out));
  g.slots = n;
  if (g.src) {
    g.src += first;
  } else {
    g.x.planes += first * g.x.kp * g.x.nplanes;
    g.x.scale += first;
    g.x.rows -= first;
  }
  return g;
}
}  // namespace

int packed_product(const GemmPair& two, int count, void* work, int64_t work_bytes,
                   hipStream_t s) {
  const GemmArgs& g = two.g[0];
  if (!g.offs && g.slots > MOST_ROWS) {
    for (int64_t first = 0; first < g.slots; first += MOST_ROWS) {
      const int64_t left = g.slots - first;
      const GemmArgs p = part_of(g, first, left < MOST_ROWS ? left : MOST_ROWS);
      if (int rc = packed_product(GemmPair{{p, p}}, 1, work, work_bytes, s)) return rc;
    }
    return HI2X_OK;
  }
  if (few_rows_product(g.slots, g.offs)) return packed_few(g, s);
  const GemmPlan p = plan_gemm(g.w, g.slots, g.offs, g.x.nplanes);
  int64_t nx = p.nx;
  if (count > 1) {
    const int64_t* m = two.g[1].w.max_tiles;
    const int64_t other = m[p.nf == 1 ? 0 : (p.nf == 2 ? 1 : 2)];
    nx = nx > other ? nx : other;
  }
  const int64_t padded = (p.ny + 31) / 32 * 32;  // whole rounds of four tiles to each XCD
  HI2X_REQUIRE(nx < (1ll << 31) && (g.offs ? nx * padded < (1ll << 31) : p.ny <= 65535),
               "packed_linear: %lld rows are too many", (long long)g.slots);
  Workspace ws;
  if (int rc = take_workspace(ws, work, work_bytes, (size_t)p.part_bytes(), s, "packed_linear"))
    return rc;
  float* part = reinterpret_cast<float*>(ws.p);
  const dim3 grid((unsigned)(g.offs ? nx * padded : nx), (unsigned)(g.offs ? 1 : p.ny),
                  (unsigned)count);
  if (p.nf == 4) {
    packed_gemm_kernel<4, 8, false><<<grid, 256, 0, s>>>(two, nullptr, 0, (int)nx);
    return launch_status("packed_linear");
  }
  return p.nf == 2 ? launch_gemm<2, 4>(two, count, part, p.splits, p.per, grid, (int)nx, s)
                   : launch_gemm<1, 4>(two, count, part, p.splits, p.per, grid, (int)nx, s);
}

}  // namespace hi2x

using namespace hi2x;

extern "C" int hi2x_packed_linear_activations(const hi2x_packed* w, const hi2x_activations* x,
                                              const int64_t* src, const int64_t* offs,
                                              int64_t slots, const hi2x_epilogue* epi, void* work,
                                              int64_t work_bytes, void* stream) {
  clear_error();
  HI2X_REQUIRE(w && x && epi, "packed_linear: null argument");
  if (int rc = check_packed(w, "packed_linear")) return rc;
  if (int rc = check_product(w, src, offs, slots, x->rows, epi, "packed_linear")) return rc;
  HI2X_REQUIRE(x->kp == w->kp, "packed_linear: activations of %lld padded columns, %lld needed",
               (long long)x->kp, (long long)w->kp);
  HI2X_REQUIRE(x->nplanes == 1 || x->nplanes == 2, "packed_linear: %d planes", x->nplanes);
  HI2X_REQUIRE(!src || x->rows * x->kp * 2 * x->nplanes < (1ll << 32) - 1,
               "packed_linear: 4 GiB of activations or more cannot be taken by index");
  if (slots == 0) return HI2X_OK;
  HI2X_REQUIRE(x->rows > 0 && x->planes && x->scale, "packed_linear: null activations");
  HI2X_REQUIRE(((uintptr_t)x->planes & 255) == 0, "packed_linear: planes not aligned");
  const GemmArgs g{*w, *x, src, offs, slots, *epi};
  return packed_product(GemmPair{{g, g}}, 1, work, work_bytes, as_stream(stream));
}

extern "C" int hi2x_packed_linear(const hi2x_packed* w, const void* x, int dtype, int64_t ldx,
                                  int64_t x_rows, int nplanes, const int64_t* src,
                                  const int64_t* offs, int64_t slots, const hi2x_epilogue* epi,
                                  void* work, int64_t work_bytes, void* stream) {
  clear_error();
  HI2X_REQUIRE(w && epi, "packed_linear: null argument");
  if (int rc = check_packed(w, "packed_linear")) return rc;
  if (int rc = check_product(w, src, offs, slots, x_rows, epi, "packed_linear")) return rc;
  if (int rc = check_x(x, dtype, ldx, x_rows, w->k, "packed_linear")) return rc;
  HI2X_REQUIRE(nplanes == 1 || nplanes == 2, "packed_linear: %d planes", nplanes);
  if (slots == 0) return HI2X_OK;
  const hipStream_t s = as_stream(stream);
  const RawRows raw{x, dtype, ldx, x_rows, nplanes};
  GemmArgs g{*w, hi2x_activations{}, src, offs, slots, *epi};
  if (few_raw_product(slots, offs)) return packed_few_raw(GemmPair{{g, g}}, 1, raw, s);
  const bool each = transform_slots(*w, x_rows);
  const int64_t rows = transform_rows(*w, x_rows, src, slots);
  HI2X_REQUIRE(rows < (1ll << 31), "packed_linear: too many rows");
  HI2X_REQUIRE(!src || each || rows * w->kp * 2 * nplanes < (1ll << 32) - 1,
               "packed_linear: 4 GiB of activations or more cannot be taken by index");
  Workspace ws;
  const int64_t need = hi2x_packed_workspace_bytes(w, x_rows, nplanes, 0, slots, src != nullptr,
                                                   offs != nullptr);
  if (int rc = take_workspace(ws, work, work_bytes, (size_t)need, s, "packed_linear")) return rc;
  const int64_t pb = plane_bytes(*w, rows, nplanes);
  g.x = hi2x_activations{reinterpret_cast<uint16_t*>(ws.p), reinterpret_cast<float*>(ws.p + pb),
                         rows, w->kp, nplanes, 0};
  if (int rc = launch_activations(raw, *w, each ? src : nullptr, w->per_expert ? offs : nullptr,
                                  g.x, s))
    return rc;
  if (each) g.src = nullptr;
  const int64_t used = pb + align256(rows * 4);
  return packed_product(GemmPair{{g, g}}, 1, ws.p + used, need - used, s);
}

extern "C" int64_t hi2x_packed_workspace_bytes(const hi2x_packed* w, int64_t x_rows, int nplanes,
                                               int given, int64_t slots, int indexed,
                                               int ranges) {
  if (!w || check_packed(w, "packed_workspace_bytes") != HI2X_OK || slots < 0 || x_rows < 0 ||
      nplanes < 1 || nplanes > 2)
    return -1;
  if (slots == 0) return 0;
  int64_t front = 0;
  if (!given) {
    if (few_raw_product(slots, ranges)) return 0;
    const int64_t rows = transform_rows(*w, x_rows, indexed, slots);
    front = plane_bytes(*w, rows, nplanes) + align256(rows * 4);
  }
  return front + packed_part_bytes(*w, slots, ranges, nplanes);
}

// ---- the gated MLP of experts ------------------------------------------------------------
namespace {

// Where the parts of hi2x_moe_mlp's workspace begin.
struct MlpSpace {
  bool half;                    // gate, up and y with exponents, else f32
  int64_t gate, up, y;          // [slots][i], [slots][i], [slots][h]
  int64_t exps[3];              // their fragments' exponents
  int64_t in[2], in_scale[2];   // the transformed tokens: shared, or per tensor
  int64_t mid, mid_scale;       // the transformed hidden values
  int64_t in_rows[2];
  int64_t bytes;
};

MlpSpace mlp_space(const hi2x_packed& gate, const hi2x_packed& up, const hi2x_packed& down,
                   int64_t t, int64_t slots, int npl, int npl_mid, bool shared) {
  MlpSpace m{};
  int64_t at = 0;
  auto take = [&](int64_t n) {
    const int64_t a = at;
    at += align256(n);
    return a;
  };
  // A bf16 result hides the rounding to fp16 (2^-11) as it hides that of one plane;
  // writing and reading the three is what the large calls are short of: 64 experts of
  // 2048 x 1024, 8 choices, 16384 tokens 2680 us in f32, 2100 so.  Short calls keep f32.
  m.half = npl_mid == 1 && !few_raw_product(slots, true);
  for (const hi2x_packed* p : {&gate, &up, &down})
    m.half = m.half && p->places && 16 * p->max_frags <= SLOTS16 &&
             16 * p->max_frags <= p->n + 16 * PK_SEGS;  // (as many as the readers' loads take)
  const int64_t size = m.half ? 2 : 4;
  m.gate = take(slots * (m.half ? 16 * gate.max_frags : gate.n) * size);
  m.up = take(slots * (m.half ? 16 * up.max_frags : gate.n) * size);
  m.y = take(slots * (m.half ? 16 * down.max_frags : down.n) * size);
  const hi2x_packed* of[3] = {&gate, &up, &down};
  for (int i = 0; i < 3 && m.half; ++i) m.exps[i] = take(slots * exps_pitch(*of[i]));
  if (!few_raw_product(slots, true)) {
    for (int i = 0; i < (shared ? 1 : 2); ++i) {
      m.in_rows[i] = (i ? up : gate).per_expert ? slots : t;
      m.in[i] = take(plane_bytes(gate, m.in_rows[i], npl));
      m.in_scale[i] = take(m.in_rows[i] * 4);
    }
    m.mid = take(plane_bytes(down, slots, npl_mid));
    m.mid_scale = take(slots * 4);
  }
  m.bytes = at;
  return m;
}

int check_mlp(const hi2x_packed* gate, const hi2x_packed* up, const hi2x_packed* down,
              int64_t slots, int npl, int npl_mid) {
  if (int rc = check_packed(gate, "moe_mlp")) return rc;
  if (int rc = check_packed(up, "moe_mlp")) return rc;
  if (int rc = check_packed(down, "moe_mlp")) return rc;
  HI2X_REQUIRE(gate->n == up->n && gate->k == up->k && gate->n == down->k && gate->k == down->n &&
                   gate->experts == up->experts && gate->experts == down->experts,
               "moe_mlp: gate and up [i, h] and down [h, i] of the same experts expected");
  HI2X_REQUIRE(slots >= 0 && slots < (1ll << 31), "moe_mlp: bad shape");
  HI2X_REQUIRE((npl == 1 || npl == 2) && (npl_mid == 1 || npl_mid == 2), "moe_mlp: %d, %d planes",
               npl, npl_mid);
  return HI2X_OK;
}

}  // namespace

extern "C" int64_t hi2x_moe_mlp_workspace_bytes(const hi2x_packed* gate, const hi2x_packed* up,
                                                const hi2x_packed* down, int64_t t, int64_t top_k,
                                                int nplanes, int nplanes_mid, int shared) {
  if (t < 0 || top_k < 1 || check_mlp(gate, up, down, t * top_k, nplanes, nplanes_mid)) return -1;
  return mlp_space(*gate, *up, *down, t, t * top_k, nplanes, nplanes_mid, shared).bytes;
}

extern "C" int hi2x_moe_mlp(const hi2x_packed* gate, const hi2x_packed* up,
                            const hi2x_packed* down, const void* x, int dtype, int64_t ldx,
                            int64_t t, int64_t top_k, int nplanes, int nplanes_mid, int shared,
                            int act, const int64_t* rows, const int64_t* offs,
                            const int64_t* slots, const float* weights, const void* residual,
                            int dt_residual, void* out, int dt_out, void* ws, int64_t ws_bytes,
                            void* stream) {
  clear_error();
  HI2X_REQUIRE(t >= 0 && top_k >= 1 && top_k < (1 << 20), "moe_mlp: bad shape");
  const int64_t n = t * top_k;
  if (int rc = check_mlp(gate, up, down, n, nplanes, nplanes_mid)) return rc;
  if (int rc = check_x(x, dtype, ldx, t, gate->k, "moe_mlp")) return rc;
  HI2X_REQUIRE(act >= HI2X_ACT_NONE && act <= HI2X_ACT_GELU_TANH, "moe_mlp: activation %d", act);
  for (int d : {dt_residual, dt_out})
    HI2X_REQUIRE(d >= 0 && d <= 2, "moe_mlp: dtype %d", d);
  if (t == 0) return HI2X_OK;
  HI2X_REQUIRE(rows && offs && slots && weights && out, "moe_mlp: null buffer");
  HI2X_REQUIRE(t * gate->kp * 2 * nplanes < (1ll << 32) - 1 || few_raw_product(n, true),
               "moe_mlp: 4 GiB of activations or more cannot be taken by index");
  const hipStream_t s = as_stream(stream);
  const MlpSpace m = mlp_space(*gate, *up, *down, t, n, nplanes, nplanes_mid, shared);
  Workspace w;
  if (int rc = take_workspace(w, ws, ws_bytes, (size_t)m.bytes, s, "moe_mlp")) return rc;
  auto product = [&](const hi2x_packed& p, const int64_t* src, int64_t at, int64_t exps) {
    GemmArgs g{p, hi2x_activations{}, src, offs, n, hi2x_epilogue{}};
    g.epi.out = w.p + at;
    g.epi.ld_out = m.half ? 16 * p.max_frags : p.n;
    if (m.half) {
      g.exps = reinterpret_cast<int8_t*>(w.p + exps);
      g.ep = exps_pitch(p);
    }
    return g;
  };
  GemmPair in{{product(*gate, rows, m.gate, m.exps[0]), product(*up, rows, m.up, m.exps[1])}};
  GemmArgs last = product(*down, nullptr, m.y, m.exps[2]);
  const RawRows tokens{x, dtype, ldx, t, nplanes};
  RawRows hidden{w.p + m.gate, 0, gate->n, n, nplanes_mid,
                 reinterpret_cast<const float*>(w.p + m.up), act};
  SlotRows results;
  if (few_raw_product(n, true)) {
    if (int rc = packed_few_raw(in, 2, tokens, s)) return rc;
    if (int rc = packed_few_raw(GemmPair{{last, last}}, 1, hidden, s)) return rc;
  } else {
    for (int i = 0; i < 2; ++i) {
      const hi2x_packed& p = in.g[i].w;
      const int j = shared ? 0 : i;
      in.g[i].x = hi2x_activations{reinterpret_cast<uint16_t*>(w.p + m.in[j]),
                                   reinterpret_cast<float*>(w.p + m.in_scale[j]), m.in_rows[j],
                                   p.kp, nplanes, 0};
      if (i == j)
        if (int rc = launch_activations(tokens, p, p.per_expert ? rows : nullptr,
                                        p.per_expert ? offs : nullptr, in.g[i].x, s))
          return rc;
      if (p.per_expert) in.g[i].src = nullptr;
    }
    if (m.half) {
      auto rows_of = [](const GemmArgs& g) {
        return SlotRows{static_cast<const uint16_t*>(g.epi.out), (int)g.epi.ld_out, g.w.places,
                        g.exps, g.ep, g.x.scale, g.src, g.x.rows, g.w.n};
      };
      hidden.s1 = rows_of(in.g[0]);
      hidden.s2 = rows_of(in.g[1]);
      hidden.offs = offs;
      last.x.scale = reinterpret_cast<float*>(w.p + m.mid_scale);
      last.x.rows = n;
      results = rows_of(last);
    }
    if (int rc = packed_product(in, 2, nullptr, 0, s)) return rc;
    last.x = hi2x_activations{reinterpret_cast<uint16_t*>(w.p + m.mid),
                              reinterpret_cast<float*>(w.p + m.mid_scale), n, down->kp,
                              nplanes_mid, 0};
    if (int rc = launch_activations(hidden, *down, nullptr, down->per_expert ? offs : nullptr,
                                    last.x, s))
      return rc;
    if (int rc = packed_product(GemmPair{{last, last}}, 1, nullptr, 0, s)) return rc;
  }
  if (m.half)
    return launch_combine(results, offs, (int)down->experts, n, slots, weights, t, top_k, residual,
                          dt_residual, out, dt_out, s);
  return launch_combine(w.p + m.y, 0, n, down->n, slots, weights, t, top_k, residual, dt_residual,
                        out, dt_out, s);
}
