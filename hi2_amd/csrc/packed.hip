// Packed tensors laid out for products, and the activations' transform in front of them.
#include "packed.h"

namespace hi2x {
namespace {

// ---- layout ------------------------------------------------------------------------------
// One thread per (fragment, chunk, lane): the 32 codes a lane feeds to the chunk's four
// MFMA steps are 32 neighbours of its row, nbits whole words.  In each laid-out dword the
// pair p of codes (2p, 2p + 1) sits at bits nbits * p and 16 + nbits * p, so that one mask
// takes a pair out as two halves.  At nbits 8 a lane's 32 bytes go as two 16-byte pieces,
// 64 lanes of each next to each other.
__global__ __launch_bounds__(256) void layout_codes_kernel(hi2x_packed w,
                                                           const int32_t* __restrict__ codes,
                                                           const int64_t* __restrict__ code_off) {
  const hi2x_packed_segment sg = w.segments[blockIdx.y];
  const int64_t e = blockIdx.y / PK_SEGS;
  const int64_t nch = w.kp / PK_CHUNK;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i == 0 && blockIdx.y == 0) *w.largest = 0.0f;  // (layout_params_kernel comes next)
  if (i >= sg.frags * nch * 64) return;
  const int lane = (int)(i & 63);
  const int64_t c = (i >> 6) % nch, f = (i >> 6) / nch;
  const int nbits = sg.nbits, per = 32 / nbits;
  const int row = w.rows[(sg.frag0 + f) * 16 + (lane & 15)];
  const int64_t k0 = c * PK_CHUNK + 32 * (lane >> 4);
  const int64_t left = w.k - k0;  // columns there are, a multiple of 16
  const int words = row < 0 || left <= 0 ? 0 : (int)(left >= 32 ? nbits : left * nbits / 32);
  const int32_t* src = row < 0 ? codes : codes + code_off[e * w.n + row] + k0 * nbits / 32;
  uint32_t* dst = reinterpret_cast<uint32_t*>(static_cast<char*>(w.codes) + sg.codes +
                                              (f * nch + c) * 256 * nbits);
  for (int q = 0; q < nbits; ++q) {
    uint32_t v = q < words ? (uint32_t)src[q] : 0u, o = 0;
    const uint32_t m = (1u << nbits) - 1u;
    for (int j = 0; j < per; ++j)
      o |= ((v >> (nbits * j)) & m) << (nbits * (j >> 1) + 16 * (j & 1));
    const int at = nbits == 8 ? (q >> 2) * 256 + lane * 4 + (q & 3) : lane * nbits + q;
    dst[at] = o;
  }
}

// One thread per (fragment, block, row): the block's fp16 lo and step (hi2/format.py:45-60:
// lo = fp16(f32(f64(u) lo_scale + lo_min)); the product of a byte and an fp16 is exact in
// f32, so one f32 fma rounds as the f64 sum does).
__global__ __launch_bounds__(256) void layout_params_kernel(
    hi2x_packed w, const uint8_t* __restrict__ params, const int64_t* __restrict__ param_off,
    const uint16_t* __restrict__ consts) {
  const hi2x_packed_segment sg = w.segments[blockIdx.y];
  if (sg.frags == 0) return;
  const int64_t e = blockIdx.y / PK_SEGS;
  const int64_t nblk = w.kp / sg.block;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const bool in = i < sg.frags * nblk * 16;
  const int64_t b = (i >> 4) % nblk, f = (i >> 4) / nblk;
  const int row = in ? w.rows[(sg.frag0 + f) * 16 + (i & 15)] : -1;
  uint32_t v = 0;
  float most = 0.0f;  // of |weight|: at the first or the last step of a ladder
  if (row >= 0 && b < w.k / sg.block) {
    const int64_t r = e * w.n + row;
    const uint8_t* p = params + 2 * (param_off[r] + b);
    const float lo = __builtin_fmaf((float)p[0], f16_from_bits(consts[3 * r + 1]),
                                    f16_from_bits(consts[3 * r]));
    const float st = (float)p[1] * f16_from_bits(consts[3 * r + 2]);
    v = (uint32_t)f16_bits(lo) | (uint32_t)f16_bits(st) << 16;
    const float l = f16_from_bits((uint16_t)v), steps = (float)((1 << sg.nbits) - 1);
    const float h = f16_from_bits(f16_bits(__builtin_fmaf(steps, f16_from_bits(v >> 16), l)));
    most = fmaxf(fabsf(l), fabsf(h));
    most = most < 65504.0f ? most : 65504.0f;  // (steps below an infinite one are finite)
  }
  if (in) reinterpret_cast<uint32_t*>(static_cast<char*>(w.params) + sg.params)[i] = v;
#pragma unroll
  for (int d = 32; d; d >>= 1) most = fmaxf(most, __shfl_xor(most, d));
  unsigned* to = reinterpret_cast<unsigned*>(w.largest);  // non-negative floats, by their bits
  if ((threadIdx.x & 63) == 0 &&
      __float_as_uint(most) > __hip_atomic_load(to, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT))
    atomicMax(to, __float_as_uint(most));
}

// ---- activations -------------------------------------------------------------------------
// Rows of SlotRows on their way through LDS: `a` and `b` hold them and their exponents slot by
// slot, then act(a) * b column by column takes their room.  Lanes take neighbouring columns, whose
// places are almost neighbours too, so that the reads by place meet on few banks; all of a row's
// loads are in flight before the first is waited for (131072 x 1024 hidden rows of 64 experts 386
// us without that).
template <int TPR>
struct SlotColumns {
  u32x4 raw[3];       // the row's slots, 8 at a time
  uint32_t exps;      // four fragments' exponents
  uint32_t place[8];  // of the columns' pairs
  __device__ __forceinline__ void load(const SlotRows& s, int64_t row, int tid) {
    const u32x4* from = reinterpret_cast<const u32x4*>(s.v + row * s.pitch);
#pragma unroll
    for (int i = 0; i < 3; ++i)
      raw[i] = tid + TPR * i < s.pitch / 8 ? from[tid + TPR * i] : u32x4{0u, 0u, 0u, 0u};
    exps = 4 * tid < s.ep ? reinterpret_cast<const uint32_t*>(s.exps + row * s.ep)[tid] : 0u;
  }
  __device__ __forceinline__ void load_places(const SlotRows& s, int expert, int tid) {
    const uint32_t* from = reinterpret_cast<const uint32_t*>(s.places + expert * s.n);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      place[i] = 2 * (tid + TPR * i) < s.n ? from[tid + TPR * i] : 0u;
  }
  __device__ __forceinline__ void put(const SlotRows& s, uint16_t* row, int8_t* ex,
                                      int tid) const {
#pragma unroll
    for (int i = 0; i < 3; ++i)
      if (tid + TPR * i < s.pitch / 8) reinterpret_cast<u32x4*>(row)[tid + TPR * i] = raw[i];
    if (4 * tid < s.ep) reinterpret_cast<uint32_t*>(ex)[tid] = exps;
  }
  __device__ __forceinline__ void take(const uint16_t* row, const int8_t* ex, float factor,
                                       float (&v)[16]) const {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const uint32_t p = i & 1 ? place[i >> 1] >> 16 : place[i >> 1] & 0xffffu;
      v[i] = ldexpf(f16_from_bits(row[p]), ex[p >> 4]) * factor;
    }
  }
};
// Bytes of a row's slots and exponents in LDS; the columns in the slots' room: 16-byte piece q
// of group g at q ^ (g / 4 % 4), so that the lanes' reads of whole groups fall on different banks.
__host__ __device__ inline int slot_bytes(const SlotRows& a, const SlotRows& b) {
  return (2 * (a.pitch + b.pitch) + a.ep + b.ep + 15) / 16 * 16;
}
__device__ __forceinline__ int group_piece(int g, int q) { return 4 * g + (q ^ (g >> 2 & 3)); }

// The 16 values of group g of a row, divided by their smoothing: of x, or (GLU) of
// act(x) * x2, or (SLOTS) of `sr` in LDS.
constexpr int SLOTS = 3;  // a type of its own
template <int DT, bool GLU>
__device__ __forceinline__ void group_values(const RawRows& x, const f32x4v* sr, int64_t base,
                                             int g, const uint16_t* cs, float (&v)[16]) {
  if constexpr (DT == SLOTS) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const f32x4v u = sr[group_piece(g, q)];
#pragma unroll
      for (int i = 0; i < 4; ++i) v[4 * q + i] = u[i];
    }
  } else {
    load16(x.x, base + 16 * (int64_t)g, DT, v);
  }
  if constexpr (GLU) {
    float u[16];
    load16(x.x2, base + 16 * (int64_t)g, 0, u);
    activate_all(v, x.act);
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] *= u[i];
  }
  if (cs) {
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = v[i] / f16_from_bits(cs[16 * g + i]);
  }
}

// TPR threads transform a row, several rows to a workgroup of 256 where that leaves room.  The
// largest finite |x / s| comes first; the rotation can grow it fourfold at most, so
// 2^(13 - exponent) brings every value to at most 2^15, with nothing of the row below fp16's
// normal range unless it is 2^-27 of the largest.  Then the values are scaled (exact), rotated
// by butterflies in f32 and rounded to fp16.  That rounding (at most 2^-11 of a value) is an
// eighth of a bf16 output's own and as large as an fp16 output's; nplanes 2 keeps the rest of it
// in a second plane.  A thread keeps its group's values between the two where one group a thread
// is all there is (KEEP, up to 16384 columns); rows beyond are read twice, the second time from
// L2.  Bound by reading x and writing the planes: 16384 x 2048 in bf16 27 us, 4.9 TB/s; the hidden
// rows of 16384 tokens and 8 of 64 experts (131072 x 1024, SlotRows) 255 us, where the way
// through LDS counts (196 us with the rows in their own order).
template <int DT, bool GLU, bool KEEP, int TPR>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void activations_kernel(
    RawRows x, int64_t k, const int64_t* __restrict__ src, const uint8_t* __restrict__ had,
    const uint16_t* __restrict__ cs, const int64_t* __restrict__ offs, int experts,
    hi2x_activations out) {
  constexpr int NT = TPR > 256 ? TPR : 256;
  const int64_t row = (int64_t)blockIdx.x * (NT / TPR) + threadIdx.x / TPR;
  const int tid = threadIdx.x % TPR;
  const bool none = row >= out.rows;
  const int64_t from = none ? -1 : (src ? src[row] : row);
  const bool bad = from < 0 || from >= x.rows;
  const int64_t base = bad ? 0 : from * x.ldx;
  SlotColumns<TPR> ca, cb;
  if constexpr (DT == SLOTS) {  // (the rows' loads before what their places wait for)
    ca.load(x.s1, none ? 0 : row, tid);
    cb.load(x.s2, none ? 0 : row, tid);
  }
  const int64_t* ranges = DT == SLOTS ? x.offs : offs;
  const int expert =
      ranges ? expert_of(range_ends(ranges, experts), ranges, experts, none ? 0 : row) : 0;
  if (offs) {
    had += (int64_t)expert * (k / 16);
    if (cs) cs += (int64_t)expert * k;
  }
  f32x4v* sr = nullptr;
  if constexpr (DT == SLOTS) {
    extern __shared__ __attribute__((aligned(16))) char rows16[];
    char* lds = rows16 + threadIdx.x / TPR * slot_bytes(x.s1, x.s2);
    uint16_t *a = reinterpret_cast<uint16_t*>(lds), *b = a + x.s1.pitch;
    int8_t *ea = reinterpret_cast<int8_t*>(b + x.s2.pitch), *eb = ea + x.s1.ep;
    const float fa = row_factor(x.s1, none ? 0 : row), fb = row_factor(x.s2, none ? 0 : row);
    sr = reinterpret_cast<f32x4v*>(lds);
    ca.load_places(x.s1, expert, tid);
    cb.load_places(x.s2, expert, tid);
    auto meet = [] {  // of the row's threads
      if constexpr (TPR > 64)
        __syncthreads();
      else
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup", "local");
    };
    ca.put(x.s1, a, ea, tid);
    cb.put(x.s2, b, eb, tid);
    meet();
    float v[16], u[16];
    ca.take(a, ea, fa, v);
    cb.take(b, eb, fb, u);
    meet();
    activate_all(v, x.act);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int p = tid + TPR * i;  // a pair of columns
      if (2 * p < x.s1.n)
        reinterpret_cast<float2*>(sr + group_piece(p >> 3, p >> 1 & 3))[p & 1] =
            make_float2(v[2 * i] * u[2 * i], v[2 * i + 1] * u[2 * i + 1]);
    }
    meet();
  }
  const int groups = (int)(k / 16), all = (int)(out.kp / 16);
  float v[16], m = 0.0f;
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = 0.0f;
  if (!bad) {
    for (int g = tid; g < groups; g += TPR) {
      group_values<DT, GLU>(x, sr, base, g, cs, v);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float a = fabsf(v[i]);
        m = fmaxf(m, a < __builtin_inff() ? a : 0.0f);
      }
    }
  }
#pragma unroll
  for (int d = 32; d; d >>= 1) m = fmaxf(m, __shfl_xor(m, d));
  if constexpr (TPR > 64) {
    __shared__ float red[NT / 64];
    const int w = threadIdx.x >> 6, w0 = w - (tid >> 6);  // the row's waves
    if ((tid & 63) == 0) red[w] = m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < TPR / 64; ++i) m = fmaxf(m, red[w0 + i]);
  }
  if (none) return;
  int ex = 0;
  if (m > 0.0f) (void)frexpf(m, &ex);
  // the exponent stays where both 2^e and 2^-e are normal
  const int e = 13 - ex > 126 ? 126 : (13 - ex < -126 ? -126 : 13 - ex);
  const float sc = ldexpf(1.0f, e);
  if (tid == 0) out.scale[row] = bad ? __builtin_nanf("") : ldexpf(1.0f, -e);
  uint16_t* dst = out.planes + row * out.kp * out.nplanes;
  for (int g = tid; g < all; g += TPR) {
    if (bad || g >= groups) {
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] = 0.0f;
    } else {
      if constexpr (!KEEP) group_values<DT, GLU>(x, sr, base, g, cs, v);
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] *= sc;
      if (had[g]) {
#pragma unroll
        for (int d = 1; d < 16; d <<= 1)
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (!(i & d)) {
              const float a = v[i], b = v[i | d];
              v[i] = a + b;
              v[i | d] = a - b;
            }
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] *= 0.25f;
      }
    }
    uint32_t h[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
      h[i] = (uint32_t)f16_bits(v[2 * i]) | (uint32_t)f16_bits(v[2 * i + 1]) << 16;
    uint16_t* at = dst + (int64_t)(g >> 3) * (PK_CHUNK * out.nplanes) + 16 * (g & 7);
    u32x4* d = reinterpret_cast<u32x4*>(at);
    d[0] = u32x4{h[0], h[1], h[2], h[3]};
    d[1] = u32x4{h[4], h[5], h[6], h[7]};
    if (out.nplanes == 2) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        h[i] = rest_bits(v[2 * i], h[i]) | rest_bits(v[2 * i + 1], h[i] >> 16) << 16;
      d = reinterpret_cast<u32x4*>(at + PK_CHUNK);
      d[0] = u32x4{h[0], h[1], h[2], h[3]};
      d[1] = u32x4{h[4], h[5], h[6], h[7]};
    }
  }
}

}  // namespace

int launch_activations(const RawRows& x, const hi2x_packed& w, const int64_t* src,
                       const int64_t* offs, const hi2x_activations& out, hipStream_t s) {
  if (out.rows == 0) return HI2X_OK;
#define HI2X_ROWS_(DT, GLU, KEEP, TPR)                                                    \
  activations_kernel<DT, GLU, KEEP, TPR>                                                  \
      <<<dim3((unsigned)(TPR < 256 ? (out.rows * TPR + 255) / 256 : out.rows)),           \
         TPR < 256 ? 256 : TPR,                                                           \
         DT == SLOTS ? (TPR < 256 ? 256 / TPR : 1) * slot_bytes(x.s1, x.s2) : 0,          \
         s>>>(x, w.k, src, w.had, w.col_scale, offs, (int)w.experts, out)
#define HI2X_ROWS(DT, GLU)                 \
  if (w.kp <= 1024)                        \
    HI2X_ROWS_(DT, GLU, true, 64);         \
  else if (w.kp <= 2048)                   \
    HI2X_ROWS_(DT, GLU, true, 128);        \
  else if (w.kp <= 4096)                   \
    HI2X_ROWS_(DT, GLU, true, 256);        \
  else if (w.kp <= 8192)                   \
    HI2X_ROWS_(DT, GLU, true, 512);        \
  else if constexpr (DT != SLOTS) {        \
    if (w.kp <= 16384)                     \
      HI2X_ROWS_(DT, GLU, true, 1024);     \
    else                                   \
      HI2X_ROWS_(DT, GLU, false, 1024);    \
  }
  if (x.s1.v) {
    HI2X_ROWS(SLOTS, false)
  } else if (x.x2) {
    HI2X_ROWS(0, true)
  } else if (x.dtype == 0) {
    HI2X_ROWS(0, false)
  } else if (x.dtype == 1) {
    HI2X_ROWS(1, false)
  } else {
    HI2X_ROWS(2, false)
  }
#undef HI2X_ROWS
#undef HI2X_ROWS_
  return launch_status("packed_activations");
}

}  // namespace hi2x

using namespace hi2x;

extern "C" int hi2x_packed_layout(const hi2x_packed* w, const int32_t* codes,
                                  const int64_t* code_off, const uint8_t* blk_params,
                                  const int64_t* param_off, const uint16_t* row_consts,
                                  void* stream) {
  clear_error();
  if (int rc = check_packed(w, "packed_layout")) return rc;
  HI2X_REQUIRE(w->largest, "packed_layout: null buffer");
  HI2X_REQUIRE(codes && code_off && blk_params && param_off && row_consts,
               "packed_layout: null buffer");
  const hipStream_t s = as_stream(stream);
  const int64_t segs = w->experts * PK_SEGS;
  // the largest segment has at most max_frags fragments; smaller ones leave workgroups idle
  const int64_t nc = (w->max_frags * (w->kp / PK_CHUNK) * 64 + 255) / 256;
  const int64_t np = (w->max_frags * (w->kp / 16) * 16 + 255) / 256;
  HI2X_REQUIRE(segs <= 65535 && nc < (1ll << 31) && np < (1ll << 31),
               "packed_layout: tensor too large");
  layout_codes_kernel<<<dim3((unsigned)nc, (unsigned)segs), 256, 0, s>>>(*w, codes, code_off);
  layout_params_kernel<<<dim3((unsigned)np, (unsigned)segs), 256, 0, s>>>(*w, blk_params,
                                                                          param_off, row_consts);
  return launch_status("packed_layout");
}

extern "C" int hi2x_packed_activations(const hi2x_packed* w, const void* x, int dtype,
                                       int64_t ldx, int64_t x_rows, const int64_t* src,
                                       const int64_t* offs, const hi2x_activations* out,
                                       void* stream) {
  clear_error();
  HI2X_REQUIRE(out, "packed_activations: null output");
  if (int rc = check_packed(w, "packed_activations")) return rc;
  if (int rc = check_x(x, dtype, ldx, x_rows, w->k, "packed_activations")) return rc;
  HI2X_REQUIRE(out->kp == w->kp, "packed_activations: %lld padded columns, %lld needed",
               (long long)out->kp, (long long)w->kp);
  HI2X_REQUIRE(out->nplanes == 1 || out->nplanes == 2, "packed_activations: %d planes",
               out->nplanes);
  HI2X_REQUIRE(out->rows >= 0 && out->rows < (1ll << 31), "packed_activations: bad shape");
  HI2X_REQUIRE(offs || !w->per_expert, "packed_activations: %lld transforms without ranges",
               (long long)w->experts);
  if (out->rows == 0) return HI2X_OK;
  HI2X_REQUIRE(out->planes && out->scale, "packed_activations: null buffer");
  HI2X_REQUIRE(src || out->rows <= x_rows, "packed_activations: %lld rows of %lld",
               (long long)out->rows, (long long)x_rows);
  HI2X_REQUIRE(((uintptr_t)out->planes & 255) == 0, "packed_activations: planes not aligned");
  return launch_activations(RawRows{x, dtype, ldx, x_rows, out->nplanes}, *w, src,
                            w->per_expert ? offs : nullptr, *out, as_stream(stream));
}
