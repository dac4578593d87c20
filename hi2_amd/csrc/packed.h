// Device-side view of a packed tensor (or the experts of one projection) laid out for
// products, and the epilogue its products share (packed.hip, packed_gemm.hip).
#pragma once
#include "common.h"

namespace hi2x {

typedef _Float16 h16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 h16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4v __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

// The columns are walked in chunks of 128.  MFMA step s (0..3) of a chunk multiplies the
// 32 columns 128 c + 32 q + 8 s + j (q = lane / 16, j < 8): the sum does not depend on the
// order of its terms, and with this one a lane's 32 codes of a chunk are neighbours in
// their row, so they lie in one ladder block (two, at 16 columns a block) and come with
// one load.
constexpr int PK_CHUNK = 128;
constexpr int PK_SEGS = HI2X_PACKED_SEGMENTS;

// Lane exchanges within rows of 16 lanes.
template <int CTRL>
__device__ __forceinline__ int dpp(int x) {
  return __builtin_amdgcn_update_dpp(x, x, CTRL, 0xf, 0xf, false);
}
// Reductions over each row of 16 lanes: neighbours, pairs, halves mirrored, row mirrored.
#define HI2X_ROW16(x, OP)   \
  x = OP(x, dpp<0xB1>(x));  \
  x = OP(x, dpp<0x4E>(x));  \
  x = OP(x, dpp<0x141>(x)); \
  x = OP(x, dpp<0x140>(x));

__device__ __forceinline__ int umax_(int a, int b) {
  return (int)((uint32_t)a > (uint32_t)b ? (uint32_t)a : (uint32_t)b);
}
__device__ __forceinline__ int umin_(int a, int b) {
  return (int)((uint32_t)a < (uint32_t)b ? (uint32_t)a : (uint32_t)b);
}
__device__ __forceinline__ int or_(int a, int b) { return a | b; }
__device__ __forceinline__ int imax_(int a, int b) { return a > b ? a : b; }
__device__ __forceinline__ uint32_t row_umax(uint32_t v) {
  int x = (int)v;
  HI2X_ROW16(x, umax_)
  return (uint32_t)x;
}
__device__ __forceinline__ uint32_t row_umin(uint32_t v) {
  int x = (int)v;
  HI2X_ROW16(x, umin_)
  return (uint32_t)x;
}
__device__ __forceinline__ uint32_t row_or(uint32_t v) {
  int x = (int)v;
  HI2X_ROW16(x, or_)
  return (uint32_t)x;
}
// Loads of a row operand (bias, factor, residual) by its type.
__device__ __forceinline__ float load_as_f32(const void* p, int64_t i, int dtype) {
  if (dtype == 0) return static_cast<const float*>(p)[i];
  const uint16_t b = static_cast<const uint16_t*>(p)[i];
  if (dtype == 1) return f16_from_bits(b);
  return __uint_as_float((uint32_t)b << 16);
}

// bf16 round to nearest even; NaN stays NaN.
__device__ __forceinline__ uint16_t bf16_bits(float x) {
  return __builtin_bit_cast(uint16_t, (__bf16)x);
}

__device__ __forceinline__ void store_from_f32(void* p, int64_t i, int dtype, float v) {
  if (dtype == 0)
    static_cast<float*>(p)[i] = v;
  else if (dtype == 1)
    static_cast<uint16_t*>(p)[i] = f16_bits(v);
  else
    static_cast<uint16_t*>(p)[i] = bf16_bits(v);
}

__device__ __forceinline__ float activate(float y, int act) {
  switch (act) {
    case HI2X_ACT_RELU:
      return y < 0.0f ? 0.0f : y;  // NaN stays
    case HI2X_ACT_SILU:
      return y / (1.0f + expf(-y));
    case HI2X_ACT_GELU:
      return 0.5f * y * (1.0f + erff(y * 0.70710678118654752f));
    case HI2X_ACT_GELU_TANH:
      return 0.5f * y * (1.0f + tanhf(0.79788456080286536f * (y + 0.044715f * y * y * y)));
    default:
      return y;
  }
}

// The same of several values, the choice made once.
template <int N>
__device__ __forceinline__ void activate_all(float (&y)[N], int act) {
#define HI2X_EACH(A)                                   \
  _Pragma("unroll") for (int i = 0; i < N; ++i) y[i] = activate(y[i], A);
  switch (act) {
    case HI2X_ACT_RELU:
      HI2X_EACH(HI2X_ACT_RELU)
      break;
    case HI2X_ACT_SILU:
      HI2X_EACH(HI2X_ACT_SILU)
      break;
    case HI2X_ACT_GELU:
      HI2X_EACH(HI2X_ACT_GELU)
      break;
    case HI2X_ACT_GELU_TANH:
      HI2X_EACH(HI2X_ACT_GELU_TANH)
      break;
    default:
      break;
  }
#undef HI2X_EACH
}

// The steps s of a chunk's weights from a lane's codes, as the MFMA's A operand: fp16
// (lo + code step) with one rounding, which is the format's own decode.  A dword holds its
// codes as pairs (bits f and 16 + f), so masking one pair leaves two codes in the
// mantissas of two halves; with the exponent of 1024 or-ed in, each half is exactly
// 1024 + code 2^f, and one exact packed fma (or add) takes that to the code itself.
// `magic` is DECODE_MAGIC in a vector register (decode_magic), which lets mask and or be one
// instruction.
constexpr uint32_t DECODE_MAGIC = 0x64006400u;
__device__ __forceinline__ uint32_t decode_magic() {
  uint32_t m = DECODE_MAGIC;
  asm("" : "+v"(m));
  return m;
}
template <int BITS>
__device__ __forceinline__ h16x8 decode_step(const uint32_t (&cw)[BITS], int s, h16x2 lo,
                                             h16x2 st, uint32_t magic) {
  h16x8 out;
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    uint32_t w;
    int f;  // bit of the pair's low code
    if constexpr (BITS == 4) {
      w = p < 2 ? cw[s] : cw[s] >> 8;
      f = 4 * (p & 1);
    } else if constexpr (BITS == 2) {
      w = (s & 1) ? cw[s >> 1] >> 8 : cw[s >> 1];
      f = 2 * p;
    } else {
      w = (p & 1) ? cw[2 * s + (p >> 1)] >> 8 : cw[2 * s + (p >> 1)];
      f = 0;
    }
    constexpr uint32_t M = (1u << BITS) - 1u;
    const uint32_t x = (w & ((M << f) | (M << (16 + f)))) | magic;
    const h16x2 v = __builtin_bit_cast(h16x2, x);
    h16x2 c;
    if (f == 0) {
      c = v - (h16x2){(_Float16)1024.0f, (_Float16)1024.0f};
    } else {
      const _Float16 sc = (_Float16)(1.0f / (float)(1 << f));
      const _Float16 of = (_Float16)(-1024.0f / (float)(1 << f));
      c = __builtin_elementwise_fma(v, (h16x2){sc, sc}, (h16x2){of, of});
    }
    const h16x2 y = __builtin_elementwise_fma(c, st, lo);
    out[2 * p] = y[0];
    out[2 * p + 1] = y[1];
  }
  return out;
}

// The expert and token tile a workgroup row works on: tile `want` in the order of the
// experts' ceil(n_e / tile) tiles.  Every wave computes it for itself; e < 0 past the end.
struct PkWork {
  int e;
  int64_t first, end;  // slots
};

__device__ __forceinline__ PkWork find_work(const int64_t* offs, int experts, int64_t slots,
                                            int tile, int64_t want) {
  PkWork w{-1, 0, 0};
  if (!offs) {
    w.e = want * tile < slots ? 0 : -1;
    w.first = want * tile;
    w.end = slots;
    return w;
  }
  const int lane = threadIdx.x & 63;
  int64_t before = 0;
  for (int e0 = 0; e0 < experts; e0 += 64) {
    const int e = e0 + lane;
    int64_t a = 0, b = 0;
    if (e < experts) {
      a = offs[e];
      b = offs[e + 1];
      a = a < 0 ? 0 : (a > slots ? slots : a);
      b = b < a ? a : (b > slots ? slots : b);
    }
    const int n = (int)((b - a + tile - 1) / tile);
    int inc = n;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int o = __shfl_up(inc, d);
      if (lane >= d) inc += o;
    }
    const int64_t upto = before + inc;
    const unsigned long long hit = __ballot(want < upto && want >= upto - n);
    if (hit) {
      const int l = __builtin_ctzll(hit);
      const int64_t base = before + __shfl(inc, l) - __shfl(n, l);
      w.e = e0 + l;
      w.first = __shfl(a, l) + (want - base) * tile;
      w.end = __shfl(b, l);
      return w;
    }
    before += __shfl(inc, 63);
  }
  return w;
}

// `exps`: the result is handed on in fp16 without its row's factor, each row in the order of its
// expert's slots and each fragment of 16 slots under a power of two of its own, 2^c with c in
// exps[slot][fragment], for a kernel that reads it with a SlotRows.  (Scattered to the rows' own
// order, a lane would store single values: the stores alone took a quarter of the products of 64
// experts of 2048 x 1024 at 16384 tokens, gate and up 1316 us and 1152 so, down 847 and 623.)
struct GemmArgs {
  hi2x_packed w;
  hi2x_activations x;
  const int64_t* src;
  const int64_t* offs;
  int64_t slots;
  hi2x_epilogue epi;
  int8_t* exps = nullptr;
  int ep = 0;  // bytes of a row of exps: the most fragments of an expert, a multiple of 4
};

// The largest finite value of a fragment comes to [2^14, 2^15): its others keep fp16's 11 bits
// down to 2^-28 of it, and what is lost below is 2^-39 of it, whatever the sizes of the experts,
// the rows and their channels.  (Under one bound for all experts' sums a row far below it lost
// its bits.)  EXP_LEAST keeps 2^c and 2^-c normal floats.
constexpr int EXP_LEAST = -120;
inline int exps_pitch(const hi2x_packed& w) { return (int)((w.max_frags + 3) / 4 * 4); }

// Rows of such a product of w [n][.]: `pitch` values each, of which `places` says where a column
// lies; its fragment's exponent and the factor of the row's activations take it back.
struct SlotRows {
  const uint16_t* v = nullptr;
  int pitch = 0;
  const uint16_t* places = nullptr;
  const int8_t* exps = nullptr;
  int ep = 0;
  const float* scale = nullptr;
  const int64_t* index = nullptr;  // row of scale, or null: the row itself
  int64_t rows = 0;                // of scale
  int64_t n = 0;
};
__device__ __forceinline__ float row_factor(const SlotRows& f, int64_t row) {
  const int64_t r = f.index ? f.index[row] : row;
  return r >= 0 && r < f.rows ? f.scale[r] : __builtin_nanf("");
}
// The expert whose range holds a slot (the same for the wave): as many as end at or before it
// come before it; the last one where the ranges end too early.  `ends` are the lanes' own of
// the first 64 experts (range_ends).
__device__ __forceinline__ int64_t range_ends(const int64_t* offs, int experts) {
  const int lane = threadIdx.x & 63;
  return lane < experts ? offs[lane + 1] : INT64_MAX;
}
__device__ __forceinline__ int expert_of(int64_t ends, const int64_t* offs, int experts,
                                         int64_t slot) {
  int e = __builtin_popcountll(__ballot(ends <= slot));
  for (int e0 = 64; e0 < experts; e0 += 64) {
    const int i = e0 + (threadIdx.x & 63);
    e += __builtin_popcountll(__ballot(i < experts && offs[i + 1] <= slot));
  }
  return e < experts ? e : experts - 1;
}
constexpr int SLOTS16 = 8192;  // most slots of a row of SlotRows (two of them lie in LDS)

// Loads go through buffer resources: a lane's offset is one 32-bit register, the walk along
// the columns is a scalar offset, and what lies past the resource reads as zero.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rsrc(const void* base, int64_t bytes) {
  const int64_t most = 0xffffffffll;
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), (short)0,
                                           (int)(uint32_t)(bytes < most ? bytes : most),
                                           0x00020000);
}

// A tile of up to `per` fragments of one segment: number t of expert e's, segment by segment.
// One expert's table comes with the arguments; of several, each lane reads one segment, so
// that finding the tile costs one load's latency.
struct Tile {
  int64_t codes, params;
  int nbits, block;
  int frag;   // first fragment, over all experts
  int first;  // and in its segment
  int base;   // first fragment of its expert
  int count;
};

__device__ __forceinline__ bool find_tile(const hi2x_packed& w, int e, int t, int per,
                                          Tile& out) {
  if (w.experts == 1) {
#pragma unroll
    for (int i = 0; i < PK_SEGS; ++i) {
      const hi2x_packed_segment& sg = w.first[i];
      const int n = (sg.frags + per - 1) / per;
      if (t >= 0 && t < n) {
        out.codes = sg.codes;
        out.params = sg.params;
        out.nbits = sg.nbits;
        out.block = sg.block;
        out.first = t * per;
        out.frag = sg.frag0 + out.first;
        out.base = 0;
        out.count = sg.frags - out.first < per ? sg.frags - out.first : per;
        return true;
      }
      t -= n;
    }
    return false;
  }
  const int lane = threadIdx.x & 63;
  hi2x_packed_segment sg{};
  if (lane < PK_SEGS) sg = w.segments[e * PK_SEGS + lane];
  const int n = (sg.frags + per - 1) / per;
  int upto = n;
#pragma unroll
  for (int d = 1; d < 16; d <<= 1) {
    const int o = __shfl_up(upto, d);
    if (lane >= d) upto += o;
  }
  const unsigned long long hit = __ballot(lane < PK_SEGS && t < upto && t >= upto - n);
  if (!hit) return false;
  const int l = __builtin_ctzll(hit);
  auto at = [&](int v) { return __builtin_amdgcn_readlane(v, l); };
  auto at64 = [&](int64_t v) {
    return (int64_t)(uint32_t)at((int)v) | (int64_t)at((int)(v >> 32)) << 32;
  };
  out.codes = at64(sg.codes);
  out.params = at64(sg.params);
  out.nbits = at(sg.nbits);
  out.block = at(sg.block);
  out.first = (t - at(upto - n)) * per;
  out.frag = at(sg.frag0) + out.first;
  out.base = __builtin_amdgcn_readlane(sg.frag0, __builtin_ctzll(__ballot(sg.frags > 0)));
  const int left = at(sg.frags) - out.first;
  out.count = left < per ? left : per;
  return true;
}

template <int BITS>
__device__ __forceinline__ void load_codes(__amdgpu_buffer_rsrc_t rs, int lane, uint32_t soff,
                                           uint32_t (&cw)[BITS]) {
  if constexpr (BITS == 2) {
    const auto v = __builtin_amdgcn_raw_buffer_load_b64(rs, 8 * lane, (int)soff, 0);
    cw[0] = v[0];
    cw[1] = v[1];
  } else {
#pragma unroll
    for (int h = 0; h < BITS / 4; ++h) {
      const auto v =
          __builtin_amdgcn_raw_buffer_load_b128(rs, 16 * lane + 1024 * h, (int)soff, 0);
#pragma unroll
      for (int i = 0; i < 4; ++i) cw[4 * h + i] = v[i];
    }
  }
}

// What fp16 `h` leaves of v, as fp16: the second plane's value.  Infinities are whole in the
// first (their difference, a NaN, would take the product's sign).
__device__ __forceinline__ uint32_t rest_bits(float v, uint32_t h) {
  const float r = v - f16_from_bits((uint16_t)h);
  return f16_bits(r == r ? r : 0.0f);
}

// 16 neighbouring activations, 16-byte aligned.
__device__ __forceinline__ void load16(const void* x, int64_t at, int dtype, float (&v)[16]) {
  if (dtype == 0) {
    const f32x4v* p = reinterpret_cast<const f32x4v*>(static_cast<const float*>(x) + at);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const f32x4v u = p[i];
#pragma unroll
      for (int j = 0; j < 4; ++j) v[4 * i + j] = u[j];
    }
    return;
  }
  const u32x4* p = reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(x) + at);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const u32x4 u = p[i];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[8 * i + 2 * j] =
          dtype == 1 ? f16_from_bits((uint16_t)u[j]) : __uint_as_float(u[j] << 16);
      v[8 * i + 2 * j + 1] =
          dtype == 1 ? f16_from_bits((uint16_t)(u[j] >> 16)) : __uint_as_float(u[j] & 0xffff0000u);
    }
  }
}

// Whether a product goes to packed_few: its rows fit one operand (4096 x 14336 at 16 rows
// takes 20 us so, 23 in 64 x 64 tiles with the columns in eight shares; 28672 x 8192 30 and
// 43).  Experts' rows take tiles: a layer of 64 experts at 64 tokens, eight each, took 315 us
// so and 128 us in tiles.
inline bool few_rows_product(int64_t slots, bool ranges) {
  return !ranges && slots <= 16;
}

constexpr int64_t FEW_RAW = 8;      // rows the few-rows kernel transforms for itself,
constexpr int64_t FEW_RANGES = 16;  // and of all experts together

// Activations as they are: rows ldx elements apart; with x2 (same type and pitch, 32 bits)
// act(x) * x2 elementwise; where s1 holds rows (s1.v) act(s1) * s2 instead, of the experts of
// `offs`.  x may be null where there are no rows.
struct RawRows {
  const void* x;
  int dtype;
  int64_t ldx, rows;
  int npl;  // planes of their transform
  const float* x2 = nullptr;
  int act = 0;
  SlotRows s1, s2;
  const int64_t* offs = nullptr;
};

// Products of `count` (1, or with ranges 2) tensors of one shape from the same activations; the
// epilogue's arguments as for hi2x_packed_linear.  Ranges take no shares of the columns and need
// no workspace.
struct GemmPair {
  GemmArgs g[2];
};
int packed_few(const GemmArgs& g, hipStream_t s);
int packed_few_raw(const GemmPair& g, int count, const RawRows& x, hipStream_t s);
int packed_product(const GemmPair& g, int count, void* work, int64_t work_bytes, hipStream_t s);
int64_t packed_part_bytes(const hi2x_packed& w, int64_t slots, bool ranges, int npl);
int launch_activations(const RawRows& x, const hi2x_packed& w, const int64_t* src,
                       const int64_t* offs, const hi2x_activations& out, hipStream_t s);
int launch_combine(const void* y, int dt_y, int64_t y_rows, int64_t n, const int64_t* slots,
                   const float* weights, int64_t t, int64_t top_k, const void* residual,
                   int dt_residual, void* out, int dt_out, hipStream_t s);
int launch_combine(const SlotRows& y, const int64_t* offs, int experts, int64_t y_rows,
                   const int64_t* slots, const float* weights, int64_t t, int64_t top_k,
                   const void* residual, int dt_residual, void* out, int dt_out, hipStream_t s);

// Whether a product takes its activations as they are and transforms them inside.  Of
// experts most have one row then: at 64 experts and 8 choices, two tokens 62 us so and 74 in
// tiles, four 84 and 75.
inline bool few_raw_product(int64_t slots, bool ranges) {
  return slots <= (ranges ? FEW_RANGES : FEW_RAW);
}

inline int64_t plane_bytes(const hi2x_packed& w, int64_t rows, int npl) {
  return rows * w.kp * 2 * npl;  // a multiple of 256
}
// Rows of the transform in front of a product: those of x, or every slot's by its own expert's
// transform.  Of no rows at all (each index lies outside) it makes every slot a row of NaN.
inline bool transform_slots(const hi2x_packed& w, int64_t x_rows) {
  return w.per_expert || x_rows == 0;
}
inline int64_t transform_rows(const hi2x_packed& w, int64_t x_rows, bool indexed, int64_t slots) {
  return !indexed || transform_slots(w, x_rows) ? slots : x_rows;
}
inline int64_t align256(int64_t n) { return (n + 255) / 256 * 256; }

inline int check_packed(const hi2x_packed* w, const char* what) {
  HI2X_REQUIRE(w, "%s: null tensor", what);
  HI2X_REQUIRE(w->experts >= 1 && w->n >= 1 && w->k >= 16 && w->k % 16 == 0,
               "%s: bad shape (%lld experts of %lld x %lld; columns a multiple of 16)", what,
               (long long)w->experts, (long long)w->n, (long long)w->k);
  HI2X_REQUIRE(w->kp % PK_CHUNK == 0 && w->kp >= w->k && w->kp < w->k + PK_CHUNK,
               "%s: %lld padded columns for %lld", what, (long long)w->kp, (long long)w->k);
  // a tile's 16 fragments stay below 4 GiB of codes (32-bit offsets)
  HI2X_REQUIRE(w->n < (1ll << 31) && w->k < (1ll << 20) && w->frags < (1ll << 27) &&
                   w->experts <= 7000,
               "%s: tensor too large", what);
  HI2X_REQUIRE(w->codes && w->params && w->rows && w->segments, "%s: null buffer", what);
  HI2X_REQUIRE((((uintptr_t)w->codes | (uintptr_t)w->params) & 255) == 0,
               "%s: layout not 256-byte aligned", what);
  return HI2X_OK;
}

inline int check_x(const void* x, int dtype, int64_t ldx, int64_t x_rows, int64_t k,
                   const char* what) {
  HI2X_REQUIRE(dtype >= 0 && dtype <= 2, "%s: dtype %d", what, dtype);
  HI2X_REQUIRE(x_rows >= 0 && ldx >= k, "%s: bad shape", what);
  HI2X_REQUIRE(x || x_rows == 0, "%s: null activations", what);
  HI2X_REQUIRE(((uintptr_t)x & 15) == 0 && ldx % (dtype == 0 ? 4 : 8) == 0,
               "%s: activations not aligned to 16 bytes", what);
  return HI2X_OK;
}

inline int check_product(const hi2x_packed* w, const int64_t* src, const int64_t* offs,
                         int64_t slots, int64_t x_rows, const hi2x_epilogue* epi,
                         const char* what) {
  HI2X_REQUIRE(offs || w->experts == 1, "%s: %lld experts without ranges", what,
               (long long)w->experts);
  HI2X_REQUIRE(slots >= 0 && slots < (1ll << 31) && x_rows >= 0, "%s: bad rows", what);
  HI2X_REQUIRE(src || slots <= x_rows, "%s: %lld rows of %lld", what, (long long)slots,
               (long long)x_rows);
  HI2X_REQUIRE(epi->act >= HI2X_ACT_NONE && epi->act <= HI2X_ACT_GELU_TANH, "%s: activation %d",
               what, epi->act);
  for (int32_t d : {epi->dt_bias, epi->dt_mul, epi->dt_residual, epi->dt_out})
    HI2X_REQUIRE(d >= 0 && d <= 2, "%s: dtype %d", what, d);
  HI2X_REQUIRE(slots == 0 || epi->out, "%s: null output", what);
  HI2X_REQUIRE(epi->ld_out >= w->n && (!epi->mul || epi->ld_mul >= w->n) &&
                   (!epi->residual || epi->ld_residual >= w->n),
               "%s: rows overlap", what);
  return HI2X_OK;
}

}  // namespace hi2x
