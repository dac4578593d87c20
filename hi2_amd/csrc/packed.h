// Device-side view of a packed tensor (or the experts of one projection) laid out for
// products, and the epilogue its products share (packed.hip, packed_gemm.hip).
#pragma once
#include "common.h"

namespace hi2x {

typedef _Float16 h16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 h16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4v __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// The columns are walked in chunks of 128.  MFMA step s (0..3) of a chunk multiplies the
// 32 columns 128 c + 32 q + 8 s + j (q = lane / 16, j < 8): the sum does not depend on the
// order of its terms, and with this one a lane's 32 codes of a chunk are neighbours in
// their row, so they lie in one ladder block (two, at 16 columns a block) and come with
// one load.
constexpr int PK_CHUNK = 128;
constexpr int PK_SEGS = HI2X_PACKED_SEGMENTS;

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

// The steps s of a chunk's weights from a lane's codes, as the MFMA's A operand: fp16
// (lo + code step) with one rounding, which is the format's own decode.  A dword holds its
// codes as pairs (bits f and 16 + f), so masking one pair leaves two codes in the
// mantissas of two halves; with the exponent of 1024 or-ed in, each half is exactly
// 1024 + code 2^f, and one exact packed fma (or add) takes that to the code itself.
template <int BITS>
__device__ __forceinline__ h16x8 decode_step(const uint32_t (&cw)[BITS], int s, h16x2 lo,
                                             h16x2 st) {
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
    const uint32_t x = (w & ((M << f) | (M << (16 + f)))) | 0x64006400u;
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

// A fragment of 16 slots (rows in layout order): where a lane's codes and ladder
// parameters are.
struct PkFrag {
  const uint8_t* codes;    // chunk c at + c * 256 * BITS
  const uint32_t* params;  // block b of the lane's row at [16 * b]
};

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

}  // namespace hi2x
