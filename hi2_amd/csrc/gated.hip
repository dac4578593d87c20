// The gated activation between the products of an MLP, out = act(gate) * up, and its gradients
//   d_gate = grad * up * act'(gate),  d_up = grad * act(gate),
// in float32 from one pass over the operands, each result rounded once.  HBM bounds both (3 and 5
// elements moved for one of the result): 131072 x 1024 in bfloat16 178 us (4.5 TB/s) and 251 (5.3),
// where a large copy has 4.9.
#include <type_traits>

#include "packed.h"

namespace hi2x {
namespace {

// 16 bytes of a row: 4 float32 values or 8 of 16 bits.
template <int DT>
constexpr int WIDE = DT == 0 ? 4 : 8;

// STREAM: past the caches, where a call touches twice what the last one holds (256 MB) and nothing of
// it would be there for the next.  131072 x 1024 in bfloat16 with gradients 399 us, so 383; 2000 x
// 14336, 92, would take 97.
constexpr int64_t STREAM_BYTES = 512ll << 20;

template <int DT, int V, bool STREAM>
__device__ __forceinline__ void load_values(const void* p, int64_t at, float (&x)[V]) {
  if constexpr (V == 1) {
    x[0] = load_as_f32(p, at, DT);
  } else if constexpr (DT == 0) {
    const f32x4v* q = reinterpret_cast<const f32x4v*>(static_cast<const float*>(p) + at);
    const f32x4v f = STREAM ? __builtin_nontemporal_load(q) : *q;
    x[0] = f.x, x[1] = f.y, x[2] = f.z, x[3] = f.w;
  } else {
    const u32x4* q = reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(p) + at);
    const u32x4 w = STREAM ? __builtin_nontemporal_load(q) : *q;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const uint16_t b = (uint16_t)(w[j / 2] >> (16 * (j & 1)));
      x[j] = DT == 1 ? f16_from_bits(b) : __uint_as_float((uint32_t)b << 16);
    }
  }
}

template <int DT, int V, bool STREAM>
__device__ __forceinline__ void store_values(void* p, int64_t at, const float (&x)[V]) {
  if constexpr (V == 1) {
    store_from_f32(p, at, DT, x[0]);
  } else if constexpr (DT == 0) {
    f32x4v* q = reinterpret_cast<f32x4v*>(static_cast<float*>(p) + at);
    const f32x4v f = {x[0], x[1], x[2], x[3]};
    if constexpr (STREAM)
      __builtin_nontemporal_store(f, q);
    else
      *q = f;
  } else {
    u32x4 w;
#pragma unroll
    for (int j = 0; j < V / 2; ++j) {
      const uint32_t a = DT == 1 ? f16_bits(x[2 * j]) : bf16_bits(x[2 * j]);
      const uint32_t b = DT == 1 ? f16_bits(x[2 * j + 1]) : bf16_bits(x[2 * j + 1]);
      w[j] = a | b << 16;
    }
    u32x4* q = reinterpret_cast<u32x4*>(static_cast<uint16_t*>(p) + at);
    if constexpr (STREAM)
      __builtin_nontemporal_store(w, q);
    else
      *q = w;
  }
}

// The activation and its derivative.  Both tails keep their relative precision: sigmoids come
// from exp(-|x|), so that p and 1 - p are products and no difference, and the normal
// distribution from erfc.
template <int ACT>
__device__ __forceinline__ void act_both(float x, float& h, float& slope) {
  if constexpr (ACT == HI2X_ACT_RELU) {
    h = x < 0.0f ? 0.0f : x;  // NaN stays
    slope = x <= 0.0f ? 0.0f : 1.0f;
  } else if constexpr (ACT == HI2X_ACT_SILU) {
    const float e = expf(-fabsf(x)), r = 1.0f / (1.0f + e), er = e * r;
    const float p = x >= 0.0f ? r : er, q = x >= 0.0f ? er : r;
    h = x * p;
    slope = p + h * q;
  } else if constexpr (ACT == HI2X_ACT_GELU) {
    const float p = 0.5f * erfcf(x * -0.70710678118654752f);
    h = x * p;
    slope = p + x * (expf(-0.5f * x * x) * 0.3989422804014327f);
  } else if constexpr (ACT == HI2X_ACT_GELU_TANH) {
    // p = sigmoid(2 u) with u = sqrt(2 / pi) (x + 0.044715 x^3); p' = 2 p (1 - p) u'
    const float u2 = 1.5957691216057308f * (x + 0.044715f * (x * x * x));
    const float e = expf(-fabsf(u2)), r = 1.0f / (1.0f + e), er = e * r;
    const float p = u2 >= 0.0f ? r : er;
    h = x * p;
    const float steep = er > 0.0f ? x * (r * er) * (1.5957691216057308f + 0.2140644488f * (x * x))
                                  : 0.0f * er;
    slope = p + steep;
  } else {
    h = x;
    slope = 1.0f;
  }
}

struct Args {
  const void *grad, *gate, *up;
  void *out, *d_gate, *d_up;
  int64_t ld_grad, ld_gate, ld_up, ld_out, ld_dgate, ld_dup;
  int64_t rows, n;
  uint32_t pieces;  // column pieces of tx vectors a row
  int shift;        // tx = 1 << shift threads along a row, 256 >> shift rows a workgroup
};

// A workgroup takes 256 >> shift rows x (1 << shift) vectors of V neighbours; a row's last
// vector may be partial.
template <int DT, int ACT, int V, bool BACK, bool STREAM>
__global__ __launch_bounds__(256) void gated_kernel(Args a) {
  const uint32_t piece = blockIdx.x % a.pieces, band = blockIdx.x / a.pieces;
  const int tx = threadIdx.x & ((1 << a.shift) - 1), ty = threadIdx.x >> a.shift;
  const int64_t row = (int64_t)band * (256 >> a.shift) + ty;
  const int64_t c = (((int64_t)piece << a.shift) + tx) * V;
  if (row >= a.rows || c >= a.n) return;
  auto some = [&](auto width, int64_t c) {
    constexpr int W = decltype(width)::value;
    float g[W], u[W], d[W], y[W];
    load_values<DT, W, STREAM>(a.gate, row * a.ld_gate + c, g);
    load_values<DT, W, STREAM>(a.up, row * a.ld_up + c, u);
    if constexpr (BACK) load_values<DT, W, STREAM>(a.grad, row * a.ld_grad + c, d);
#pragma unroll
    for (int j = 0; j < W; ++j) {
      float h, slope;
      act_both<ACT>(g[j], h, slope);
      if constexpr (BACK) {
        g[j] = d[j] * u[j] * slope;
        u[j] = d[j] * h;
      } else {
        y[j] = h * u[j];
      }
    }
    if constexpr (BACK) {
      store_values<DT, W, STREAM>(a.d_gate, row * a.ld_dgate + c, g);
      store_values<DT, W, STREAM>(a.d_up, row * a.ld_dup + c, u);
    } else {
      store_values<DT, W, STREAM>(a.out, row * a.ld_out + c, y);
    }
  };
  if (V == 1 || c + V <= a.n) {
    some(std::integral_constant<int, V>{}, c);
  } else {
    for (int64_t i = c; i < a.n; ++i) some(std::integral_constant<int, 1>{}, i);
  }
}

template <int DT, int ACT, bool BACK>
void launch_act(const Args& a, bool wide, unsigned grid, hipStream_t s) {
  if (wide && a.rows * a.n * (DT == 0 ? 4 : 2) * (BACK ? 5 : 3) > STREAM_BYTES)
    gated_kernel<DT, ACT, WIDE<DT>, BACK, true><<<grid, 256, 0, s>>>(a);
  else if (wide)
    gated_kernel<DT, ACT, WIDE<DT>, BACK, false><<<grid, 256, 0, s>>>(a);
  else
    gated_kernel<DT, ACT, 1, BACK, false><<<grid, 256, 0, s>>>(a);
}

template <int DT, bool BACK>
void launch_type(const Args& a, int act, bool wide, unsigned grid, hipStream_t s) {
  switch (act) {
    case HI2X_ACT_RELU: return launch_act<DT, HI2X_ACT_RELU, BACK>(a, wide, grid, s);
    case HI2X_ACT_SILU: return launch_act<DT, HI2X_ACT_SILU, BACK>(a, wide, grid, s);
    case HI2X_ACT_GELU: return launch_act<DT, HI2X_ACT_GELU, BACK>(a, wide, grid, s);
    case HI2X_ACT_GELU_TANH: return launch_act<DT, HI2X_ACT_GELU_TANH, BACK>(a, wide, grid, s);
    default: return launch_act<DT, HI2X_ACT_NONE, BACK>(a, wide, grid, s);
  }
}

template <bool BACK>
int gated(Args a, int dtype, int act, const char* what, void* stream) {
  HI2X_REQUIRE(dtype >= 0 && dtype <= 2, "%s: dtype %d", what, dtype);
  HI2X_REQUIRE(act >= HI2X_ACT_NONE && act <= HI2X_ACT_GELU_TANH, "%s: activation %d", what, act);
  HI2X_REQUIRE(a.rows >= 0 && a.n >= 0 && a.rows < (1ll << 40) && a.n < (1ll << 40),
               "%s: bad shape", what);
  if (a.rows == 0 || a.n == 0) return HI2X_OK;
  const void* ps[6] = {a.gate, a.up, BACK ? a.grad : a.gate, BACK ? a.d_gate : a.out,
                       BACK ? a.d_up : a.out, a.up};
  int64_t* lds[6] = {&a.ld_gate, &a.ld_up, BACK ? &a.ld_grad : &a.ld_gate,
                     BACK ? &a.ld_dgate : &a.ld_out, BACK ? &a.ld_dup : &a.ld_out, &a.ld_up};
  const int size = dtype == 0 ? 4 : 2;
  bool whole = true, wide = true;
  for (int i = 0; i < 6; ++i) {
    HI2X_REQUIRE(ps[i], "%s: null buffer", what);
    HI2X_REQUIRE(a.rows == 1 || *lds[i] >= a.n, "%s: rows overlap", what);
    whole = whole && (a.rows == 1 || *lds[i] == a.n);
    wide = wide && ((uintptr_t)ps[i] & 15) == 0;
  }
  if (whole) {  // one row of all elements
    a.n *= a.rows;
    a.rows = 1;
  } else {
    for (int i = 0; i < 6; ++i) wide = wide && (*lds[i] * size & 15) == 0;
  }
  const int64_t vec = wide ? 16 / size : 1, nv = (a.n + vec - 1) / vec;
  a.shift = 8;
  while (a.shift > 0 && (1ll << (a.shift - 1)) >= nv) --a.shift;
  const int64_t pieces = (nv + (1ll << a.shift) - 1) >> a.shift;
  const int64_t bands = (a.rows + (256 >> a.shift) - 1) / (256 >> a.shift);
  HI2X_REQUIRE(pieces < (1ll << 31) && bands < (1ll << 31) && pieces * bands < (1ll << 31),
               "%s: too many elements", what);
  a.pieces = (uint32_t)pieces;
  const unsigned grid = (unsigned)(pieces * bands);
  const hipStream_t s = as_stream(stream);
  if (dtype == 0)
    launch_type<0, BACK>(a, act, wide, grid, s);
  else if (dtype == 1)
    launch_type<1, BACK>(a, act, wide, grid, s);
  else
    launch_type<2, BACK>(a, act, wide, grid, s);
  return launch_status(what);
}

}  // namespace
}  // namespace hi2x

using namespace hi2x;

extern "C" int hi2x_gated(const void* gate, int64_t ld_gate, const void* up, int64_t ld_up,
                          int64_t rows, int64_t n, int dtype, int act, void* out, int64_t ld_out,
                          void* stream) {
  clear_error();
  Args a{};
  a.gate = gate, a.up = up, a.out = out;
  a.ld_gate = ld_gate, a.ld_up = ld_up, a.ld_out = ld_out;
  a.rows = rows, a.n = n;
  return gated<false>(a, dtype, act, "gated", stream);
}

extern "C" int hi2x_gated_backward(const void* grad, int64_t ld_grad, const void* gate,
                                   int64_t ld_gate, const void* up, int64_t ld_up, int64_t rows,
                                   int64_t n, int dtype, int act, void* d_gate, int64_t ld_dgate,
                                   void* d_up, int64_t ld_dup, void* stream) {
  clear_error();
  Args a{};
  a.grad = grad, a.gate = gate, a.up = up, a.d_gate = d_gate, a.d_up = d_up;
  a.ld_grad = ld_grad, a.ld_gate = ld_gate, a.ld_up = ld_up;
  a.ld_dgate = ld_dgate, a.ld_dup = ld_dup;
  a.rows = rows, a.n = n;
  return gated<true>(a, dtype, act, "gated_backward", stream);
}
