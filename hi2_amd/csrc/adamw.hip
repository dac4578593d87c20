// The AdamW step over many tensors at once, with the moments in 32 bits or in 8.
//
//   m = b1 m + (1 - b1) g,   v = b2 v + (1 - b2) g^2,
//   p = p (1 - lr wd) - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// in float32, each product and sum rounded by itself.  Nothing is reused, so HBM bounds it: 28
// bytes of a float32 weight with 32-bit moments, 16 with 8-bit ones.  192 tensors of 1024 x 2048 in
// bfloat16 with masters 2049 us (5.9 TB/s), 3 of 14336 x 4096 in float32 with 8-bit moments 600 (4.7).
//
// 8-bit moments: blocks of 256 elements (one wave's 64 lanes x 4) hold m = +-q^2 d with |q| <=
// 127, and the root of v as q^2 d with q <= 255, d the block's largest over 127^2 or 255^2.  The
// squares put the codes where small values need them (the least nonzero m is 2^-14 of the
// largest, the least nonzero v 2^-32), and both ways are exact but for one rounding of a product:
// the borders (q + 1/2)^2 between codes are floats, so a code is found from an approximate root
// and two comparisons.  A root that is not zero keeps at least the code 1: a v that vanished under
// a living m would make the quotient explode.  A block whose largest is not finite becomes NaN.
#include "packed.h"

namespace hi2x {
namespace {

constexpr int BLOCK = HI2X_ADAMW_BLOCK, CHUNK = HI2X_ADAMW_CHUNK;
constexpr int TENSORS = 192, GROUPS = 16;  // of one launch: its arguments stay below 4 KB

struct Launch {
  void* p[TENSORS];
  const void* g[TENSORS];
  hi2x_adamw_group group[GROUPS];
  const hi2x_adamw_tensor* tensors;  // device, those of this launch
  int64_t first_chunk;
  void* m;
  void* v;
  float* md;
  float* vd;
  float* master;
  int64_t* steps;  // those of this launch
  int32_t* done;
  int32_t count, first_group;
};
static_assert(sizeof(Launch) <= 4096 - 64, "kernel arguments");

// Elements i .. i + 3 of a tensor of n, zero past its end.  `vec`: they are there and aligned.
// STREAM: past the caches, where a call touches twice what the last one holds (256 MB) and nothing of
// it would be there for the next.  192 tensors of 1024 x 2048 in bfloat16 with masters 2135 us,
// so 2049; 1024 x 4096 in float32, 29, would take 33.
constexpr int64_t STREAM_BYTES = 512ll << 20;
template <bool STREAM>
__device__ __forceinline__ float4 get(const float4* p) {
  if constexpr (!STREAM) return *p;
  const f32x4v f = __builtin_nontemporal_load(reinterpret_cast<const f32x4v*>(p));
  return make_float4(f.x, f.y, f.z, f.w);
}
template <bool STREAM>
__device__ __forceinline__ uint2 get(const uint2* p) {
  if constexpr (!STREAM) return *p;
  const u32x2 h = __builtin_nontemporal_load(reinterpret_cast<const u32x2*>(p));
  return make_uint2(h.x, h.y);
}
template <bool STREAM>
__device__ __forceinline__ uint32_t get(const uint32_t* p) {
  return STREAM ? __builtin_nontemporal_load(p) : *p;
}
template <bool STREAM>
__device__ __forceinline__ void put(float4* p, float4 v) {
  if constexpr (STREAM)
    __builtin_nontemporal_store(f32x4v{v.x, v.y, v.z, v.w}, reinterpret_cast<f32x4v*>(p));
  else
    *p = v;
}
template <bool STREAM>
__device__ __forceinline__ void put(uint2* p, uint2 v) {
  if constexpr (STREAM)
    __builtin_nontemporal_store(u32x2{v.x, v.y}, reinterpret_cast<u32x2*>(p));
  else
    *p = v;
}
template <bool STREAM>
__device__ __forceinline__ void put(uint32_t* p, uint32_t v) {
  if constexpr (STREAM)
    __builtin_nontemporal_store(v, p);
  else
    *p = v;
}

template <int DT, bool STREAM = false>
__device__ __forceinline__ void load4(const void* p, int64_t i, int64_t n, bool vec,
                                      float (&x)[4]) {
  if (vec) {
    if constexpr (DT == 0) {
      const float4 f =
          get<STREAM>(reinterpret_cast<const float4*>(static_cast<const float*>(p) + i));
      x[0] = f.x, x[1] = f.y, x[2] = f.z, x[3] = f.w;
    } else {
      const uint2 h =
          get<STREAM>(reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p) + i));
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint16_t b = (uint16_t)((j < 2 ? h.x : h.y) >> (16 * (j & 1)));
        x[j] = DT == 1 ? f16_from_bits(b) : __uint_as_float((uint32_t)b << 16);
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = i + j < n ? load_as_f32(p, i + j, DT) : 0.0f;
  }
}

template <int DT, bool STREAM = false>
__device__ __forceinline__ void store4(void* p, int64_t i, int64_t n, bool vec,
                                       const float (&x)[4]) {
  if (vec) {
    if constexpr (DT == 0) {
      put<STREAM>(reinterpret_cast<float4*>(static_cast<float*>(p) + i),
                  make_float4(x[0], x[1], x[2], x[3]));
    } else {
      uint32_t w[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const uint32_t a = DT == 1 ? f16_bits(x[2 * j]) : bf16_bits(x[2 * j]);
        const uint32_t b = DT == 1 ? f16_bits(x[2 * j + 1]) : bf16_bits(x[2 * j + 1]);
        w[j] = a | b << 16;
      }
      put<STREAM>(reinterpret_cast<uint2*>(static_cast<uint16_t*>(p) + i), make_uint2(w[0], w[1]));
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (i + j < n) store_from_f32(p, i + j, DT, x[j]);
  }
}

// The largest over the wave.  Magnitudes as their bits: a NaN is above infinity, and stays.
__device__ __forceinline__ uint32_t wave_largest(const float (&x)[4]) {
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t b = __float_as_uint(x[j]) & 0x7fffffffu;
    m = m > b ? m : b;
  }
#pragma unroll
  for (int d = 32; d; d >>= 1) {
    const uint32_t o = (uint32_t)__shfl_xor((int)m, d);
    m = m > o ? m : o;
  }
  return m;
}

// A block's unit from the bits of its largest, and its reciprocal for the codes.
template <int STEPS>
__device__ __forceinline__ float block_unit(uint32_t largest, float& r) {
  if (largest >= 0x7f800000u) {
    r = 0.0f;
    return __uint_as_float(0x7fc00000u);
  }
  const float d = __uint_as_float(largest) * (float)(1.0 / (STEPS * STEPS));
  const bool normal = d >= 1.1754943508222875e-38f;
  r = normal ? 1.0f / d : 0.0f;
  return normal ? d : 0.0f;
}

// The code nearest to sqrt(z), halves up.
__device__ __forceinline__ int code_of(float z) {
  const float q = __builtin_floorf(__builtin_amdgcn_sqrtf(z) + 0.5f);
  const float q2 = q * q;
  int c = (int)q;
  if (q > 0.0f && z < q2 - q + 0.25f) --c;
  if (z >= q2 + q + 0.25f) ++c;
  return c;
}

__device__ __forceinline__ uint32_t encode_m(const float (&m)[4], float& unit) {
  float r;
  unit = block_unit<127>(wave_largest(m), r);
  uint32_t w = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int c = code_of(fabsf(m[j]) * r);
    w |= ((uint32_t)(m[j] < 0.0f ? -c : c) & 255u) << (8 * j);
  }
  return w;
}

__device__ __forceinline__ uint32_t encode_root(const float (&s)[4], float& unit) {
  float r;
  unit = block_unit<255>(wave_largest(s), r);
  uint32_t w = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    int c = code_of(s[j] * r);
    if (c == 0 && s[j] > 0.0f) c = 1;
    w |= (uint32_t)c << (8 * j);
  }
  return w;
}

__device__ __forceinline__ void decode_m(uint32_t w, float unit, float (&m)[4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int c = (int)(int8_t)(w >> (8 * j));
    m[j] = (float)(c * (c < 0 ? -c : c)) * unit;
  }
}

__device__ __forceinline__ void decode_root(uint32_t w, float unit, float (&v)[4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int c = (int)((w >> (8 * j)) & 255u);
    const float s = (float)(c * c) * unit;
    v[j] = s * s;
  }
}

// b^t by squaring.
__device__ __forceinline__ double power(double b, int64_t t) {
  double p = 1.0;
  for (; t > 0; t >>= 1, b *= b)
    if (t & 1) p *= b;
  return p;
}

// A group's factors at a tensor's step.
struct Factors {
  float b1, c1, b2, c2, root, eps, decay, step;
};

// One chunk of a tensor.  The factors of a tensor's step are found once a workgroup (in 64 bits)
// from its own count of steps on the device, so that a captured step counts on in its replays;
// the last of a tensor's workgroups to end writes the new count.
template <int DT, int BITS, bool MASTER, bool STREAM>
__global__ __launch_bounds__(256) void adamw_kernel(Launch a) {
  __shared__ Factors shared;
  __shared__ int which;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t chunk = a.first_chunk + blockIdx.x;
  // the tensor whose chunks hold this one: the last that begins at or before it and has any
  if (wave == 0) {
    for (int i0 = 0; i0 < a.count; i0 += 64) {
      const int i = i0 + lane;
      bool here = false;
      if (i < a.count) {
        const int64_t f = a.tensors[i].first_chunk;
        here = chunk >= f && chunk < f + (a.tensors[i].n + CHUNK - 1) / CHUNK;
      }
      if (here) which = i;
    }
  }
  __syncthreads();
  const int i = __builtin_amdgcn_readfirstlane(which);
  const void* gp = a.g[i];
  if (!gp) return;
  void* pp = a.p[i];
  const hi2x_adamw_tensor t = a.tensors[i];
  if (tid == 0) {
    const hi2x_adamw_group& h = a.group[t.group - a.first_group];
    const int64_t count = a.steps[i] + 1;
    const double lr = h.lr_tensor ? (double)*h.lr_tensor : h.lr;
    const double c1 = 1.0 - power(h.beta1, count), c2 = 1.0 - power(h.beta2, count);
    shared = Factors{(float)h.beta1, (float)(1.0 - h.beta1), (float)h.beta2,
                     (float)(1.0 - h.beta2), (float)(1.0 / sqrt(c2)), (float)h.eps,
                     (float)(1.0 - lr * h.weight_decay), (float)(lr / c1)};
  }
  __syncthreads();
  const Factors f = shared;
  const uintptr_t mask = DT == 0 ? 15 : 7;
  const bool aligned = (((uintptr_t)pp | (uintptr_t)gp) & mask) == 0;
  const int64_t begin = (chunk - t.first_chunk) * CHUNK;
  for (int b = wave; b < CHUNK / BLOCK; b += 4) {
    const int64_t i0 = begin + b * BLOCK;
    if (i0 >= t.n) break;
    const int64_t e = i0 + 4 * lane, at = t.start + e;  // at: in the moments
    const bool vec = aligned && e + 4 <= t.n;
    float p[4], g[4], m[4], v[4], s[4];
    load4<DT, STREAM>(gp, e, t.n, vec, g);
    if constexpr (MASTER)
      load4<0, STREAM>(a.master, at, at + 4, true, p);
    else
      load4<DT, STREAM>(pp, e, t.n, vec, p);
    const int64_t blk = (t.start + i0) / BLOCK;
    if constexpr (BITS == 32) {
      load4<0, STREAM>(a.m, at, at + 4, true, m);
      load4<0, STREAM>(a.v, at, at + 4, true, v);
    } else {
      decode_m(get<STREAM>(static_cast<const uint32_t*>(a.m) + at / 4), a.md[blk], m);
      decode_root(get<STREAM>(static_cast<const uint32_t*>(a.v) + at / 4), a.vd[blk], v);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      m[j] = m[j] * f.b1 + g[j] * f.c1;
      v[j] = v[j] * f.b2 + (g[j] * g[j]) * f.c2;
      s[j] = sqrtf(v[j]);
      p[j] = p[j] * f.decay - (m[j] / (s[j] * f.root + f.eps)) * f.step;
    }
    store4<DT, STREAM>(pp, e, t.n, vec, p);
    // (past the tensor's end p may be 0 / 0, where eps is 0: the masters stay zero there)
    if constexpr (MASTER) store4<0, STREAM>(a.master + t.start, e, t.n, e + 4 <= t.n, p);
    if constexpr (BITS == 32) {
      store4<0, STREAM>(a.m, at, at + 4, true, m);
      store4<0, STREAM>(a.v, at, at + 4, true, v);
    } else {
      float md, vd;
      const uint32_t mc = encode_m(m, md), vc = encode_root(s, vd);
      put<STREAM>(static_cast<uint32_t*>(a.m) + at / 4, mc);
      put<STREAM>(static_cast<uint32_t*>(a.v) + at / 4, vc);
      if (lane == 0) a.md[blk] = md, a.vd[blk] = vd;
    }
  }
  if (tid == 0) {
    const int chunks = (int)((t.n + CHUNK - 1) / CHUNK);
    if (atomicAdd(&a.done[i], 1) == chunks - 1) {
      a.done[i] = 0;
      a.steps[i] += 1;
    }
  }
}

// Moments between 32 bits and 8, a block to a wave.
__global__ __launch_bounds__(256) void adamw_hold_kernel(const float* m, const float* v,
                                                         int64_t blocks, uint32_t* mc,
                                                         uint32_t* vc, float* md, float* vd) {
  const int lane = threadIdx.x & 63;
  const int64_t b = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (b >= blocks) return;
  const int64_t e = b * BLOCK + 4 * lane;
  float x[4], s[4], u;
  load4<0>(m, e, e + 4, true, x);
  load4<0>(v, e, e + 4, true, s);
  mc[e / 4] = encode_m(x, u);
  if (lane == 0) md[b] = u;
#pragma unroll
  for (int j = 0; j < 4; ++j) s[j] = sqrtf(s[j]);
  vc[e / 4] = encode_root(s, u);
  if (lane == 0) vd[b] = u;
}

__global__ __launch_bounds__(256) void adamw_moments_kernel(const uint32_t* mc,
                                                            const uint32_t* vc, const float* md,
                                                            const float* vd, int64_t blocks,
                                                            float* m, float* v) {
  const int lane = threadIdx.x & 63;
  const int64_t b = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (b >= blocks) return;
  const int64_t e = b * BLOCK + 4 * lane;
  float x[4];
  decode_m(mc[e / 4], md[b], x);
  store4<0>(m, e, e + 4, true, x);
  decode_root(vc[e / 4], vd[b], x);
  store4<0>(v, e, e + 4, true, x);
}

int64_t chunks_of(int64_t n) { return (n + CHUNK - 1) / CHUNK; }

template <int DT, int BITS, bool STREAM>
void launch_stream(const Launch& a, unsigned grid, hipStream_t s) {
  if constexpr (DT != 0) {
    if (a.master) {
      adamw_kernel<DT, BITS, true, STREAM><<<grid, 256, 0, s>>>(a);
      return;
    }
  }
  adamw_kernel<DT, BITS, false, STREAM><<<grid, 256, 0, s>>>(a);
}

// elements: of the whole step
template <int DT, int BITS>
void launch(const Launch& a, unsigned grid, int64_t elements, hipStream_t s) {
  const int64_t each = (DT == 0 ? 12 : 6) + (BITS == 32 ? 16 : 4) + (a.master ? 8 : 0);
  if (elements * each > STREAM_BYTES)
    launch_stream<DT, BITS, true>(a, grid, s);
  else
    launch_stream<DT, BITS, false>(a, grid, s);
}

int check_blocks(const void* a, const void* b, const void* c, const void* d, const void* e,
                 const void* f, int64_t blocks, const char* what) {
  HI2X_REQUIRE(blocks >= 0 && blocks < (1ll << 32), "%s: %lld blocks", what, (long long)blocks);
  if (blocks == 0) return HI2X_OK;
  HI2X_REQUIRE(a && b && c && d && e && f, "%s: null buffer", what);
  HI2X_REQUIRE((((uintptr_t)a | (uintptr_t)b | (uintptr_t)c | (uintptr_t)d) & 15) == 0,
               "%s: buffers not aligned to 16 bytes", what);
  return HI2X_OK;
}

}  // namespace
}  // namespace hi2x

using namespace hi2x;

extern "C" int hi2x_adamw_step(const hi2x_adamw_tensor* tensors,
                               const hi2x_adamw_tensor* device_tensors, void* const* params,
                               const void* const* grads, int64_t count, int dtype, int bits,
                               const hi2x_adamw_group* groups, int64_t n_groups, void* m, void* v,
                               float* m_unit, float* v_unit, float* master, int64_t* steps,
                               int32_t* done, void* stream) {
  clear_error();
  HI2X_REQUIRE(count >= 0 && n_groups >= 0, "adamw_step: bad counts");
  HI2X_REQUIRE(dtype >= 0 && dtype <= 2, "adamw_step: dtype %d", dtype);
  HI2X_REQUIRE(bits == 32 || bits == 8, "adamw_step: moments of %d bits", bits);
  HI2X_REQUIRE(!master || dtype != 0, "adamw_step: a master of float32 parameters");
  if (count == 0) return HI2X_OK;
  HI2X_REQUIRE(tensors && device_tensors && params && grads && groups && m && v && steps && done,
               "adamw_step: null argument");
  HI2X_REQUIRE(bits == 32 || (m_unit && v_unit), "adamw_step: null argument");
  HI2X_REQUIRE((((uintptr_t)m | (uintptr_t)v | (uintptr_t)master) & 15) == 0,
               "adamw_step: moments not aligned to 16 bytes");
  int64_t next = 0, chunk = 0, elements = 0;
  for (int64_t i = 0; i < count; ++i) {
    const hi2x_adamw_tensor& t = tensors[i];
    HI2X_REQUIRE(t.n > 0 && t.start >= next && t.start % BLOCK == 0,
                 "adamw_step: tensor %lld overlaps the one before it", (long long)i);
    HI2X_REQUIRE(t.first_chunk >= 0 && (i == 0 || t.first_chunk == chunk),
                 "adamw_step: chunks of tensor %lld", (long long)i);
    HI2X_REQUIRE(t.group >= 0 && t.group < n_groups && (i == 0 || t.group >= tensors[i - 1].group),
                 "adamw_step: group %d of tensor %lld", t.group, (long long)i);
    HI2X_REQUIRE(!grads[i] || params[i], "adamw_step: null parameter %lld", (long long)i);
    next = t.start + t.n;
    chunk = t.first_chunk + chunks_of(t.n);
    if (grads[i]) elements += t.n;
  }
  const hipStream_t s = as_stream(stream);
  for (int64_t i = 0; i < count;) {
    Launch a;
    a.count = 0;
    a.first_group = tensors[i].group;
    const int64_t first = i;
    int last_group = a.first_group;
    bool any = false;
    for (; i < count && a.count < TENSORS && tensors[i].group < a.first_group + GROUPS; ++i) {
      a.p[a.count] = params[i];
      a.g[a.count] = grads[i];
      any |= grads[i] != nullptr;
      last_group = tensors[i].group;
      ++a.count;
    }
    if (!any) continue;
    for (int g = a.first_group; g <= last_group; ++g) a.group[g - a.first_group] = groups[g];
    a.tensors = device_tensors + first;
    a.first_chunk = tensors[first].first_chunk;
    a.m = m, a.v = v, a.md = m_unit, a.vd = v_unit, a.master = master;
    a.steps = steps + first, a.done = done + first;
    const int64_t grid = tensors[i - 1].first_chunk + chunks_of(tensors[i - 1].n) - a.first_chunk;
    HI2X_REQUIRE(grid < (1ll << 31), "adamw_step: too many elements");
    switch (dtype * 2 + (bits == 8)) {
      case 0: launch<0, 32>(a, (unsigned)grid, elements, s); break;
      case 1: launch<0, 8>(a, (unsigned)grid, elements, s); break;
      case 2: launch<1, 32>(a, (unsigned)grid, elements, s); break;
      case 3: launch<1, 8>(a, (unsigned)grid, elements, s); break;
      case 4: launch<2, 32>(a, (unsigned)grid, elements, s); break;
      default: launch<2, 8>(a, (unsigned)grid, elements, s);
    }
    if (int rc = launch_status("adamw_step")) return rc;
  }
  return HI2X_OK;
}

extern "C" int hi2x_adamw_hold(const float* m, const float* v, int64_t blocks, void* m_codes,
                               void* v_codes, float* m_unit, float* v_unit, void* stream) {
  clear_error();
  if (int rc = check_blocks(m, v, m_codes, v_codes, m_unit, v_unit, blocks, "adamw_hold"))
    return rc;
  if (blocks == 0) return HI2X_OK;
  adamw_hold_kernel<<<(unsigned)((blocks + 3) / 4), 256, 0, as_stream(stream)>>>(
      m, v, blocks, static_cast<uint32_t*>(m_codes), static_cast<uint32_t*>(v_codes), m_unit,
      v_unit);
  return launch_status("adamw_hold");
}

extern "C" int hi2x_adamw_moments(const void* m_codes, const void* v_codes, const float* m_unit,
                                  const float* v_unit, int64_t blocks, float* m, float* v,
                                  void* stream) {
  clear_error();
  if (int rc = check_blocks(m, v, m_codes, v_codes, m_unit, v_unit, blocks, "adamw_moments"))
    return rc;
  if (blocks == 0) return HI2X_OK;
  adamw_moments_kernel<<<(unsigned)((blocks + 3) / 4), 256, 0, as_stream(stream)>>>(
      static_cast<const uint32_t*>(m_codes), static_cast<const uint32_t*>(v_codes), m_unit, v_unit,
      blocks, m, v);
  return launch_status("adamw_moments");
}
