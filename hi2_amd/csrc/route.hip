// The router of an MoE layer: scores, top-k, weights and the experts' slot order, its
// gradient, and the weighted sum of the experts' outputs.
//
// 16 lanes hold one token's E scores (expert 16 i + lane in register i), so four tokens
// share a wave and every reduction over the experts is four DPP steps without LDS.  The
// passes read a few MB at most: what bounds them is launches and the latency of the top-k
// loop, so a workgroup does up to 64 tokens from logits to indices, and where they are all there
// are the slot order too.  That order needs no sort: a token chooses an expert at most once,
// so 64 tokens' choices of an expert are one 64-bit mask, a choice's rank is the number of
// lower bits, and the stable order follows from the masks' popcounts.
#include "packed.h"

namespace hi2x {
namespace {

constexpr int RK = 32;      // most choices
constexpr int RE = 512;     // most experts
constexpr int RG = 64;      // most groups
constexpr int SCAN_OVER = 1024;  // workgroups above which the counts get a scan of their own

template <int CTRL>
__device__ __forceinline__ double dpp_d(double v) {
  const long long b = __builtin_bit_cast(long long, v);
  const uint32_t lo = (uint32_t)dpp<CTRL>((int)b), hi = (uint32_t)dpp<CTRL>((int)(b >> 32));
  return __builtin_bit_cast(double, (long long)((unsigned long long)hi << 32 | lo));
}
__device__ __forceinline__ double row_sum(double v) {
  v += dpp_d<0xB1>(v);
  v += dpp_d<0x4E>(v);
  v += dpp_d<0x141>(v);
  v += dpp_d<0x140>(v);
  return v;
}

// An order of u32 that is the floats' (no NaN here; -0 counts as 0); above 0 always.
__device__ __forceinline__ uint32_t order_key(float v) {
  const uint32_t b = __float_as_uint(v + 0.0f);
  return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}

// One token's logits (-inf where there is no expert, or for NaN) and scores.  The softmax's
// sum is taken in f64 and rounded once, so that scores do not depend on the order of its
// terms: experts ranked by score + bias come out the same however the sum is formed.
template <int EPL>
__device__ __forceinline__ void token_scores(const void* logits, int dtype, int64_t at, int e,
                                             int scoring, int l16, float (&v)[EPL],
                                             float (&p)[EPL]) {
  const float ninf = -__builtin_inff();
  // all loads in flight before the first conversion (past the end: the last expert's)
  if (dtype == 0) {
    const float* p = static_cast<const float*>(logits) + at;
#pragma unroll
    for (int i = 0; i < EPL; ++i) v[i] = p[16 * i + l16 < e ? 16 * i + l16 : e - 1];
  } else {
    const uint16_t* p = static_cast<const uint16_t*>(logits) + at;
    uint16_t r[EPL];
#pragma unroll
    for (int i = 0; i < EPL; ++i) r[i] = p[16 * i + l16 < e ? 16 * i + l16 : e - 1];
#pragma unroll
    for (int i = 0; i < EPL; ++i)
      v[i] = dtype == 1 ? f16_from_bits(r[i]) : __uint_as_float((uint32_t)r[i] << 16);
  }
#pragma unroll
  for (int i = 0; i < EPL; ++i) v[i] = 16 * i + l16 < e && v[i] == v[i] ? v[i] : ninf;
  if (scoring == 1) {
#pragma unroll
    for (int i = 0; i < EPL; ++i) p[i] = 1.0f / (1.0f + expf(-v[i]));
    return;
  }
  uint32_t mk = 0;
#pragma unroll
  for (int i = 0; i < EPL; ++i) {
    const uint32_t k = order_key(v[i]);
    mk = k > mk ? k : mk;
  }
  mk = row_umax(mk);
  const float m = __uint_as_float((mk & 0x80000000u) ? mk & 0x7fffffffu : ~mk);
  double sum = 0.0;
#pragma unroll
  for (int i = 0; i < EPL; ++i) {
    p[i] = v[i] > ninf ? expf(v[i] - m) : 0.0f;
    sum += (double)p[i];
  }
  const float s = (float)row_sum(sum);
#pragma unroll
  for (int i = 0; i < EPL; ++i) p[i] = s > 0.0f ? p[i] / s : (s == s ? 0.0f : s);
}

// The best two values of a row of lanes, from each lane's two.
template <int CTRL>
__device__ __forceinline__ void best2_step(float& b1, float& b2) {
  const float o1 = __int_as_float(dpp<CTRL>(__float_as_int(b1)));
  const float o2 = __int_as_float(dpp<CTRL>(__float_as_int(b2)));
  b2 = fmaxf(fminf(b1, o1), fmaxf(b2, o2));
  b1 = fmaxf(b1, o1);
}
__device__ __forceinline__ void row_best2(float& b1, float& b2) {
  best2_step<0xB1>(b1, b2);
  best2_step<0x4E>(b1, b2);
  best2_step<0x141>(b1, b2);
  best2_step<0x140>(b1, b2);
}

// Whether groups of gs experts are whole registers of a token, at most one to a lane.
__host__ __device__ inline bool whole_rows(int64_t gs, int64_t groups) {
  return gs % 16 == 0 && groups <= 16;
}

struct RouteArgs {
  const void* logits;
  int dtype;
  int64_t ld, t;
  int e, k, scoring;
  const float* bias;
  int groups, top_groups, renorm;
  float scale;
  int64_t* index;
  float* weights;
  int64_t* rows;
  int64_t* offs;
  int64_t* slots;
  uint8_t* hist;    // [e][nbp] tokens of each workgroup
  int32_t* prefix;  // [e][nbp] tokens of earlier workgroups, or null
  int nbp;          // workgroups, up to a multiple of 16 (the rest counts nothing)
};

// cnt[0..e) -> running sums in place, by the first wave.
__device__ __forceinline__ void scan_experts(int* cnt, int e) {
  if (threadIdx.x < 64) {
    const int lane = threadIdx.x;
    int before = 0;
    for (int e0 = 0; e0 < e; e0 += 64) {
      int v = e0 + lane < e ? cnt[e0 + lane] : 0;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(v, d);
        if (lane >= d) v += o;
      }
      v += before;
      if (e0 + lane < e) cnt[e0 + lane] = v;
      before = __shfl(v, 63);
    }
  }
  __syncthreads();
}

// NT / 16 tokens to a workgroup.
template <int EPL, int NT>
__global__ __launch_bounds__(NT) void route_kernel(RouteArgs a) {
  constexpr int RT = NT / 16;
  __shared__ int sel_e[RT][RK];
  __shared__ float sel_p[RT][RK];
  __shared__ uint32_t mask[RE][2];
  __shared__ int cnt[RE];
  extern __shared__ float keys[];  // with groups: [RT][e + groups]
  const int tid = threadIdx.x, tok = tid >> 4, l16 = tid & 15;
  const int64_t t0 = (int64_t)blockIdx.x * RT, t = t0 + tok;
  const bool live = t < a.t;
  const int e = a.e, k = a.k;
  for (int i = tid; i < e; i += NT) mask[i][0] = mask[i][1] = 0;
  float v[EPL], p[EPL];
  token_scores<EPL>(a.logits, a.dtype, (live ? t : a.t - 1) * a.ld, e, a.scoring, l16, v, p);
  // the keys the experts are ranked by; 0: taken, or not taking part
  const float ninf = -__builtin_inff();
  uint32_t key[EPL];
  if (a.bias) {
    float b[EPL];
#pragma unroll
    for (int i = 0; i < EPL; ++i) b[i] = a.bias[16 * i + l16 < e ? 16 * i + l16 : e - 1];
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      const float c = p[i] + b[i];
      v[i] = v[i] > ninf && c == c ? c : ninf;
    }
  }
#pragma unroll
  for (int i = 0; i < EPL; ++i) key[i] = 16 * i + l16 < e ? order_key(v[i]) : 0u;
  if (a.top_groups < a.groups) {
    const int gs = e / a.groups, pitch = e + a.groups;
    const float inv = 1.0f / (float)gs;
    uint32_t gk[RG / 16];
#pragma unroll
    for (int i = 0; i < RG / 16; ++i) gk[i] = 0;
    if (whole_rows(gs, a.groups)) {
      // whole registers to a group: its best two by exchanges over the 16 lanes
      float b1 = ninf, b2 = ninf;
      int left = gs / 16, g = 0;
#pragma unroll
      for (int i = 0; i < EPL; ++i) {
        b2 = v[i] > b1 ? b1 : (v[i] > b2 ? v[i] : b2);
        b1 = v[i] > b1 ? v[i] : b1;
        if (--left == 0) {
          row_best2(b1, b2);
          const float s = a.bias ? b1 + b2 : b1;
          if (l16 == g) gk[0] = order_key(s == s ? s : ninf);
          b1 = b2 = ninf;
          left = gs / 16;
          ++g;
        }
      }
      if (l16 >= a.groups) gk[0] = 0;
    } else {
#pragma unroll
      for (int i = 0; i < EPL; ++i) {
        const int x = 16 * i + l16;
        if (x < e) keys[tok * pitch + x + (int)(((float)x + 0.5f) * inv)] = v[i];
      }
      __syncthreads();
#pragma unroll
      for (int i = 0; i < RG / 16; ++i) {
        const int g = 16 * i + l16;
        if (g >= a.groups) continue;
        float b1 = ninf, b2 = ninf;
        for (int x = 0; x < gs; ++x) {
          const float c = keys[tok * pitch + g * (gs + 1) + x];
          b2 = c > b1 ? b1 : (c > b2 ? c : b2);
          b1 = c > b1 ? c : b1;
        }
        const float s = a.bias && gs > 1 ? b1 + b2 : b1;
        gk[i] = order_key(s == s ? s : ninf);
      }
    }
    uint32_t keep0 = 0, keep1 = 0;
    for (int j = 0; j < a.top_groups; ++j) {
      uint32_t bk = 0;
      int bg = RG;
#pragma unroll
      for (int i = 0; i < RG / 16; ++i)
        if (gk[i] > bk) {
          bk = gk[i];
          bg = 16 * i + l16;
        }
      const uint32_t m = row_umax(bk);
      const int w = (int)row_umin(bk == m ? (uint32_t)bg : 0xffffu);
#pragma unroll
      for (int i = 0; i < RG / 16; ++i)
        if (16 * i + l16 == w) gk[i] = 0;
      keep0 |= w < 32 ? 1u << (w & 31) : 0u;
      keep1 |= w >= 32 ? 1u << (w & 31) : 0u;
    }
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      const int x = 16 * i + l16;
      const int g = (int)(((float)x + 0.5f) * inv);
      if (!(((g < 32 ? keep0 : keep1) >> (g & 31)) & 1u)) key[i] = 0;
    }
  }
  for (int j = 0; j < k; ++j) {
    uint32_t bk = 0;
#pragma unroll
    for (int i = 0; i < EPL; ++i) bk = key[i] > bk ? key[i] : bk;
    const uint32_t m = row_umax(bk);
    uint32_t be = RE;
#pragma unroll
    for (int i = EPL - 1; i >= 0; --i) be = key[i] == m ? (uint32_t)(16 * i + l16) : be;
    const uint32_t w = row_umin(be);
    if (be == w) {
      float bp = 0.0f;
#pragma unroll
      for (int i = 0; i < EPL; ++i) {
        const bool it = (uint32_t)(16 * i + l16) == w;
        bp = it ? p[i] : bp;
        key[i] = it ? 0u : key[i];
      }
      sel_e[tok][j] = (int)w;
      sel_p[tok][j] = bp;
    }
  }
  __syncthreads();
  float sum = 0.0f;
  for (int j = 0; j < k; ++j) sum += sel_p[tok][j];
  for (int j = l16; j < k; j += 16) {
    if (!live) break;
    const int x = sel_e[tok][j];
    float w = sel_p[tok][j];
    if (a.renorm) w = sum == 0.0f ? 0.0f : w / sum;
    a.index[t * k + j] = x;
    a.weights[t * k + j] = w * a.scale;
    atomicOr(&mask[x][tok >> 5], 1u << (tok & 31));
  }
  __syncthreads();
  if (a.hist) {
    for (int i = tid; i < e; i += NT) {
      uint8_t* h = a.hist + (int64_t)i * a.nbp;
      h[blockIdx.x] =
          (uint8_t)(__builtin_popcount(mask[i][0]) + __builtin_popcount(mask[i][1]));
      if (blockIdx.x == gridDim.x - 1)
        for (int b = gridDim.x; b < a.nbp; ++b) h[b] = 0;
    }
    return;
  }
  // one workgroup in all: the slot order at once
  for (int i = tid; i < e; i += NT)
    cnt[i] = __builtin_popcount(mask[i][0]) + __builtin_popcount(mask[i][1]);
  __syncthreads();
  scan_experts(cnt, e);
  for (int i = tid; i < e; i += NT) a.offs[i + 1] = cnt[i];
  if (tid == 0) a.offs[0] = 0;
  for (int j = l16; j < k; j += 16) {
    if (!live) break;
    const int x = sel_e[tok][j];
    const uint32_t m0 = mask[x][0], m1 = mask[x][1];
    const int all = __builtin_popcount(m0) + __builtin_popcount(m1);
    const uint32_t below = (1u << (tok & 31)) - 1u;
    const int rank = tok < 32 ? __builtin_popcount(m0 & below)
                              : __builtin_popcount(m0) + __builtin_popcount(m1 & below);
    const int64_t at = cnt[x] - all + rank;
    a.rows[at] = t;
    a.slots[t * k + j] = at;
  }
}

// prefix[x][b] = sum of hist[x][b'] over b' < b, a workgroup for each expert.
__global__ __launch_bounds__(1024) void route_scan_kernel(const uint8_t* __restrict__ hist,
                                                          int nbp, int32_t* __restrict__ prefix) {
  __shared__ int part[16];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const uint8_t* h = hist + (int64_t)blockIdx.x * nbp;
  int32_t* p = prefix + (int64_t)blockIdx.x * nbp;
  int before = 0;
  for (int b0 = 0; b0 < nbp; b0 += 1024) {
    const int b = b0 + threadIdx.x;
    const int own = b < nbp ? h[b] : 0;
    int v = own;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int o = __shfl_up(v, d);
      if (lane >= d) v += o;
    }
    if (lane == 63) part[w] = v;
    __syncthreads();
    int front = before, all = before;
    for (int i = 0; i < 16; ++i) {
      front += i < w ? part[i] : 0;
      all += part[i];
    }
    if (b < nbp) p[b] = front + v - own;
    before = all;
    __syncthreads();
  }
}

// The slot order of workgroup b's tokens, given every workgroup's counts.
__global__ __launch_bounds__(1024) void route_order_kernel(RouteArgs a, int nb, int rt) {
  __shared__ uint32_t mask[RE][2];
  __shared__ int cnt[RE];   // tokens per expert, then their running sum
  __shared__ int base[RE];  // tokens of earlier workgroups
  const int tid = threadIdx.x, tok = tid >> 4, l16 = tid & 15;
  const int b = blockIdx.x, e = a.e, k = a.k;
  const int64_t t = (int64_t)b * rt + tok;
  const bool live = tok < rt && t < a.t;
  for (int i = tid; i < e; i += 1024) {
    mask[i][0] = mask[i][1] = 0;
    cnt[i] = base[i] = 0;
  }
  __syncthreads();
  if (live)
    for (int j = l16; j < k; j += 16)
      atomicOr(&mask[(int)a.index[t * k + j]][tok >> 5], 1u << (tok & 31));
  if (a.prefix) {
    for (int x = tid; x < e; x += 1024) {
      const int64_t at = (int64_t)x * a.nbp;
      base[x] = a.prefix[at + b];
      cnt[x] = a.prefix[at + nb - 1] + a.hist[at + nb - 1];
    }
  } else {
    const int ep = e <= 64 ? 64 : (e <= 128 ? 128 : (e <= 256 ? 256 : 512));
    const int x = tid & (ep - 1), parts = 1024 / ep;
    if (x < e) {
      // 16 workgroups' counts a load, four a sum of bytes
      uint32_t all = 0, pre = 0;
      const u32x4* h = reinterpret_cast<const u32x4*>(a.hist + (int64_t)x * a.nbp);
      for (int i = tid / ep; i < a.nbp / 16; i += parts) {
        const u32x4 v = h[i];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int n = b - 16 * i - 4 * q;  // of these four, how many come before
          const uint32_t m = n <= 0 ? 0u : (n >= 4 ? ~0u : (1u << (8 * n)) - 1u);
          all = __builtin_amdgcn_sad_u8(v[q], 0u, all);
          pre = __builtin_amdgcn_sad_u8(v[q] & m, 0u, pre);
        }
      }
      atomicAdd(&cnt[x], (int)all);
      atomicAdd(&base[x], (int)pre);
    }
  }
  __syncthreads();
  scan_experts(cnt, e);
  if (b == 0) {
    for (int x = tid; x < e; x += 1024) a.offs[x + 1] = cnt[x];
    if (tid == 0) a.offs[0] = 0;
  }
  if (!live) return;
  for (int j = l16; j < k; j += 16) {
    const int x = (int)a.index[t * k + j];
    const uint32_t m0 = mask[x][0], m1 = mask[x][1];
    const uint32_t below = (1u << (tok & 31)) - 1u;
    const int rank = tok < 32 ? __builtin_popcount(m0 & below)
                              : __builtin_popcount(m0) + __builtin_popcount(m1 & below);
    const int64_t at = (int64_t)(x ? cnt[x - 1] : 0) + base[x] + rank;
    a.rows[at] = t;
    a.slots[t * k + j] = at;
  }
}

// The gradient: with dp the gradient at the scores (zero for experts not chosen),
//   weights = c p              dp_j = c g_j
//   weights = c p / S          dp_j = c (g_j - sum_i g_i p_i / S) / S
// and through the scores dl = dp p (1 - p) (sigmoid) or p (dp - sum dp p) (softmax; that sum
// is zero where the weights are renormalised, and not formed).
template <int EPL>
__global__ __launch_bounds__(256) void route_backward_kernel(
    const void* __restrict__ logits, int dtype, int64_t ld, int64_t n_tok, int e, int k,
    int scoring, int renorm, float scale, const int64_t* __restrict__ index,
    const float* __restrict__ grad, void* __restrict__ dlogits) {
  const int l16 = threadIdx.x & 15;
  const int64_t tt = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4);
  const bool live = tt < n_tok;
  const int64_t t = live ? tt : n_tok - 1;
  float v[EPL], p[EPL], d[EPL];
  bool chosen[EPL];
  __shared__ int64_t at[16][RK];
  __shared__ float up[16][RK];
  const int tok = threadIdx.x >> 4;
  for (int j = l16; j < k; j += 16) {
    at[tok][j] = index[t * k + j];
    up[tok][j] = grad[t * k + j];
  }
  token_scores<EPL>(logits, dtype, t * ld, e, scoring, l16, v, p);
  __syncthreads();
#pragma unroll
  for (int i = 0; i < EPL; ++i) {
    d[i] = 0.0f;
    chosen[i] = false;
  }
  for (int j = 0; j < k; ++j) {
    const int64_t x = at[tok][j];
    const float g = up[tok][j];
#pragma unroll
    for (int i = 0; i < EPL; ++i)
      if (x == 16 * i + l16) {
        d[i] += g;
        chosen[i] = true;
      }
  }
  double sp = 0.0, sgp = 0.0;
#pragma unroll
  for (int i = 0; i < EPL; ++i)
    if (chosen[i]) {
      sp += (double)p[i];
      sgp += (double)(d[i] * p[i]);
    }
  sp = row_sum(sp);
  sgp = row_sum(sgp);
  const float total = (float)sp;
  const float mean = total == 0.0f ? 0.0f : (float)(sgp / sp);
  const float dot = scale * (float)sgp;
#pragma unroll
  for (int i = 0; i < EPL; ++i) {
    float dp = 0.0f;
    if (chosen[i]) {
      if (renorm)
        dp = total == 0.0f ? 0.0f : scale * (d[i] - mean) / total;
      else
        dp = scale * d[i];
    }
    float dl;
    if (scoring == 1)
      dl = dp * p[i] * (1.0f - p[i]);
    else
      dl = p[i] * (renorm ? dp : dp - dot);
    const int x = 16 * i + l16;
    if (live && x < e) store_from_f32(dlogits, t * e + x, dtype, dl);
  }
}

// out[t] = residual[t] + sum_j w[t][j] y[slots[t][j]]: 64, 128 or 256 threads (tpt) on a
// token, 16 bytes of a row of y at a time, four rows in flight.  Bound by reading y once: 16384
// tokens of 8 rows of 2048 in fp16 157 us, 3.8 TB/s (one row in flight, in f32: 267).
template <int DT, int V>
struct Piece {  // V neighbouring values of y
  static constexpr int W = V == 1 ? 1 : V * (DT == 0 ? 4 : 2) / 4;
  uint32_t u[W];
  __device__ __forceinline__ void load(const void* p, int64_t at) {
    if constexpr (V == 1) {
      if constexpr (DT == 0)
        u[0] = static_cast<const uint32_t*>(p)[at];
      else
        u[0] = static_cast<const uint16_t*>(p)[at];
    } else {
      const u32x4 v = *reinterpret_cast<const u32x4*>(static_cast<const char*>(p) +
                                                      at * (DT == 0 ? 4 : 2));
#pragma unroll
      for (int i = 0; i < 4; ++i) u[i] = v[i];
    }
  }
  __device__ __forceinline__ float operator[](int i) const {
    if constexpr (DT == 0) return __uint_as_float(u[i]);
    const uint32_t h = V == 1 ? u[0] : u[i >> 1] >> (16 * (i & 1));
    if constexpr (DT == 1) return f16_from_bits((uint16_t)h);
    return __uint_as_float(h << 16);
  }
};

template <int DT, int V>
__global__ __launch_bounds__(256) void combine_kernel(
    const void* __restrict__ y, int64_t y_rows, int64_t n,
    const int64_t* __restrict__ slots, const float* __restrict__ weights, int64_t tokens, int k,
    int tpt, const void* __restrict__ residual, int dt_res, void* __restrict__ out, int dt_out) {
  const int at = __builtin_amdgcn_readfirstlane(threadIdx.x / tpt);
  const int64_t t = (int64_t)blockIdx.x * (256 / tpt) + at;
  if (t >= tokens) return;
  for (int64_t c = ((int64_t)blockIdx.y * tpt + (threadIdx.x - at * tpt)) * V; c < n;
       c += (int64_t)gridDim.y * tpt * V) {
    float acc[V];
#pragma unroll
    for (int i = 0; i < V; ++i)
      acc[i] = residual ? load_as_f32(residual, t * n + c + i, dt_res) : 0.0f;
    for (int j0 = 0; j0 < k; j0 += 4) {
      Piece<DT, V> p[4];
      float w[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int j = j0 + u < k ? j0 + u : k - 1;
        int64_t s = slots[t * k + j];
        w[u] = weights[t * k + j];
        if (s < 0 || s >= y_rows) {
          w[u] = __builtin_nanf("");
          s = 0;
        }
        if (y_rows) p[u].load(y, s * n + c);
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        if (j0 + u >= k) break;
#pragma unroll
        for (int i = 0; i < V; ++i)
          acc[i] = __builtin_fmaf(w[u], y_rows ? p[u][i] : 0.0f, acc[i]);
      }
    }
#pragma unroll
    for (int i = 0; i < V; ++i) store_from_f32(out, t * n + c + i, dt_out, acc[i]);
  }
}

// The same of SlotRows: two rows at a time go through LDS, from where columns are taken by
// their places, a pair of neighbours to a thread (and CH pairs tpt apart), so that a wave's reads
// meet on few banks: 16384 tokens of 8 rows of 2048 197 us (four rows at a time, which leave room
// for fewer waves, 232; combine_kernel, rows in their own order, 157; what the products' stores
// save is 390).
template <int CH>
__global__ __launch_bounds__(256) void combine_slots_kernel(
    SlotRows y, const int64_t* __restrict__ offs, int experts, int64_t y_rows,
    const int64_t* __restrict__ slots, const float* __restrict__ weights, int64_t tokens, int k,
    int tpt, const void* __restrict__ residual, int dt_res, void* __restrict__ out, int dt_out) {
  extern __shared__ __attribute__((aligned(16))) uint16_t rows16[];
  const int at = __builtin_amdgcn_readfirstlane(threadIdx.x / tpt), tid = threadIdx.x - at * tpt;
  const int64_t tt = (int64_t)blockIdx.x * (256 / tpt) + at;
  const bool live = tt < tokens;  // (all threads meet at the barriers)
  const int64_t t = live ? tt : tokens - 1;
  const int n = (int)y.n;
  constexpr int R = 2;
  uint16_t* rows = rows16 + at * R * (y.pitch + y.ep / 2);
  int8_t* ex = reinterpret_cast<int8_t*>(rows + R * y.pitch);  // their exponents
  const int share = tpt / R, ei = tid & (share - 1);  // of the threads, to a row's exponents
  float acc[CH][2];
#pragma unroll
  for (int h = 0; h < CH; ++h)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int c = 2 * (tid + h * tpt) + i;
      acc[h][i] = residual && c < n ? load_as_f32(residual, t * n + c, dt_res) : 0.0f;
    }
  constexpr int IT = CH == 4 ? 2 : 4;  // pieces of a row's slots a thread
  const int64_t ends = range_ends(offs, experts);
  for (int j0 = 0; j0 < k; j0 += R) {
    const uint32_t* places[R];
    float w[R], factor[R];
    u32x4 raw[R][IT];
    uint32_t exps = 0;  // four fragments'
    uint32_t p[CH][R];
#pragma unroll
    for (int u = 0; u < R; ++u) {
      const int j = j0 + u < k ? j0 + u : k - 1;
      int64_t s = slots[t * k + j];
      w[u] = weights[t * k + j];
      if (s < 0 || s >= y_rows) {
        w[u] = __builtin_nanf("");
        s = 0;
      }
      factor[u] = y.scale[s];
      places[u] = reinterpret_cast<const uint32_t*>(
          y.places + (int64_t)expert_of(ends, offs, experts, s) * n);
      const u32x4* from = reinterpret_cast<const u32x4*>(y.v + s * y.pitch);
#pragma unroll
      for (int i = 0; i < IT; ++i)
        if (tid + i * tpt < y.pitch / 8) raw[u][i] = from[tid + i * tpt];
    }
    if (4 * ei < y.ep) {
      const int j = j0 + tid / share;
      const int64_t s = slots[t * k + (j < k ? j : k - 1)];
      exps = reinterpret_cast<const uint32_t*>(y.exps +
                                               (s < 0 || s >= y_rows ? 0 : s) * y.ep)[ei];
    }
#pragma unroll
    for (int h = 0; h < CH; ++h)
#pragma unroll
      for (int u = 0; u < R; ++u)
        if (2 * (tid + h * tpt) < n) p[h][u] = places[u][tid + h * tpt];
#pragma unroll
    for (int u = 0; u < R; ++u)
#pragma unroll
      for (int i = 0; i < IT; ++i)
        if (tid + i * tpt < y.pitch / 8)
          reinterpret_cast<u32x4*>(rows + u * y.pitch)[tid + i * tpt] = raw[u][i];
    if (4 * ei < y.ep) reinterpret_cast<uint32_t*>(ex + tid / share * y.ep)[ei] = exps;
    __syncthreads();
#pragma unroll
    for (int h = 0; h < CH; ++h) {
      const int c = tid + h * tpt;
      if (2 * c >= n) break;
#pragma unroll
      for (int u = 0; u < R; ++u) {
        if (j0 + u >= k) break;
        const uint16_t* row = rows + u * y.pitch;
        const int8_t* by = ex + u * y.ep;
        const uint32_t a = p[h][u] & 0xffffu, b = p[h][u] >> 16;
        acc[h][0] = __builtin_fmaf(
            w[u], ldexpf(f16_from_bits(row[a]), by[a >> 4]) * factor[u], acc[h][0]);
        acc[h][1] = __builtin_fmaf(
            w[u], ldexpf(f16_from_bits(row[b]), by[b >> 4]) * factor[u], acc[h][1]);
      }
    }
    __syncthreads();
  }
  if (!live) return;
#pragma unroll
  for (int h = 0; h < CH; ++h) {
    const int c = tid + h * tpt;
    if (2 * c >= n) break;
    const int64_t o = t * n + 2 * c;  // (even)
    if (dt_out == 0)
      *reinterpret_cast<float2*>(static_cast<float*>(out) + o) = make_float2(acc[h][0], acc[h][1]);
    else
      *reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(out) + o) =
          dt_out == 1 ? (uint32_t)f16_bits(acc[h][0]) | (uint32_t)f16_bits(acc[h][1]) << 16
                      : (uint32_t)bf16_bits(acc[h][0]) | (uint32_t)bf16_bits(acc[h][1]) << 16;
  }
}

// The weighted sum's gradients, a wave on a slot (t, j): dw = sum_c g[t][c] y[slot][c], dy[slot]
// = w g[t].  Bound by reading y and writing dy once (g's rows are read by their k slots from
// cache).  A row of y that several slots name takes the sum of theirs: the wave of the first one
// looks for the others between it and the last (`named`), and adds them in their order.
template <int DT, int V>
__device__ __forceinline__ void load_values(const void* p, int64_t at, float (&v)[V]) {
  if constexpr (V == 1) {
    v[0] = load_as_f32(p, at, DT);
  } else if constexpr (DT == 0) {
    const f32x4v u = *reinterpret_cast<const f32x4v*>(static_cast<const float*>(p) + at);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = u[i];
  } else {
    const uint2 u = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p) + at);
    const uint32_t h[4] = {u.x & 0xffffu, u.x >> 16, u.y & 0xffffu, u.y >> 16};
#pragma unroll
    for (int i = 0; i < 4; ++i)
      v[i] = DT == 1 ? f16_from_bits((uint16_t)h[i]) : __uint_as_float(h[i] << 16);
  }
}

// named[row] = {last + 1, count - first} of the slots that name a row of y, from zeros.
__global__ void combine_named_kernel(const int64_t* __restrict__ slots, int64_t count,
                                     int64_t y_rows, uint2* named) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= count) return;
  const int64_t s = slots[i];
  if (s < 0 || s >= y_rows) return;
  atomicMax(&named[s].x, (uint32_t)(i + 1));
  atomicMax(&named[s].y, (uint32_t)(count - i));
}

template <int DG, int DT, int V>
__global__ __launch_bounds__(256) void combine_backward_kernel(
    const void* __restrict__ grad, const void* __restrict__ y, int64_t y_rows, int64_t n,
    const int64_t* __restrict__ slots, const float* __restrict__ weights, int64_t count, int k,
    float* __restrict__ dw, void* __restrict__ dy, const uint2* __restrict__ named) {
  const int64_t i = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  if (i >= count) return;
  const int64_t t = i / k, s = slots[i];
  if (s < 0 || s >= y_rows) {
    if (dw && lane == 0) dw[i] = __builtin_nanf("");
    return;
  }
  const float w = weights[i];
  float sum = 0.0f;
  int64_t first = i, last = i;
  if (dy) {
    last = (int64_t)named[s].x - 1;
    first = count - (int64_t)named[s].y;
  }
  for (int64_t c = lane * V; c < n; c += 64 * V) {
    float g[V], v[V];
    load_values<DG, V>(grad, t * n + c, g);
    if (dw) {
      load_values<DT, V>(y, s * n + c, v);
#pragma unroll
      for (int u = 0; u < V; ++u) sum = __builtin_fmaf(g[u], v[u], sum);
    }
    if (dy && first == last) {
#pragma unroll
      for (int u = 0; u < V; ++u) store_from_f32(dy, s * n + c + u, DT, w * g[u]);
    }
  }
  if (dy && i == first && first < last)
    for (int64_t c0 = 0; c0 < n; c0 += 64 * V) {  // (the whole wave)
      const int64_t c = c0 + lane * V;
      float g[V], acc[V];
#pragma unroll
      for (int u = 0; u < V; ++u) acc[u] = 0.0f;
      for (int64_t j0 = first; j0 <= last; j0 += 64) {
        unsigned long long more = __ballot(j0 + lane <= last && slots[j0 + lane] == s);
        for (; more; more &= more - 1) {
          const int64_t j = j0 + __builtin_ctzll(more);
          const float wj = weights[j];
          if (c < n) load_values<DG, V>(grad, j / k * n + c, g);
#pragma unroll
          for (int u = 0; u < V; ++u)
            if (c < n) acc[u] = __builtin_fmaf(wj, g[u], acc[u]);
        }
      }
#pragma unroll
      for (int u = 0; u < V; ++u)
        if (c < n) store_from_f32(dy, s * n + c + u, DT, acc[u]);
    }
#pragma unroll
  for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
  if (dw && lane == 0) dw[i] = sum;
}

int check_route(const char* what, const void* logits, int dtype, int64_t ld, int64_t t,
                int64_t e, int64_t k, int scoring) {
  HI2X_REQUIRE(dtype >= 0 && dtype <= 2, "%s: dtype %d", what, dtype);
  HI2X_REQUIRE(e >= 1 && e <= RE, "%s: %lld experts (1 to %d)", what, (long long)e, RE);
  HI2X_REQUIRE(k >= 1 && k <= RK && k <= e, "%s: %lld choices of %lld experts (at most %d)",
               what, (long long)k, (long long)e, RK);
  HI2X_REQUIRE(t >= 0 && t < (1ll << 31) / RK && ld >= e, "%s: bad shape", what);
  HI2X_REQUIRE(scoring == 0 || scoring == 1, "%s: scoring %d", what, scoring);
  HI2X_REQUIRE(logits || t == 0, "%s: null logits", what);
  return HI2X_OK;
}

// Tokens to a workgroup.  Four where that is all there are (barriers of one wave: one token
// of 64 experts 7.2 -> 5.6 us); up to the 64 that one launch orders (32 above 256 experts,
// whose registers leave room for half the waves) one workgroup; up to 4096 16, which spreads
// them over the CUs (4096 tokens of 256 experts in groups 20 -> 11.5 us); then 64 again.
int route_tokens(int64_t t, int64_t e) {
  const int most = e <= 256 ? 64 : 32;
  return t <= 4 ? 4 : (t <= most ? most : (t <= 4096 ? 16 : most));
}

// Clears offs where there are no tokens, and tables in front of their kernels.
__global__ void zero_i64_kernel(int64_t* p, int64_t n) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i < n) p[i] = 0;
}

}  // namespace

int launch_combine(const SlotRows& y, const int64_t* offs, int experts, int64_t y_rows,
                   const int64_t* slots, const float* weights, int64_t t, int64_t top_k,
                   const void* residual, int dt_residual, void* out, int dt_out, hipStream_t s) {
  const int64_t pieces = y.n / 8;  // (n is a multiple of 16)
  const int tpt = pieces <= 64 ? 64 : (pieces <= 128 ? 128 : 256), each = 256 / tpt;
  const dim3 grid((unsigned)((t + each - 1) / each));
  const size_t lds = (size_t)each * 2 * (y.pitch * 2 + y.ep);  // (at most 33 KiB)
  if (pieces <= 256)
    combine_slots_kernel<4><<<grid, 256, lds, s>>>(y, offs, experts, y_rows, slots, weights, t,
                                                   (int)top_k, tpt, residual, dt_residual, out,
                                                   dt_out);
  else
    combine_slots_kernel<16><<<grid, 256, lds, s>>>(y, offs, experts, y_rows, slots, weights, t,
                                                    (int)top_k, tpt, residual, dt_residual, out,
                                                    dt_out);
  return launch_status("moe_combine");
}

int launch_combine(const void* y, int dt_y, int64_t y_rows, int64_t n, const int64_t* slots,
                   const float* weights, int64_t t, int64_t top_k, const void* residual,
                   int dt_residual, void* out, int dt_out, hipStream_t s) {
  const int wide = dt_y == 0 ? 4 : 8;
  const int v = n % wide == 0 && (uintptr_t)y % 16 == 0 ? wide : 1;
  const int64_t pieces = n / v;
  const int tpt = pieces <= 64 ? 64 : (pieces <= 128 ? 128 : 256);
  const int64_t cols = (pieces + tpt - 1) / tpt;
  const dim3 grid((unsigned)((t + 256 / tpt - 1) / (256 / tpt)), (unsigned)(cols < 64 ? cols : 64));
#define HI2X_COMBINE(DT, V)                                                                    \
  combine_kernel<DT, V><<<grid, 256, 0, s>>>(y, y_rows, n, slots, weights, t, (int)top_k,      \
                                             tpt, residual, dt_residual, out, dt_out)
  if (dt_y == 0) {
    if (v == 4)
      HI2X_COMBINE(0, 4);
    else
      HI2X_COMBINE(0, 1);
  } else if (dt_y == 1) {
    if (v == 8)
      HI2X_COMBINE(1, 8);
    else
      HI2X_COMBINE(1, 1);
  } else {
    if (v == 8)
      HI2X_COMBINE(2, 8);
    else
      HI2X_COMBINE(2, 1);
  }
#undef HI2X_COMBINE
  return launch_status("moe_combine");
}

}  // namespace hi2x

using namespace hi2x;

extern "C" int64_t hi2x_route_workspace_bytes(int64_t t, int64_t e) {
  if (t < 0 || e < 1 || e > RE) return -1;
  const int64_t nb = (t + route_tokens(t, e) - 1) / route_tokens(t, e);
  if (nb <= 1) return 0;
  const int64_t nbp = (nb + 15) / 16 * 16;
  return align256(nbp * e) + (nb > SCAN_OVER ? nbp * e * 4 : 0);
}

extern "C" int hi2x_route(const void* logits, int dtype, int64_t ld, int64_t t, int64_t e,
                          int64_t top_k, int scoring, const float* bias, int64_t groups,
                          int64_t top_groups, int renormalise, float scale, int64_t* index,
                          float* weights, int64_t* rows, int64_t* offs, int64_t* slots, void* ws,
                          int64_t ws_bytes, void* stream) {
  clear_error();
  if (int rc = check_route("route", logits, dtype, ld, t, e, top_k, scoring)) return rc;
  HI2X_REQUIRE(groups >= 1 && groups <= RG && e % groups == 0,
               "route: %lld experts in %lld groups (equal ones, at most %d)", (long long)e,
               (long long)groups, RG);
  HI2X_REQUIRE(top_groups >= 1 && top_groups <= groups && top_k <= e / groups * top_groups,
               "route: %lld choices from %lld of %lld groups", (long long)top_k,
               (long long)top_groups, (long long)groups);
  HI2X_REQUIRE(offs && (t == 0 || (index && weights && rows && slots)), "route: null output");
  const hipStream_t s = as_stream(stream);
  if (t == 0) {
    zero_i64_kernel<<<dim3((unsigned)(e / 256 + 1)), 256, 0, s>>>(offs, e + 1);
    return launch_status("route");
  }
  const int rt = route_tokens(t, e);
  const int64_t nb = (t + rt - 1) / rt;
  Workspace w;
  const int64_t need = hi2x_route_workspace_bytes(t, e);
  if (int rc = take_workspace(w, ws, ws_bytes, (size_t)need, s, "route")) return rc;
  RouteArgs a{logits, dtype,  ld,      t,     (int)e, (int)top_k, scoring, bias,
              (int)groups, (int)top_groups, renormalise, scale, index, weights, rows, offs,
              slots, nullptr, nullptr, 0};
  if (nb > 1) {
    a.nbp = (int)((nb + 15) / 16 * 16);
    a.hist = reinterpret_cast<uint8_t*>(w.p);
    if (nb > SCAN_OVER)
      a.prefix = reinterpret_cast<int32_t*>(w.p + align256((int64_t)a.nbp * e));
  }
  const size_t dyn = top_groups < groups && !whole_rows(e / groups, groups)
                         ? (size_t)rt * (e + groups) * 4
                         : 0;
  const dim3 grid((unsigned)nb);
  // (each kernel's limit is its own largest, not this call's: threads share it)
#define HI2X_ROUTE_(EPL, NT)                                                                   \
  {                                                                                            \
    if (dyn > 32768)                                                                           \
      HI2X_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(route_kernel<EPL, NT>),       \
                                   hipFuncAttributeMaxDynamicSharedMemorySize,                 \
                                   NT / 16 * (16 * EPL + RG) * 4));                            \
    route_kernel<EPL, NT><<<grid, NT, dyn, s>>>(a);                                            \
  }
#define HI2X_ROUTE(EPL, MOST)                       \
  {                                                 \
    if (rt == 4)                                    \
      HI2X_ROUTE_(EPL, 64)                          \
    else if (rt == 16)                              \
      HI2X_ROUTE_(EPL, 256)                         \
    else                                            \
      HI2X_ROUTE_(EPL, MOST)                        \
  }
  if (e <= 64)
    HI2X_ROUTE(4, 1024)
  else if (e <= 128)
    HI2X_ROUTE(8, 1024)
  else if (e <= 256)
    HI2X_ROUTE(16, 1024)
  else
    HI2X_ROUTE(32, 512)
#undef HI2X_ROUTE_
#undef HI2X_ROUTE
  if (nb > 1) {
    if (a.prefix)
      route_scan_kernel<<<dim3((unsigned)e), 1024, 0, s>>>(a.hist, a.nbp, a.prefix);
    route_order_kernel<<<grid, 1024, 0, s>>>(a, (int)nb, rt);
  }
  return launch_status("route");
}

extern "C" int hi2x_route_backward(const void* logits, int dtype, int64_t ld, int64_t t,
                                   int64_t e, int64_t top_k, int scoring, int renormalise,
                                   float scale, const int64_t* index, const float* grad,
                                   void* dlogits, void* stream) {
  clear_error();
  if (int rc = check_route("route_backward", logits, dtype, ld, t, e, top_k, scoring)) return rc;
  if (t == 0) return HI2X_OK;
  HI2X_REQUIRE(index && grad && dlogits, "route_backward: null buffer");
  const hipStream_t s = as_stream(stream);
  const dim3 grid((unsigned)((t + 15) / 16));
#define HI2X_ROUTE(EPL)                                                                     \
  route_backward_kernel<EPL><<<grid, 256, 0, s>>>(logits, dtype, ld, t, (int)e, (int)top_k, \
                                                  scoring, renormalise, scale, index, grad, \
                                                  dlogits)
  if (e <= 64)
    HI2X_ROUTE(4);
  else if (e <= 128)
    HI2X_ROUTE(8);
  else if (e <= 256)
    HI2X_ROUTE(16);
  else
    HI2X_ROUTE(32);
#undef HI2X_ROUTE
  return launch_status("route_backward");
}

extern "C" int hi2x_moe_combine(const void* y, int dt_y, int64_t y_rows, int64_t n,
                                const int64_t* slots, const float* weights, int64_t t,
                                int64_t top_k, const void* residual, int dt_residual, void* out,
                                int dt_out, void* stream) {
  clear_error();
  for (int d : {dt_y, dt_residual, dt_out})
    HI2X_REQUIRE(d >= 0 && d <= 2, "moe_combine: dtype %d", d);
  HI2X_REQUIRE(t >= 0 && t < (1ll << 31) && n >= 1 && top_k >= 1 && top_k < (1 << 20) &&
                   y_rows >= 0,
               "moe_combine: bad shape");
  if (t == 0) return HI2X_OK;
  HI2X_REQUIRE((y || y_rows == 0) && slots && weights && out, "moe_combine: null buffer");
  return launch_combine(y, dt_y, y_rows, n, slots, weights, t, top_k, residual,
                        dt_residual, out, dt_out, as_stream(stream));
}

extern "C" int64_t hi2x_moe_combine_grad_workspace_bytes(int64_t y_rows) {
  return y_rows < 0 ? -1 : align256(y_rows * (int64_t)sizeof(uint2));
}

extern "C" int hi2x_moe_combine_backward(const void* grad, int dt_grad, const void* y, int dt_y,
                                         int64_t y_rows, int64_t n, const int64_t* slots,
                                         const float* weights, int64_t t, int64_t top_k,
                                         float* grad_weights, void* grad_y, void* stream) {
  return hi2x_moe_combine_grad(grad, dt_grad, y, dt_y, y_rows, n, slots, weights, t, top_k,
                               grad_weights, grad_y, nullptr, 0, stream);
}

extern "C" int hi2x_moe_combine_grad(const void* grad, int dt_grad, const void* y, int dt_y,
                                     int64_t y_rows, int64_t n, const int64_t* slots,
                                     const float* weights, int64_t t, int64_t top_k,
                                     float* grad_weights, void* grad_y, void* ws,
                                     int64_t ws_bytes, void* stream) {
  clear_error();
  for (int d : {dt_grad, dt_y})
    HI2X_REQUIRE(d >= 0 && d <= 2, "moe_combine_backward: dtype %d", d);
  HI2X_REQUIRE(y_rows >= 0 && y_rows < (1ll << 38) && n >= 0 && t >= 0 && t < (1ll << 31) && top_k >= 1 &&
                   top_k < (1 << 20) && t * top_k < (1ll << 32),
               "moe_combine_backward: bad shape");
  if (t == 0 || (!grad_weights && !grad_y)) return HI2X_OK;
  HI2X_REQUIRE((grad || n == 0) && (y || y_rows == 0 || n == 0) && slots && weights,
               "moe_combine_backward: null buffer");
  const int64_t count = t * top_k;
  const hipStream_t s = as_stream(stream);
  Workspace w;
  if (grad_y) {
    const size_t need = (size_t)hi2x_moe_combine_grad_workspace_bytes(y_rows);
    if (int rc = take_workspace(w, ws, ws_bytes, need, s, "moe_combine_backward")) return rc;
    if (y_rows > 0) {
      zero_i64_kernel<<<dim3((unsigned)(y_rows / 256 + 1)), 256, 0, s>>>(
          reinterpret_cast<int64_t*>(w.p), y_rows);
      combine_named_kernel<<<dim3((unsigned)((count + 255) / 256)), 256, 0, s>>>(
          slots, count, y_rows, reinterpret_cast<uint2*>(w.p));
    }
  }
  const uint2* named = reinterpret_cast<const uint2*>(w.p);
  const dim3 grid((unsigned)((count + 3) / 4));
  const bool vec = n % 4 == 0 &&
                   (((uintptr_t)grad | (uintptr_t)y | (uintptr_t)grad_y) & 15) == 0;
#define HI2X_BACK_(DG, DT, V)                                                              \
  combine_backward_kernel<DG, DT, V><<<grid, 256, 0, s>>>(grad, y, y_rows, n, slots, weights, \
                                                          count, (int)top_k, grad_weights, \
                                                          grad_y, named);
#define HI2X_BACK(DG)         \
  if (vec && dt_y == 0)       \
    HI2X_BACK_(DG, 0, 4)      \
  else if (vec && dt_y == 1)  \
    HI2X_BACK_(DG, 1, 4)      \
  else if (vec)               \
    HI2X_BACK_(DG, 2, 4)      \
  else if (dt_y == 0)         \
    HI2X_BACK_(DG, 0, 1)      \
  else if (dt_y == 1)         \
    HI2X_BACK_(DG, 1, 1)      \
  else                        \
    HI2X_BACK_(DG, 2, 1)
  if (dt_grad == 0) {
    HI2X_BACK(0)
  } else if (dt_grad == 1) {
    HI2X_BACK(1)
  } else {
    HI2X_BACK(2)
  }
#undef HI2X_BACK
#undef HI2X_BACK_
  return launch_status("moe_combine_backward");
}
