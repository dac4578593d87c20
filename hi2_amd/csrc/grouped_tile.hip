// Products grouped by expert in 16 bits: tiles of 256 x 256 or 128 x 128 results through LDS and
// the matrix units.
//
// An operand of a tile is T rows of the contraction's values.  Where these are neighbours in
// memory (x and w of the product, dy of the tokens' gradient) a stage of 32 of them is 64 bytes a
// row, and a lane reads its 8 as one piece; where they are a row apart (w of the tokens'
// gradient, dy and x of the weights') a stage is 32 rows of T values, and LDS's transposing read
// hands a lane its column.  Both are loaded as they lie, 16 bytes a lane, straight into LDS.
//
// A wave holds T/2 x T/2 results in registers; a ring of four stages (or two) is in flight.  64 experts
// of 1024 x 2048, 2048 slots each in bfloat16: 533 us (1032 TFLOP/s), the tokens' gradient 570 (965;
// of tokens with eight slots each 825 with its float32 rows and their sums), the weights' 478 (1150); one
// library product of the size reaches 1298, 1080 and 625.
#include <type_traits>

#include "grouped.h"

namespace hi2x {
namespace {

typedef __bf16 b16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x8 __attribute__((ext_vector_type(8)));
typedef float f32x16v __attribute__((ext_vector_type(16)));

// Offsets past every resource: a row's, a piece's, and their sum.
constexpr uint32_t ROW_DEAD = 0x80000000u, PIECE_DEAD = GROUPED_SPAN;

// 64 lanes x 16 bytes from memory into LDS at byte `la` (+ 16 lane), in inline assembly so that the
// compiler does not wait for it before every later LDS read.  One wait state lies between the
// write of M0 and the load.
__device__ __forceinline__ void lds_load16(__amdgpu_buffer_rsrc_t rs, uint32_t voff, uint32_t la) {
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
               :
               : "s"(la), "v"(voff), "s"(rs)
               : "m0");
#pragma clang diagnostic pop
}

__device__ __forceinline__ int64_t uniform(int64_t v) {
  const uint32_t lo = __builtin_amdgcn_readfirstlane((int)(uint32_t)v);
  const uint32_t hi = __builtin_amdgcn_readfirstlane((int)(uint32_t)((uint64_t)v >> 32));
  return (int64_t)((uint64_t)hi << 32 | lo);
}

constexpr int wait_for(int vm, int lgkm) {
  return (vm & 15) | ((vm >> 4) << 14) | (7 << 4) | (lgkm << 8);
}

// LDS accesses stay on their side.
__device__ __forceinline__ void meet() {
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
  __builtin_amdgcn_s_barrier();
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
}

template <int DT>
__device__ __forceinline__ f32x16v product(const s16x8& a, const s16x8& b, const f32x16v& c) {
  if constexpr (DT == 1)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h16x8, a),
                                                  __builtin_bit_cast(h16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b16x8, a),
                                                   __builtin_bit_cast(b16x8, b), c, 0, 0, 0);
}

// A row's last piece counts whole: what lies in its 16 bytes behind the row is zero (along the
// contraction) or comes out in columns that are not stored.
__device__ __forceinline__ int whole(int n) { return (n + 7) & ~7; }

constexpr int STAGE = 32;  // of the contraction

// Neighbours of the contraction are neighbours in memory.  LDS: T rows of four 16-byte pieces,
// piece q of row r at q ^ ((r / 4) % 4), so that the 16 rows that a read of one piece touches at
// a time lie on different banks.
template <int T>
struct AlongOperand {
  static constexpr bool PAIRED = true;
  static constexpr int NC = T / 64;  // a wave's loads of a stage, 16 rows each
  __amdgpu_buffer_rsrc_t rs;
  uint32_t row[NC];  // this lane's rows' offsets
  uint32_t piece;    // its piece's, behind `from`
  int len;           // end of the contraction
  uint32_t at;       // LDS byte of the wave's first load
  uint32_t read0, read1;
  __device__ __forceinline__ void init(uint32_t lds, int wv, int first, int from, int end) {
    const int lane = threadIdx.x & 63;
    len = end;
    piece = from + 8 * ((lane & 3) ^ ((lane >> 4) & 3));
    at = lds + NC * wv * 1024;
    const uint32_t r = first + (lane & 31);
    const int h = lane >> 5, x = (lane >> 2) & 3;
    read0 = r * 64 + 16 * (h ^ x);
    read1 = r * 64 + 16 * ((2 + h) ^ x);
  }
  // row of load i that this lane brings
  static __device__ __forceinline__ int row_of(int wv, int i) {
    return 16 * (NC * wv + i) + ((threadIdx.x & 63) >> 2);
  }
  struct Stage {
    uint32_t k;
  };
  __device__ __forceinline__ Stage begin(int st) const {
    const uint32_t c = (uint32_t)st * STAGE + piece;
    return Stage{c < (uint32_t)len ? 2 * c : PIECE_DEAD};
  }
  __device__ __forceinline__ void load(const Stage& s, int i, uint32_t buffer) const {
    lds_load16(rs, row[i] + s.k, at + buffer + i * 1024);
  }
  // fragment t of 16 of the stage's 32
  __device__ __forceinline__ s16x8 read(const char* from, int step, int t) const {
    return *reinterpret_cast<const s16x8*>(from + (step ? read1 : read0) + t * 2048);
  }
};

// Neighbours of the contraction are a row apart.  LDS: 32 rows of T / 8 pieces, piece p of row r
// at p ^ (4 (r % 4)): a transposing read's 16 lanes take 4 rows x 32 bytes, and the four rows
// lie on different banks.
template <int T>
struct AcrossOperand {
  static constexpr bool PAIRED = false;
  static constexpr int NC = T / 64, LP = T / 8, RPC = 64 / LP;  // lanes a row, rows a load
  const char* base;
  int64_t pitch;     // bytes
  int64_t rows;      // of the contraction
  uint32_t last;     // bytes of a row that count
  uint32_t own[NC];  // this lane's offsets within a stage
  uint32_t at;
  uint32_t read_at[NC];
  __device__ __forceinline__ void init(uint32_t lds, int wv, int first, int cols) {
    const int lane = threadIdx.x & 63;
    at = lds + NC * wv * 1024;
    last = 2 * whole(cols);
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int r = RPC * (NC * wv + i) + lane / LP;
      const int p = (lane % LP) ^ (4 * (r & 3));
      own[i] = 8 * p < cols ? (uint32_t)(r * pitch) + 16 * p : PIECE_DEAD;
    }
    const int s = lane & 15, g = lane >> 4;
#pragma unroll
    for (int t = 0; t < NC; ++t)
      read_at[t] = (8 * (g >> 1) + (s >> 2)) * (2 * T) + 8 * (s & 1) +
                   16 * (((first / 8 + 4 * t) ^ (4 * (s >> 2))) + 2 * (g & 1) +
                         ((s & 3) >> 1));
  }
  struct Stage {
    __amdgpu_buffer_rsrc_t rs;
  };
  __device__ __forceinline__ Stage begin(int st) const {
    // (scalar instructions by hand: the compiler clamps in a vector register, and the load would
    // have to wait for what comes out of it)
    int left = (int)rows - st * STAGE, bytes;
    asm("s_min_i32 %0, %1, 32" : "=s"(left) : "s"(left) : "scc");
    static_assert(STAGE == 32, "above");
    bytes = __builtin_amdgcn_readfirstlane(left) * (int)pitch - ((int)pitch - (int)last);
    asm("s_max_i32 %0, %1, 0"
        : "=s"(bytes)
        : "s"(__builtin_amdgcn_readfirstlane(bytes))
        : "scc");
    return Stage{__builtin_amdgcn_make_buffer_rsrc(
        reinterpret_cast<char*>(uniform((int64_t)(base + (int64_t)st * (STAGE * pitch)))),
        (short)0, bytes, 0x00020000)};
  }
  __device__ __forceinline__ void load(const Stage& s, int i, uint32_t buffer) const {
    lds_load16(s.rs, own[i], at + buffer + i * 1024);
  }
  __device__ __forceinline__ s16x8 read(const char* from, int step, int t) const {
    const char* p = from + read_at[t] + step * (16 * 2 * T);
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (__attribute__((address_space(3))) s16x4*)(p));
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (__attribute__((address_space(3))) s16x4*)(p + 4 * 2 * T));
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  }
};

// The same of rows that an index names: their offsets in x lie in LDS, dead ones behind the last.
template <int T>
struct IndexedOperand : AcrossOperand<T> {
  using Base = AcrossOperand<T>;
  using Base::LP, Base::NC, Base::RPC;
  const uint32_t* table;  // in LDS
  __amdgpu_buffer_rsrc_t all;
  int lane_row;  // of the wave's first load
  __device__ __forceinline__ void init(uint32_t lds, int wv, int first, int cols) {
    this->pitch = 0;
    Base::init(lds, wv, first, cols);
    lane_row = RPC * NC * wv + (threadIdx.x & 63) / LP;
  }
  struct Stage {
    uint32_t row[NC];
  };
  __device__ __forceinline__ Stage begin(int st) const {
    Stage s;
#pragma unroll
    for (int i = 0; i < NC; ++i) s.row[i] = table[st * STAGE + lane_row + RPC * i];
    return s;
  }
  __device__ __forceinline__ void load(const Stage& s, int i, uint32_t buffer) const {
    lds_load16(all, s.row[i] + this->own[i], this->at + buffer + i * 1024);
  }
};

template <bool NEEDED, class O>
__device__ __forceinline__ auto pair_stage(O& o, int st) {
  if constexpr (NEEDED)
    return o.begin(st);
  else
    return 0;
}

// acc += A B^T over `len` > 0 of the contraction.  Each accumulator has results' columns (B's rows)
// in its registers and their rows (A's) over the lanes.
//
// A ring of four stages, or of two where more workgroups to a CU hide what it does not.  The two
// stages of a 128-byte line of an AlongOperand are asked for one right after the other, every other
// stage: a stage apart, the second comes when the line has left the CU's cache, and every line
// crosses from L2 twice (16384 x 4096 x 4096: 6.7e7 requests and 536 us; so half as many and 461, by
// now 440).
// Loads are issued behind products of the stage whose place they take, and always as many (what lies
// past the end reads as zeros), so that "landed" is a count.
template <int DT, int T, int RING, int MA, int MB, class A, class B>
__device__ __forceinline__ void tile_loop(A& a, B& b, const char* lds, int len,
                                          f32x16v (&acc)[T / 64][T / 64]) {
  constexpr int NA = T / 64, BYTES = T * 64;  // of an operand's stage
  constexpr bool PA = A::PAIRED, PB = B::PAIRED;
  static_assert(RING == 4 || (RING == 2 && !PA && !PB), "pairs need four stages");
  const int nst = (len + STAGE - 1) / STAGE;
  const char* la = lds;
  const char* lb = lds + RING * BYTES;
  // The loads of stages s0 (into x0) and s0 + 1 (into x1): those of paired operands, line by line,
  // in front of the others'.
  auto both = [&](int s0, uint32_t x0, uint32_t x1) {
    const auto a0 = a.begin(s0);
    const auto a1 = a.begin(s0 + 1);
    const auto b0 = b.begin(s0);
    const auto b1 = b.begin(s0 + 1);
    if constexpr (PA) {
#pragma unroll
      for (int i = 0; i < NA; ++i) a.load(a0, i, x0), a.load(a1, i, x1);
    }
    if constexpr (PB) {
#pragma unroll
      for (int i = 0; i < NA; ++i) b.load(b0, i, x0), b.load(b1, i, x1);
    }
#pragma unroll
    for (int i = 0; i < NA; ++i) {
      if constexpr (!PA) a.load(a0, i, x0);
      if constexpr (!PB) b.load(b0, i, x0);
    }
#pragma unroll
    for (int i = 0; i < NA; ++i) {
      if constexpr (!PA) a.load(a1, i, x1);
      if constexpr (!PB) b.load(b1, i, x1);
    }
  };
  both(0, 0, BYTES);
  if constexpr (RING == 4) both(2, 2 * BYTES, 3 * BYTES);
  // stage 0 landed, and with a ring of four stage 1
  __builtin_amdgcn_s_waitcnt(wait_for(RING == 4 ? 4 * NA : 2 * NA, 15));
  meet();
  s16x8 a0[MA], b0[MB], a1[MA], b1[MB];
  // Read r of a step's fragments, those of B first.
  auto fragment = [&](auto number, s16x8(&av)[MA], s16x8(&bv)[MB], uint32_t buffer, int step) {
    constexpr int r = decltype(number)::value;
    if constexpr (r < MB)
      bv[r] = b.read(lb + buffer, step, r);
    else if constexpr (r < MA + MB)
      av[r - MB] = a.read(la + buffer, step, r - MB);
  };
  auto fragments = [&](auto self, auto number) {
    constexpr int r = decltype(number)::value;
    if constexpr (r < MA + MB) {
      fragment(number, a0, b0, 0, 0);
      self(self, std::integral_constant<int, r + 1>{});
    }
  };
  fragments(fragments, std::integral_constant<int, 0>{});
  // Stage st in `cur`.  ODD: st is, and paired operands' stages st + 3 (into `prv`, where st - 1
  // was) and st + 4 are asked for.
  auto stage = [&](auto odd, int st, uint32_t prv, uint32_t cur, uint32_t nxt) {
    constexpr bool ODD = decltype(odd)::value;
    constexpr int PAIR = ODD ? 2 : 0;
    constexpr int LA = NA * (PA ? PAIR : 1), LB = NA * (PB ? PAIR : 1), ALL = LA + LB;
    // newer loads than the next stage's
    constexpr int NEWER = RING == 2 ? 0 : NA * (!ODD ? 4 : (PA ? 0 : 2) + (PB ? 0 : 2));
    const auto sa = a.begin(st + RING);
    const auto sb = b.begin(st + RING);
    const auto pa = pair_stage<PA && ODD>(a, st + RING - 1);
    const auto pb = pair_stage<PB && ODD>(b, st + RING - 1);
    __builtin_amdgcn_sched_barrier(0);
    // (a read behind each product: the matrix unit would wait for eight in a row; 131072 slots of 64
    // experts of 1024 x 2048 550 us, so 533, the weights' gradient 517 and 485)
    auto first = [&](auto self, auto number) {
      constexpr int m = decltype(number)::value;
      if constexpr (m < MA * MB) {
        acc[m / MB][m % MB] = product<DT>(b0[m % MB], a0[m / MB], acc[m / MB][m % MB]);
        static_assert(MA + MB <= MA * MB, "a product to each read");
        fragment(number, a1, b1, cur, 1);
        __builtin_amdgcn_sched_barrier(0);
        self(self, std::integral_constant<int, m + 1>{});
      }
    };
    first(first, std::integral_constant<int, 0>{});
    // this wave has read stage st, and stage st + 1 has landed; behind the barrier nobody reads
    // stage st any more
    __builtin_amdgcn_s_waitcnt(wait_for(NEWER, 0));
    meet();
    auto one = [&](auto number, const auto& pa, const auto& pb) {
      constexpr int l = decltype(number)::value;
      if constexpr (PA && l < LA) {
        if constexpr (l & 1)
          a.load(sa, l >> 1, cur);
        else
          a.load(pa, l >> 1, prv);
      } else if constexpr (PB && l - (PA ? LA : 0) < LB) {
        constexpr int m = l - (PA ? LA : 0);
        if constexpr (m & 1)
          b.load(sb, m >> 1, cur);
        else
          b.load(pb, m >> 1, prv);
      } else if constexpr (PA) {
        b.load(sb, l - LA, cur);
      } else if constexpr (PB) {
        a.load(sa, l - LB, cur);
      } else {
        if constexpr (l & 1)
          b.load(sb, l >> 1, cur);
        else
          a.load(sa, l >> 1, cur);
      }
    };
    auto products = [&](auto self, auto number, auto done) {
      constexpr int m = decltype(number)::value, d = decltype(done)::value;
      if constexpr (m < MA * MB) {
        acc[m / MB][m % MB] = product<DT>(b1[m % MB], a1[m / MB], acc[m / MB][m % MB]);
        fragment(number, a0, b0, nxt, 0);
        __builtin_amdgcn_sched_barrier(0);
        constexpr int upto = ALL * (m + 1) / (MA * MB);
        if constexpr (upto > d) {
          one(std::integral_constant<int, d>{}, pa, pb);
          if constexpr (upto > d + 1) one(std::integral_constant<int, d + 1>{}, pa, pb);
          __builtin_amdgcn_sched_barrier(0);
        }
        self(self, std::integral_constant<int, m + 1>{}, std::integral_constant<int, upto>{});
      }
    };
    products(products, std::integral_constant<int, 0>{}, std::integral_constant<int, 0>{});
    __builtin_amdgcn_sched_barrier(0);
  };
  int st = 0;
  uint32_t cur = 0;
  do {
    const uint32_t other = RING == 2 ? 0 : cur ^ (2 * BYTES);
    stage(std::false_type{}, st, 0, cur, cur + BYTES);
    stage(std::true_type{}, st + 1, cur, cur + BYTES, other);
    cur = other;
    st += 2;
  } while (st < nst);
  __builtin_amdgcn_s_waitcnt(wait_for(0, 0));
}

// The tile through LDS to rows of `out`, 16 bytes a lane where the rows allow it.  NAN_BY: rows
// whose flag in `bad` is set become NaN (1), or all of them by the first flag (2).
template <int DT, int T, int NAN_BY, int MB = T / 64>
__device__ __forceinline__ void store_tile(char* lds, f32x16v (&acc)[T / 64][T / 64],
                                           uint16_t* out, int64_t cols, int rows, int width,
                                           const uint8_t* bad, bool past) {
  constexpr int NA = T / 64, PITCH = 2 * T + 16;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int wr = wave >> 1, wc = wave & 1;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < NA; ++i)
#pragma unroll
    for (int j = 0; j < MB; ++j) {
      // (held where the matrix units write until its turn: all at once they would not fit)
      if constexpr (T == 256) asm volatile("" : "+a"(acc[i][j]));
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        uint32_t w[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const float x = acc[i][j][4 * q + 2 * u], y = acc[i][j][4 * q + 2 * u + 1];
          w[u] = DT == 1 ? (uint32_t)f16_bits(x) | (uint32_t)f16_bits(y) << 16
                         : (uint32_t)bf16_bits(x) | (uint32_t)bf16_bits(y) << 16;
        }
        const int r = (MB == NA ? wr * (T / 2) : 0) + 32 * i + (lane & 31);
        const int c = (MB == NA ? wc * (T / 2) : wave * (T / 4)) + 32 * j + 8 * q + 4 * (lane >> 5);
        *reinterpret_cast<uint2*>(lds + r * PITCH + 2 * c) = make_uint2(w[0], w[1]);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  __syncthreads();
  constexpr int LP = T / 8;
  const uint32_t nan = DT == 1 ? 0x7e007e00u : 0x7fc07fc0u;
  const bool wide = cols % 8 == 0 && ((uintptr_t)out & 15) == 0;
  const int c = 8 * (tid % LP);
  if (c >= width) return;
  // (two loops: of two stores at one place the compiler makes one, which is not past the caches)
  auto store = [&](auto stream) {
#pragma unroll 4
    for (int r = tid / LP; r < rows; r += 256 / LP) {
      u32x4 v = *reinterpret_cast<const u32x4*>(lds + r * PITCH + 2 * c);
      if (NAN_BY && bad[NAN_BY == 2 ? 0 : r]) v = u32x4{nan, nan, nan, nan};
      uint16_t* to = out + r * cols + c;
      if (wide && c + 8 <= width) {
        if constexpr (decltype(stream)::value)
          __builtin_nontemporal_store(v, reinterpret_cast<u32x4*>(to));
        else
          *reinterpret_cast<u32x4*>(to) = v;
      } else {
#pragma unroll
        for (int u = 0; u < 8; ++u)
          if (c + u < width) to[u] = (uint16_t)(v[u / 2] >> (16 * (u & 1)));
      }
    }
  };
  if (past)
    store(std::true_type{});
  else
    store(std::false_type{});
}

// The tile's sums as they are, to float32 rows of `out`, half of its rows through LDS at a time; 16 bytes a
// lane where the rows allow it.  Twice the bytes of store_tile's (131072 slots of 64 experts of 1024 x 2048
// 617 us for 570).
template <int T, int MB = T / 64>
__device__ __forceinline__ void store_sums(char* lds, f32x16v (&acc)[T / 64][T / 64], float* out,
                                           int64_t cols, int rows, int width, bool past) {
  constexpr int NA = T / 64, PITCH = 4 * T + 16, LP = T / 4;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int wr = wave >> 1, wc = wave & 1;
  const bool wide = cols % 4 == 0 && ((uintptr_t)out & 15) == 0;
  const int c = 4 * (tid % LP);
  for (int half = 0; half < (MB == NA ? 2 : 1); ++half) {
    __syncthreads();  // what was in LDS has been read
    if (MB != NA || wr == half) {
#pragma unroll
      for (int i = 0; i < NA; ++i)
#pragma unroll
        for (int j = 0; j < MB; ++j) {
          if constexpr (T == 256) asm volatile("" : "+a"(acc[i][j]));  // (as in store_tile)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int r = 32 * i + (lane & 31);
            const int at = (MB == NA ? wc * (T / 2) : wave * (T / 4)) + 32 * j + 8 * q +
                           4 * (lane >> 5);
            *reinterpret_cast<f32x4v*>(lds + r * PITCH + 4 * at) =
                f32x4v{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2],
                       acc[i][j][4 * q + 3]};
            __builtin_amdgcn_sched_barrier(0);
          }
        }
    }
    __syncthreads();
    const int live = rows - half * (T / 2) < T / 2 ? rows - half * (T / 2) : T / 2;
    if (c >= width) continue;
    auto store = [&](auto stream) {
#pragma unroll 4
      for (int r = tid / LP; r < live; r += 256 / LP) {
        const f32x4v v = *reinterpret_cast<const f32x4v*>(lds + r * PITCH + 4 * c);
        float* to = out + (half * (T / 2) + r) * cols + c;
        if (wide && c + 4 <= width) {
          if constexpr (decltype(stream)::value)
            __builtin_nontemporal_store(v, reinterpret_cast<f32x4v*>(to));
          else
            *reinterpret_cast<f32x4v*>(to) = v;
        } else {
#pragma unroll
          for (int u = 0; u < 4; ++u)
            if (c + u < width) to[u] = v[u];
        }
      }
    };
    if (past)
      store(std::true_type{});
    else
      store(std::false_type{});
  }
}

// Zeros where there is nothing to sum.
template <int T, class V>
__device__ __forceinline__ void store_zeros(V* out, int64_t cols, int rows, int width) {
  constexpr int TX = T < 256 ? T : 256;
  const int c = threadIdx.x % TX;
  if (c >= width) return;
  for (int r = threadIdx.x / TX; r < rows; r += 256 / TX) out[r * cols + c] = 0;
}

template <int T, int RING>
constexpr int LDS_BYTES = 2 * RING * T * 64 > T * (2 * T + 16) ? 2 * RING * T * 64
                                                               : T * (2 * T + 16);

// Slots whose rows' offsets are in LDS at a time, and offsets behind them that the ring reads.
template <int T, int RING>
constexpr int SEGMENT = T == 256 ? 4096 : (RING == 4 ? 2048 : 1024);
constexpr int BEHIND = 224;

// The plan's row tiles.  One workgroup: the ranges' first tiles by a scan, then a thread to a tile.
// (Found by every workgroup for itself, a tile's expert cost 2 us, and nobody knew how many tiles
// there are.)
constexpr int MOST_EXPERTS = 7000;
__global__ __launch_bounds__(1024) void grouped_plan_kernel(GroupedArgs g, int T, Plan* plan,
                                                            int64_t most) {
  __shared__ int first_tile[MOST_EXPERTS + 3];
  __shared__ int sums[16];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int experts = (int)g.experts, ranges = experts + 2;
  auto range = [&](int e, int64_t& a, int64_t& b) {
    auto clamp = [&](int64_t v) { return v < 0 ? 0 : (v > g.slots ? g.slots : v); };
    if (e < experts) {
      slot_range(g, e, a, b);
    } else {
      a = e == experts ? clamp(g.offs[experts]) : 0;
      b = e == experts ? g.slots : clamp(g.offs[0]);
    }
  };
  int64_t before = 0;  // (ranges that overlap, as they should not, can make very many)
  for (int e0 = 0; e0 < ranges; e0 += 1024) {
    const int e = e0 + tid;
    int64_t a = 0, b = 0;
    if (e < ranges) range(e, a, b);
    const int n = (int)((b - a + T - 1) / T);
    int inc = n;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int o = __shfl_up(inc, d);
      if (lane >= d) inc += o;
    }
    if (lane == 63) sums[wave] = inc;
    __syncthreads();
    int64_t base = before, all = 0;
    for (int w = 0; w < 16; ++w) {
      if (w < wave) base += sums[w];
      all += sums[w];
    }
    base += inc - n;
    if (e < ranges) first_tile[e] = base < most ? (int)base : (int)most;
    before += all;
    __syncthreads();
  }
  const int count = (int)(before < most ? before : most);
  if (tid == 0) {
    first_tile[ranges] = count;
    plan->count = count;
  }
  __syncthreads();
  for (int y = tid; y < count; y += 1024) {
    int lo = 0, hi = ranges - 1;  // the last range whose first tile is y or before
    while (lo < hi) {
      const int mid = (lo + hi + 1) / 2;
      if (first_tile[mid] <= y)
        lo = mid;
      else
        hi = mid - 1;
    }
    int64_t a, b;
    range(lo, a, b);
    const int64_t at = a + (int64_t)(y - first_tile[lo]) * T, left = b - at;
    plan->tile[y] = RowTile{at, (int32_t)(left < T ? left : T), lo < experts ? lo : -1};
  }
}

// A tile's sums (+ add) to `part`, a tile after a tile, as the accumulators hold them.
template <int T>
__device__ __forceinline__ void store_part(float* part, uint64_t tile,
                                           const f32x16v (&acc)[T / 64][T / 64], float add) {
  f32x4v* to = reinterpret_cast<f32x4v*>(part) + tile * (T * T / 4) + (threadIdx.x >> 6) * (T * T / 16) +
               (threadIdx.x & 63);
#pragma unroll
  for (int i = 0; i < T / 64; ++i)
#pragma unroll
    for (int j = 0; j < T / 64; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q, to += 64)
        *to = f32x4v{acc[i][j][4 * q] + add, acc[i][j][4 * q + 1] + add,
                     acc[i][j][4 * q + 2] + add, acc[i][j][4 * q + 3] + add};
}

// SPLIT: a tile's contraction is cut into `splits` ranges, of `per` stages (of the
// weights' gradient: of as many as its expert's slots need), and grouped_join_kernel adds their sums.
template <int DT, int WHAT, int T, int RING, bool INDEXED, bool SPLIT>
__global__ __launch_bounds__(256, T == 256 ? 1 : 8 / RING) void grouped_tile_kernel(
    GroupedArgs g, uint32_t nx, uint32_t ny, const void* plan, float* part, int splits, int per) {
  constexpr int NA = T / 64, BYTES = T * 64;
  __shared__ __attribute__((aligned(1024))) char lds[LDS_BYTES<T, RING>];
  __shared__ uint8_t bad[T];
  constexpr bool TABLE = WHAT == GROUPED_GRAD_W && INDEXED;
  __shared__ uint32_t table[TABLE ? SEGMENT<T, RING> + BEHIND : 1];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wr = wv >> 1, wc = wv & 1;
  const uint32_t base = __builtin_amdgcn_readfirstlane(
      (uint32_t)(size_t)(__attribute__((address_space(3))) char*)lds);
  const int n = (int)g.n, k = (int)g.k;
  f32x16v acc[NA][NA];
#pragma unroll
  for (int i = 0; i < NA; ++i)
#pragma unroll
    for (int j = 0; j < NA; ++j)
#pragma unroll
      for (int u = 0; u < 16; ++u) acc[i][j][u] = 0.0f;
  uint16_t* const out = static_cast<uint16_t*>(g.out);
  if constexpr (WHAT == GROUPED_GRAD_W) {
    // An expert's tiles over all XCDs, 2 x 4 of them at a time, one to each.
    const uint32_t xcd = blockIdx.x & 7, j = blockIdx.x >> 3;
    const uint32_t hx = nx / 4, tiles = hx * (ny / 2);  // (nx, ny: rounded up to whole rounds)
    // (what comes out of a division is in a vector register, and would keep what follows there)
    const uint32_t ez = __builtin_amdgcn_readfirstlane(j / tiles);
    const int e = SPLIT ? __builtin_amdgcn_readfirstlane(ez / splits) : ez;
    const uint32_t sub = j - ez * tiles, my = (xcd + ez) & 7;
    const uint32_t sy = __builtin_amdgcn_readfirstlane(sub / hx), sx = sub - sy * hx;
    const int64_t r0 = (int64_t)(sy * 2 + (my >> 2)) * T;
    const int64_t c0 = (int64_t)(sx * 4 + (my & 3)) * T;
    if (r0 >= n || c0 >= k) return;
    int64_t first, end;
    slot_range(g, e, first, end);
    first = uniform(first);
    end = uniform(end);
    const int rows = (int)(n - r0 < T ? n - r0 : T), cols = (int)(k - c0 < T ? k - c0 : T);
    uint16_t* const to = out + ((int64_t)e * n + r0) * k + c0;
    const uint32_t z = SPLIT ? ez - e * splits : 0;
    if (first == end) {
      if (z == 0) store_zeros<T>(to, k, rows, cols);
      return;
    }
    if (SPLIT) {  // a range of whole stages, which may hold nothing
      const uint32_t len = (uint32_t)(end - first);
      const int64_t by = __builtin_amdgcn_readfirstlane((len + splits - 1) / splits + STAGE - 1) &
                         ~(STAGE - 1);
      const int64_t at = first + z * by;
      first = at < end ? at : end;
      end = at + by < end ? at + by : end;
    }
    AcrossOperand<T> a;
    a.base = static_cast<const char*>(g.dy) + (first * g.ldy + r0) * 2;
    a.pitch = g.ldy * 2;
    a.rows = end - first;
    a.init(base, wv, wr * (T / 2), rows);
    if constexpr (INDEXED) {
      if (tid == 0) bad[0] = 0;
      IndexedOperand<T> b;
      b.table = table;
      b.all = rsrc(static_cast<const char*>(g.x) + c0 * 2,
                   g.x_rows > 0 ? ((g.x_rows - 1) * g.ldx + whole(cols)) * 2 : 0);
      b.init(base + RING * BYTES, wv, wc * (T / 2), cols);
      constexpr int SEG = SEGMENT<T, RING>;
      const int all = (int)(end - first);
      const int64_t* const index = g.rows + first;
      for (int at = 0; at < all; at += SEG) {
        const int len = all - at < SEG ? all - at : SEG;
        __syncthreads();  // the segment before has been read
        for (int u = tid; u < SEG + BEHIND; u += 256) {
          uint32_t off = ROW_DEAD;
          if (u < len) {
            const uint64_t r = (uint64_t)index[at + u];
            if (r < (uint64_t)g.x_rows)
              off = (uint32_t)r * (uint32_t)(g.ldx * 2);
            else
              bad[0] = 1;
          }
          table[u] = off;
          if (u >= len + BEHIND) break;
        }
        __syncthreads();
        a.base = static_cast<const char*>(g.dy) + ((first + at) * g.ldy + r0) * 2;
        a.rows = len;
        tile_loop<DT, T, RING, NA, NA>(a, b, lds, len, acc);
      }
    } else {
      AcrossOperand<T> b;
      b.base = static_cast<const char*>(g.x) + (first * g.ldx + c0) * 2;
      b.pitch = g.ldx * 2;
      b.rows = end - first;
      b.init(base + RING * BYTES, wv, wc * (T / 2), cols);
      if (!SPLIT || first < end) tile_loop<DT, T, RING, NA, NA>(a, b, lds, (int)(end - first), acc);
    }
    if constexpr (SPLIT) {
      // (all of the tile is NaN then, by any of its ranges)
      const float add = INDEXED && first < end && bad[0] ? __builtin_nanf("") : 0.0f;
      const uint32_t y = e * ((n + T - 1) / T) + (uint32_t)(r0 / T), across = (k + T - 1) / T;
      store_part<T>(part, ((uint64_t)y * across + c0 / T) * splits + z, acc, add);
    } else {
      store_tile<DT, T, INDEXED ? 2 : 0>(lds, acc, to, k, rows, cols, bad, g.past);
    }
  } else {
    RowTile w;
    uint32_t xt, y;
    if (!plan_tile(static_cast<const Plan*>(plan), nx * splits, blockIdx.x, w, xt, y)) return;
    const uint32_t z = SPLIT ? xt % splits : 0;
    if (SPLIT) xt = __builtin_amdgcn_readfirstlane(xt / splits);
    const int e = __builtin_amdgcn_readfirstlane(w.e);
    const int live = __builtin_amdgcn_readfirstlane(w.live);
    const int64_t first = uniform(w.first);
    const int64_t width = WHAT == GROUPED_LINEAR ? n : k, c0 = (int64_t)xt * T;
    const int cols = (int)(width - c0 < T ? width - c0 : T);
    uint16_t* const to = out + first * width + c0;
    const bool sums = WHAT == GROUPED_GRAD_X && g.f32_out;
    static_assert(T / 2 * (4 * T + 16) <= LDS_BYTES<T, 4>, "store_sums");
    float* const to_sums = static_cast<float*>(g.out) + first * width + c0;
    if (e < 0) {
      if (z == 0 && sums)
        store_zeros<T>(to_sums, width, live, cols);
      else if (z == 0)
        store_zeros<T>(to, width, live, cols);
      return;
    }
    const int all = WHAT == GROUPED_LINEAR ? k : n;  // of the contraction
    const int from = SPLIT ? __builtin_amdgcn_readfirstlane(z * per * STAGE) : 0;
    const int end = SPLIT && from + per * STAGE < all ? from + per * STAGE : all;
    // Of 256 x 256 with half the rows at most a wave takes 128 x 64, half as many products (64 experts
    // of 1024 x 2048 with 64 slots each 78 us, so 66).
    const bool half = T == 256 && live <= T / 2;
    auto finish = [&](auto& a, auto& b) {
      if constexpr (T == 256) {
        if (half) {
          tile_loop<DT, T, RING, NA, NA / 2>(a, b, lds, end - from, acc);
          if (sums)
            store_sums<T, NA / 2>(lds, acc, to_sums, width, live, cols, g.past);
          else
            store_tile<DT, T, INDEXED ? 1 : 0, NA / 2>(lds, acc, to, width, live, cols, bad, g.past);
          return;
        }
      }
      tile_loop<DT, T, RING, NA, NA>(a, b, lds, end - from, acc);
      if constexpr (SPLIT)
        store_part<T>(part, ((uint64_t)y * nx + xt) * splits + z, acc, 0.0f);
      else if (sums)
        store_sums<T>(lds, acc, to_sums, width, live, cols, g.past);
      else
        store_tile<DT, T, INDEXED ? 1 : 0>(lds, acc, to, width, live, cols, bad, g.past);
    };
    AlongOperand<T> a;
    if constexpr (WHAT == GROUPED_LINEAR) {
      a.init(base, wv, half ? 0 : wr * (T / 2), from, end);
      if constexpr (INDEXED) {
        a.rs = rsrc(g.x, g.x_rows > 0 ? ((g.x_rows - 1) * g.ldx + whole(k)) * 2 : 0);
#pragma unroll
        for (int i = 0; i < NA; ++i) {
          const int t = a.row_of(wv, i);
          int64_t s = t < live ? g.rows[first + t] : 0;
          const bool in = s >= 0 && s < g.x_rows;
          if ((lane & 3) == 0) bad[t] = t < live && !in;
          a.row[i] = t < live && in ? (uint32_t)(s * g.ldx * 2) : ROW_DEAD;
        }
      } else {
        a.rs = rsrc(static_cast<const char*>(g.x) + first * g.ldx * 2,
                    ((int64_t)(live - 1) * g.ldx + whole(k)) * 2);
#pragma unroll
        for (int i = 0; i < NA; ++i) {
          const int t = a.row_of(wv, i);
          a.row[i] = t < live ? (uint32_t)(t * g.ldx * 2) : ROW_DEAD;
        }
      }
      AlongOperand<T> b;
      b.init(base + RING * BYTES, wv, half ? wv * (T / 4) : wc * (T / 2), from, end);
      b.rs = rsrc(static_cast<const char*>(g.w) + ((int64_t)e * n + c0) * g.ldw * 2,
                  ((int64_t)(cols - 1) * g.ldw + whole(k)) * 2);
#pragma unroll
      for (int i = 0; i < NA; ++i) {
        const int t = b.row_of(wv, i);
        b.row[i] = t < cols ? (uint32_t)(t * g.ldw * 2) : ROW_DEAD;
      }
      finish(a, b);
    } else {
      a.init(base, wv, half ? 0 : wr * (T / 2), from, end);
      a.rs = rsrc(static_cast<const char*>(g.dy) + first * g.ldy * 2,
                  ((int64_t)(live - 1) * g.ldy + whole(n)) * 2);
#pragma unroll
      for (int i = 0; i < NA; ++i) {
        const int t = a.row_of(wv, i);
        a.row[i] = t < live ? (uint32_t)(t * g.ldy * 2) : ROW_DEAD;
      }
      AcrossOperand<T> b;
      b.base = static_cast<const char*>(g.w) + (((int64_t)e * n + from) * g.ldw + c0) * 2;
      b.pitch = g.ldw * 2;
      b.rows = end - from;
      b.init(base + RING * BYTES, wv, half ? wv * (T / 4) : wc * (T / 2), cols);
      finish(a, b);
    }
  }
}

// The sums of a tile's ranges, added in their order; a workgroup to the quarter that one wave of the
// product held, a wave to 32 x 32 of its results.
template <int DT, int WHAT, bool INDEXED>
__global__ __launch_bounds__(256) void grouped_join_kernel(GroupedArgs g, int width, uint32_t nx,
                                                           uint32_t ny, const Plan* plan,
                                                           const float* part, int splits) {
  constexpr int T = 128;
  const uint32_t tile = blockIdx.x / 4, quarter = blockIdx.x & 3, y = tile / nx, xt = tile - y * nx;
  RowTile w;
  if constexpr (WHAT == GROUPED_GRAD_W) {
    const int e = y / ny, r0 = (y - e * ny) * T;
    int64_t first, end;
    slot_range(g, e, first, end);
    if (first == end) return;
    w = RowTile{e * g.n + r0, (int32_t)(g.n - r0), e};
  } else {
    if (y >= (uint32_t)plan->count) return;
    w = plan->tile[y];
    if (w.e < 0) return;
  }
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const f32x4v* from = reinterpret_cast<const f32x4v*>(part) + (int64_t)tile * splits * (T * T / 4) +
                       quarter * (T * T / 16) + wave * 256 + lane;
  f32x4v sum[4] = {};
  for (int z = 0; z < splits; ++z)
#pragma unroll
    for (int q = 0; q < 4; ++q) sum[q] += from[(int64_t)z * (T * T / 4) + q * 64];
  const int r = (quarter >> 1) * 64 + (wave >> 1) * 32 + (lane & 31);
  if (r >= w.live) return;
  if constexpr (INDEXED && WHAT == GROUPED_LINEAR) {
    if ((uint64_t)g.rows[w.first + r] >= (uint64_t)g.x_rows)
#pragma unroll
      for (int q = 0; q < 4; ++q) sum[q] = sum[q] + __builtin_nanf("");
  }
  const int dt = WHAT == GROUPED_GRAD_X && g.f32_out ? 0 : DT;
  char* const to = static_cast<char*>(g.out) + (w.first + r) * width * (dt == 0 ? 4 : 2);
  const int c0 = (int)xt * T + (quarter & 1) * 64 + (wave & 1) * 32 + 4 * (lane >> 5);
#pragma unroll
  for (int q = 0; q < 4; ++q)
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int c = c0 + 8 * q + u;
      if (c < width) store_from_f32(to, c, dt, sum[q][u]);
    }
}

// How a product goes: in tiles of T, its contraction cut into `splits` ranges of `per` stages.
struct Cut {
  int T, splits, per;
};

template <int DT, int WHAT, int T, int RING, bool INDEXED>
int launch_tile(const GroupedArgs& g, const Cut& cut, char* plan, hipStream_t s,
                const char* what) {
  const int64_t cols = WHAT == GROUPED_LINEAR ? g.n : g.k;
  int64_t nx = (cols + T - 1) / T, ny = (g.n + T - 1) / T, count;
  const int64_t tiles = nx * (WHAT == GROUPED_GRAD_W ? ny * g.experts : most_tiles(g, T));
  const uint32_t across = (uint32_t)nx, down = (uint32_t)ny;
  if constexpr (WHAT == GROUPED_GRAD_W) {
    nx = (nx + 3) / 4 * 4;
    ny = (ny + 1) / 2 * 2;
    count = nx * ny * g.experts * cut.splits;
  } else {
    ny = most_tiles(g, T);
    count = (nx * cut.splits * ny + 7) / 8 * 8;
    if (int rc = launch_plan(g, T, reinterpret_cast<Plan*>(plan), s, what)) return rc;
  }
  if constexpr (T == 128) {
    if (cut.splits > 1) {
      const Plan* p = reinterpret_cast<const Plan*>(plan);
      float* part = reinterpret_cast<float*>(
          plan + (WHAT == GROUPED_GRAD_W ? 0 : plan_bytes(g, T)));
      grouped_tile_kernel<DT, WHAT, T, RING, INDEXED, true><<<(unsigned)count, 256, 0, s>>>(
          g, (uint32_t)nx, (uint32_t)ny, p, part, cut.splits, cut.per);
      grouped_join_kernel<DT, WHAT, INDEXED><<<(unsigned)(tiles * 4), 256, 0, s>>>(
          g, (int)cols, across, down, p, part, cut.splits);
      return launch_status(what);
    }
  }
  grouped_tile_kernel<DT, WHAT, T, RING, INDEXED, false>
      <<<(unsigned)count, 256, 0, s>>>(g, (uint32_t)nx, (uint32_t)ny, plan, nullptr, 1, 0);
  return launch_status(what);
}

template <int DT, int WHAT, int T, int RING>
int launch_indexed(const GroupedArgs& g, const Cut& cut, char* plan, hipStream_t s,
                   const char* what) {
  if constexpr (WHAT != GROUPED_GRAD_X) {
    if (g.rows) return launch_tile<DT, WHAT, T, RING, true>(g, cut, plan, s, what);
  }
  return launch_tile<DT, WHAT, T, RING, false>(g, cut, plan, s, what);
}

// What `tiles` tiles of `stages` stages take, in us: rounds of `cap` of them, a + b for each stage,
// and where a last round leaves half the places empty b2.
double rounds(double tiles, double cap, double a, double stages, double b, double b2) {
  const double whole = __builtin_floor(tiles / cap), rest = tiles - whole * cap;
  return whole * (a + b * stages) +
         (rest <= 0 ? 0 : a + stages * (2 * rest <= cap ? b2 : b));
}

// 256-tiles, one workgroup to a CU, read LDS half as often for a product; 128-tiles, two to a CU,
// fill the chip with fewer results and leave less of a range's last tile empty.  The rule counts
// rounds of the chip with what was measured a stage (us, at full and half chips): 0.87 for 256-tiles,
// 0.55 and 0.35 for 128-tiles.  Over 80 products of ragged ranges, 32 to 1024 slots an expert, what
// it takes is 1.3% slower than the better on average and 21% at most (always 128: 3%, always 256:
// 13%); 8 experts of 14336 x 4096 with 256 slots each 380 us and 465, 16 of 2048 x 4096 with 384 each
// 220 and 152.  It goes by the mean range, as the ranges are on the device: where one of 64 experts of
// 1024 x 2048 has nine tenths of 131072 slots, its 32 tiles of the weights' gradient run alone, 1872 us
// for 552 of even ranges.
// The weights' gradient takes 0.75 a stage in 256-tiles, and in 128-tiles of a two-stage ring, four
// to a CU, hides the stores of short sums behind others: ranges of 64 slots 72 us and 62, of 512 585
// and 619.
// Tiles that leave half the chip empty split their contraction where that saves more than the join
// costs, 4 us and 0.025 for each range that a tile is cut into: 512 slots of 8 experts of 1024 x 4096
// 44 us and 27, 300 of one of 1024 x 14336 133 and 33; 256 of 8 of 2048 x 1024 17 and, split, 22; the
// gradient of 8 of 512 x 512 from 65536 slots 121 and 71, of one of 1024 x 1024 from 131072 2560 and
// 373.
Cut cut_of(const GroupedArgs& g, int what) {
  const bool grad_w = what == GROUPED_GRAD_W;
  const double cols = what == GROUPED_LINEAR ? g.n : g.k;
  const int stages = (int)(((what == GROUPED_LINEAR ? g.k : grad_w ? g.slots / g.experts : g.n) +
                            STAGE - 1) / STAGE);
  // a live expert's last row tile is half full on average
  const double live = g.slots < g.experts ? g.slots : g.experts;
  auto tiles = [&](int T, double part) {
    const double rows = (double)g.slots / T + part * live, least = T == 256 ? part * live : live;
    return __builtin_ceil(cols / T) * (grad_w         ? g.experts * __builtin_ceil((double)g.n / T)
                                       : rows > least ? rows
                                                      : least);
  };
  const double all = tiles(128, 0.5);
  if (grad_w ? tiles(256, 0) >= 192 && g.slots >= 384 * g.experts
             : 0.9 * rounds(tiles(256, 0.6), 256, 5, stages, 0.87, 0.87) <
                   rounds(all, 512, 3, stages, 0.55, 0.35))
    return Cut{256, 1, 0};
  Cut c{128, 1, stages};
  // (the weights come from memory at 4.5e6 bytes a us whatever the cut)
  const double read = grad_w ? 0 : live * g.n * g.k * 2 / 4.5e6;
  double best = 0.8 * (stages * 0.35 > read ? stages * 0.35 : read);
  for (int splits = 2; splits <= 16 && all >= 1 && all * splits <= 512; ++splits) {
    int per = (stages + splits - 1) / splits;
    per += per & 1;  // (whole lines of 128 bytes)
    const double work = per * (all * splits > 256 ? 0.55 : 0.35);
    const double us = (work > read ? work : read) + 4 + 0.025 * all * splits;
    if (us < best) {
      best = us;
      c.per = per;
      c.splits = (stages + per - 1) / per;
    }
  }
  return c;
}

template <int DT, int WHAT>
int launch_size(const GroupedArgs& g, char* plan, hipStream_t s, const char* what) {
  const Cut cut = cut_of(g, WHAT);
  if (cut.T == 256) return launch_indexed<DT, WHAT, 256, 4>(g, cut, plan, s, what);
  return launch_indexed<DT, WHAT, 128, WHAT == GROUPED_GRAD_W ? 2 : 4>(g, cut, plan, s, what);
}

}  // namespace

int launch_plan(const GroupedArgs& g, int T, Plan* plan, hipStream_t s, const char* name) {
  grouped_plan_kernel<<<1, 1024, 0, s>>>(g, T, plan, most_tiles(g, T));
  return launch_status(name);
}

int64_t grouped_plan_bytes(const GroupedArgs& g, int what, int dtype) {
  const bool grad_w = what == GROUPED_GRAD_W;
  if (dtype == 0) return grad_w ? 0 : plan_bytes(g, 64);
  const Cut cut = cut_of(g, what);
  const int64_t nx = ((what == GROUPED_LINEAR ? g.n : g.k) + cut.T - 1) / cut.T;
  const int64_t tiles = nx * (grad_w ? g.experts * ((g.n + cut.T - 1) / cut.T) : most_tiles(g, cut.T));
  return (grad_w ? 0 : plan_bytes(g, cut.T)) +
         (cut.splits > 1 ? tiles * cut.splits * cut.T * cut.T * 4 : 0);
}

int grouped_tile_side(const GroupedArgs& g, int what, int64_t& splits) {
  const Cut cut = cut_of(g, what);
  splits = cut.splits;
  return cut.T;
}

int grouped_tiles(const GroupedArgs& args, int what, int dtype, char* plan, hipStream_t s,
                  const char* name) {
  GroupedArgs g = args;
  // Results that fill half of the last cache (256 MB) would only push the operands out (the weights'
  // gradient of 8 experts of 14336 x 4096 from 2048 slots 411 us, so 363; of 64 of 1024 x 2048 from
  // 16384 131 and 109).
  const int64_t results = what == GROUPED_GRAD_W   ? g.experts * g.n * g.k
                          : what == GROUPED_LINEAR ? g.slots * g.n
                                                   : g.slots * g.k;
  g.past = results * (g.f32_out ? 4 : 2) > 128ll << 20;
#define HI2X_GROUPED(WHAT)                                     \
  return dtype == 1 ? launch_size<1, WHAT>(g, plan, s, name) : \
                      launch_size<2, WHAT>(g, plan, s, name)
  if (what == GROUPED_LINEAR) HI2X_GROUPED(GROUPED_LINEAR);
  if (what == GROUPED_GRAD_X) HI2X_GROUPED(GROUPED_GRAD_X);
  HI2X_GROUPED(GROUPED_GRAD_W);
#undef HI2X_GROUPED
}

}  // namespace hi2x
