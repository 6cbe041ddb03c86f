// Products of atoms' rows with learned weights, one weight for all or one for each species.
//
//   z = x W + b                   (W, b of the row's species)
//   y = residual + D(act(z))      D: dropout
//
// Gradient for the adjoint g of y:
//
//   dz = D(g act'(z)),  dx = dz W^T,  dW = x^T dz,  db = sum of dz over rows
//
// Rows of one species are found through an order of the rows (species.hip), so
// neither x nor y is moved.  A workgroup owns a tile of one species' rows (forward and dx,
// linear_rows.hip) or of a weight's gradient over a share of the rows
// (linear_weights.hip), stages both operands in LDS and multiplies with the
// 32 x 32 x 16 matrix instruction, bf16 x bf16 -> fp32.
//
// fp32 operands are held as three bf16 parts, x = h + m + l: h is x rounded to
// bf16, m the rest rounded, l what is left, 24 bits in all.  A product takes the
// six terms hh, hm, mh, mm, hl, lh; those left out are below 2^-26 of it, less than
// fp32's own rounding (Henry, Tang and Heinecke, "Leveraging the bfloat16
// artificial intelligence datatype for higher-precision computations", 2019).  All six go into one
// accumulator, the small ones first: a step of sixteen adds to the running sum six times, where sixteen fp32 products one
// after the other add to it sixteen times.  Six bf16
// instructions of 32 cycles cover what eight fp32 ones of 64 would.  Values of 2^-110
// and below lose their last bits, 2^-133 at most.  A value that is not finite, or
// rounds to infinity in bf16, would leave NaN where fp32 leaves an infinity or a
// number: results that are not finite are computed again, value by value in fp32
// (exact_dots).
#pragma once

#include <type_traits>

#include "random.h"
#include "tiles.h"

namespace ye3t {
namespace linear {

using namespace tiles;

constexpr float kLog2e = 1.44269504f;

enum Activation { kNone = 0, kRelu = 1, kSilu = 2, kGelu = 3 };

// Phi(z), the normal distribution's integral, and exp(-z^2 / 2).  The smaller tail is
// exp(-x^2) f(x) / 2 with x = |z| / sqrt 2; f, the scaled complementary error function,
// is a polynomial in t = 1 / (1 + 0.44 x) fitted for the least relative error, 1.9e-7 up to
// x = 14 (beyond, exp(-x^2) is zero).  The exponent's rounding is more than that far out: the tail is
// good to 5e-7 up to |z| = 1, 2e-6 up to 6, 4e-6 up to 9 and 7e-6 up to 12.5 (measured), about z^2 2^-24.
struct Normal {
  float phi, bell;
};
__device__ inline Normal normal_of(float z) {
  const float t = __builtin_amdgcn_rcpf(1.0f + 0.311126984f * fabsf(z));
  const float f =
      t * (0.248216531f +
           t * (0.248935427f +
                t * (0.216934685f +
                     t * (0.216993537f +
                          t * (-0.0222940624f + t * (0.298866830f + t * (-0.279152495f + t * 0.0714997336f)))))));
  const float bell = __builtin_amdgcn_exp2f(z * z * (-0.5f * kLog2e)), tail = 0.5f * bell * f;
  return {z < 0.0f ? tail : 1.0f - tail, bell};
}

// 1 / (1 + exp(-z)) = scaled unit.  Of negative z the exponential is held times 2^24, as its instruction gives no
// subnormal values and z times them may be a normal one.
struct Logistic {
  float scaled, unit;
};
__device__ inline Logistic logistic_of(float z) {
  constexpr float kUnit = 5.9604644775390625e-8f;  // 2^-24
  const float t = __builtin_amdgcn_exp2f(fmaf(-kLog2e, fabsf(z), 24.0f)), r = __builtin_amdgcn_rcpf(fmaf(t, kUnit, 1.0f));
  return {z < 0.0f ? t * r : r, z < 0.0f ? kUnit : 1.0f};
}

// Eight values; the choice is made once for them.
__device__ inline void activate(int act, float* v) {
  if (act == kRelu) {
#pragma unroll
    for (int q = 0; q < 8; ++q) v[q] = v[q] <= 0.0f ? 0.0f : v[q];
  } else if (act == kSilu) {
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      const Logistic e = logistic_of(v[q]);
      v[q] = v[q] * e.scaled * e.unit;
    }
  } else {
#pragma unroll
    for (int q = 0; q < 8; ++q) v[q] = v[q] * normal_of(v[q]).phi;
  }
}

// g act'(z).  relu passes g or stops it: a unit that is dead gives zero for an infinite g too, and one of NaN, which
// activate() passes, passes g.
__device__ inline float through(int act, float g, float z) {
  if (act == kRelu) return z <= 0.0f ? 0.0f : g;
  if (act == kSilu) {
    const Logistic e = logistic_of(z);
    return g * (fmaf(z * e.scaled, 1.0f - e.scaled * e.unit, e.scaled) * e.unit);
  }
  const Normal n = normal_of(z);
  return g * (n.phi + z * n.bell * 0.398942280f);
}

// f(0) .. f(N - 1) with the number as a type
template <int N, int I = 0, typename F>
__device__ inline void repeat(F f) {
  if constexpr (I < N) {
    f(std::integral_constant<int, I>());
    repeat<N, I + 1>(f);
  }
}

// ---- operands ------------------------------------------------------------------
template <typename T>
constexpr int kParts = sizeof(T) == 4 ? 3 : 1;

// A tile of a matrix operand: LINES rows or columns of the result by KT of the
// contraction, as bf16, kParts of it one after the other.
//   along   LINES x KT: memory runs along the contraction
//   across  KT x LINES: memory runs across it, and the transposing read turns it
template <typename T, int LINES, int KT, bool ACROSS>
struct Tile {
  static constexpr int kValues = LINES * KT, kChunks = kValues / 8, kRow = (ACROSS ? LINES : KT) / 8;
  static constexpr int kBytes = kParts<T> * kValues * 2;

  // chunk x of the tile, in the order of its lines (across: of its contraction)
  __device__ static inline int line_of(int x) { return x / kRow; }
  __device__ static inline int column_of(int x) { return x % kRow * 8; }
  __device__ static inline void put(__bf16* tile, int x, const Chunk<T, 8>& c) {
    const int line = line_of(x);
    __bf16* to = tile + (line * kRow + (x % kRow ^ turn<__bf16, kRow * 8>(line))) * 8;
    bf16x8 part[kParts<T>];
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      if (kParts<T> == 1) {
        part[0][q] = __bf16(c.v[q]);
      } else {
        const float v = float(c.v[q]);
        const __bf16 h = __bf16(v);
        const float rest = v - float(h);
        const __bf16 m = __bf16(rest);
        part[0][q] = h;
        part[1 % kParts<T>][q] = m;
        part[2 % kParts<T>][q] = __bf16(rest - float(m));
      }
    }
#pragma unroll
    for (int n = 0; n < kParts<T>; ++n) *reinterpret_cast<bf16x8*>(to + n * kValues) = part[n];
  }

  // Operand of 32 lines from `line`, contraction k .. k + 15: a lane holds line
  // lane % 32, contraction k + 8 (lane / 32) + 0 .. 7.
  __device__ static inline bf16x8 operand(const __bf16* tile, int line, int k, int lane) {
    const int half = lane / 32;
    if (!ACROSS) {
      const int own = line + (lane & 31);
      return *reinterpret_cast<const bf16x8*>(tile + own * KT + ((k / 8 + half) ^ turn<__bf16, KT>(own)) * 8);
    }
    typedef short s16x4 __attribute__((ext_vector_type(4)));
    typedef short s16x8 __attribute__((ext_vector_type(8)));
    typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
    // lane l of a block of 16 gives the address of four values of contraction l / 4, lines
    // 4 (l % 4) .. + 3, and gets four of line l's
    const int at = k + 8 * half + (lane & 15) / 4, chunk = line / 8 + (lane & 16) / 8 + (lane & 3) / 2;
    const __bf16* from = tile + at * LINES + 4 * (lane & 1);
    const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(from + (chunk ^ turn<__bf16, LINES>(at)) * 8));
    const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (lds_s16x4*)(from + 4 * LINES + (chunk ^ turn<__bf16, LINES>(at + 4)) * 8));
    const s16x8 both = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    return __builtin_bit_cast(bf16x8, both);
  }
};

// The chunks of a tile that one of NT threads loads and puts.
template <typename T, int LINES, int KT, bool ACROSS, int NT>
struct Loads {
  typedef Tile<T, LINES, KT, ACROSS> Of;
  static constexpr int kEach = Of::kChunks / NT;
  Chunk<T, 8> held[kEach];

  __device__ static inline int line_of(int n) { return Of::line_of(n * NT + int(threadIdx.x)); }
  __device__ static inline int column_of(int n) { return Of::column_of(n * NT + int(threadIdx.x)); }
  static_assert(Of::kChunks % NT == 0, "every thread loads as many chunks");
  // Whole chunks
  __device__ inline void load(const T* const* from) {
#pragma unroll
    for (int n = 0; n < kEach; ++n) held[n] = Chunk<T, 8>::load(from[n]);
  }
  // left(n): values that exist from from[n] on.  Eight or none, which needs no branches (1 000 x 1 000 x 1 000 in
  // bf16, whose last tiles are all of these: 14 us with them, 11 without), or any number.
  template <typename L>
  __device__ inline void load_chunks(const T* const* from, L left) {
#pragma unroll
    for (int n = 0; n < kEach; ++n)
      held[n] = Chunk<T, 8>::load(left(n) > 0 ? from[n] : reinterpret_cast<const T*>(kZeros));
  }
  template <typename L>
  __device__ inline void load(const T* const* from, L left) {
#pragma unroll
    for (int n = 0; n < kEach; ++n) {
      const int most = left(n);
      held[n] = most > 0 ? Chunk<T, 8>::load(from[n], most) : Chunk<T, 8>::zero();
    }
  }
  __device__ inline void put(__bf16* tile) const {
#pragma unroll
    for (int n = 0; n < kEach; ++n) {
      Of::put(tile, n * NT + int(threadIdx.x), held[n]);
    }
  }
};

// The same straight to LDS, where every chunk is 16 whole aligned bytes.  A wave's 64 chunks lie one after the
// other, so the thread at place x of a line takes the chunk that belongs there.  The instruction has no
// result, but the compiler takes every transposing read of LDS to wait for it and would wait for the next tile's
// loads before it reads this one's (8192^3, both operands along and across: 1 004 and 1 094 us by
// the builtin, 968 and 970 so); it is written out, and the kernels count the loads themselves.
template <int LINES, int KT, bool ACROSS, int NT>
struct DirectLoads {
  typedef Tile<__bf16, LINES, KT, ACROSS> Of;
  static constexpr int kEach = Of::kChunks / NT;
  static_assert(Of::kChunks % NT == 0, "every thread loads as many chunks");

  __device__ static inline int line_of(int n) { return Of::line_of(n * NT + int(threadIdx.x)); }
  __device__ static inline int column_of(int n) {
    const int x = n * NT + int(threadIdx.x);
    return (x % Of::kRow ^ turn<__bf16, Of::kRow * 8>(Of::line_of(x))) * 8;
  }
  __device__ static inline const __bf16* none() { return reinterpret_cast<const __bf16*>(kZeros); }
  // Chunk n of this thread
  __device__ static inline void load(__bf16* tile, int n, int wave, const __bf16* p) {
    const unsigned to = unsigned(uintptr_t((__attribute__((address_space(3))) void*)(tile + (n * NT + 64 * wave) * 8)));
    // m0, the place in LDS, takes one instruction between to be there
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(to), "v"(p) : "m0");
  }
};

template <typename T, int LINES, int KT, bool ACROSS, int NT, bool DIRECT>
using LoadsOf = std::conditional_t<DIRECT, DirectLoads<LINES, KT, ACROSS, NT>, Loads<T, LINES, KT, ACROSS, NT>>;

// All but the newest N loads of this wave have arrived, its reads of LDS are done, and so are the other waves'.
template <int N>
__device__ inline void arrive_and_meet() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

// A workgroup's tile: WM x WN waves of FM x FN squares of 32 x 32 each, times WK shares of
// the contraction, of which a step takes BK each.
template <int WM_, int WN_, int WK_, int FM_, int FN_, int BK_, int BUFFERS_, int WAVES_>
struct Shape {
  static constexpr int WM = WM_, WN = WN_, WK = WK_, FM = FM_, FN = FN_, BK = BK_, BUFFERS = BUFFERS_;
  static constexpr int TM = WM * FM * 32, TN = WN * FN * 32, KT = WK * BK, NT = 64 * WM * WN * WK;
  static constexpr int kPerSimd = WAVES_;  // waves a SIMD that the registers are set for
  // rows of a wave's square rows on their way out: 16 bytes more than the values, so that 16 rows' chunks lie in
  // different banks
  static constexpr int kOutRow = FN * 32 + 4;
  static constexpr int kOutBytes = WM * WN * WK * 32 * kOutRow * 4;
};

__device__ inline void multiply(const bf16x8& a, const bf16x8& b, f32x16& c) {
  c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

// sum[i][j] += the wave's squares over one step of the contraction.  The columns' operand comes first, so
// that a lane holds row lane % 32 and, in register 4 b + j, column 8 b + 4 (lane / 32) + j.
template <typename T, typename S>
struct Operands {
  bf16x8 x[S::FM][kParts<T>], y[S::FN][kParts<T>];
};
template <typename T, typename S, typename A, typename B>
__device__ inline void read_operands(const __bf16* a, const __bf16* b, int wm, int wn, int k, int lane, Operands<T, S>& o) {
#pragma unroll
  for (int n = 0; n < kParts<T>; ++n) {
#pragma unroll
    for (int j = 0; j < S::FN; ++j) o.y[j][n] = B::operand(b + n * B::kValues, (wn * S::FN + j) * 32, k, lane);
#pragma unroll
    for (int i = 0; i < S::FM; ++i) o.x[i][n] = A::operand(a + n * A::kValues, (wm * S::FM + i) * 32, k, lane);
  }
}
template <typename T, typename S>
__device__ inline void multiply_operands(const Operands<T, S>& o, f32x16 (*sum)[S::FN]) {
  constexpr int P = kParts<T>;
#pragma unroll
  for (int i = 0; i < S::FM; ++i)
#pragma unroll
    for (int j = 0; j < S::FN; ++j) {
      if constexpr (P == 3) {
        multiply(o.y[j][2], o.x[i][0], sum[i][j]);
        multiply(o.y[j][0], o.x[i][2], sum[i][j]);
        multiply(o.y[j][1], o.x[i][1], sum[i][j]);
        multiply(o.y[j][1], o.x[i][0], sum[i][j]);
        multiply(o.y[j][0], o.x[i][1], sum[i][j]);
      }
      multiply(o.y[j][0], o.x[i][0], sum[i][j]);
    }
}
template <typename T, typename S, typename A, typename B>
__device__ inline void multiply_tiles(const __bf16* a, const __bf16* b, int wm, int wn, int wk, int lane,
                                      f32x16 (*sum)[S::FN]) {
#pragma unroll
  for (int k = 0; k < S::BK; k += 16) {
    Operands<T, S> o;
    read_operands<T, S, A, B>(a, b, wm, wn, wk * S::BK + k, lane, o);
    multiply_operands<T, S>(o, sum);
  }
}

// sum[i][j] over all `steps` tiles of direct loads.  load(t, part, parts): issues a part of tile t's LOADS loads of
// a thread; with(t): while tile t is there.  A step of 16 along the contraction reads the
// operands of the next one between its products, and the last of a tile meets the other waves first, so
// that no product waits for a barrier.  With two buffers a tile's loads are issued in the first half
// of the one before: in four parts, the last right before the wait, 8192^3 took 970 us, so 893.
// Where STARTED the first tile's loads have been issued, and `behind` (0, 16 or 32) memory operations or more after them.
template <typename S, typename A, typename B, int LOADS, bool STARTED, typename TileA, typename TileB, typename Load,
          typename With>
__device__ inline void multiply_direct(int steps, int behind, TileA tile_a, TileB tile_b, int wm, int wn, int wk,
                                       int lane, Load load, With with, f32x16 (*sum)[S::FN]) {
  typedef __bf16 T;
  constexpr int AHEAD = S::BUFFERS - 1, SUB = S::BK / 16, PARTS = AHEAD == 1 ? SUB / 2 : SUB;
  typedef std::integral_constant<int, 0> Zero;
  typedef std::integral_constant<int, 1> One;
#pragma unroll
  for (int t = 0; t < AHEAD && !STARTED; ++t)
    if (t < steps) load(t, Zero(), One());
  static_assert(!STARTED || AHEAD == 1, "one tile is loaded ahead");
  auto meet = [&](int t) {  // tile t is there, and tile t - 1 has been read
    if (t + AHEAD <= steps) arrive_and_meet<(AHEAD - 1) * LOADS>();
    else arrive_and_meet<0>();
  };
  Operands<T, S> o[2];
  if (steps) {
    if (STARTED && behind >= 32) arrive_and_meet<32>();
    else if (STARTED && behind >= 16) arrive_and_meet<16>();
    else meet(0);
    read_operands<T, S, A, B>(tile_a(0), tile_b(0), wm, wn, wk * S::BK, lane, o[0]);
  }
  for (int t = 0; t < steps; ++t) {
    repeat<SUB>([&](auto sub) {
      constexpr int k = decltype(sub)::value;
      if constexpr (k < PARTS) {
        if (t + AHEAD < steps) load(t + AHEAD, sub, std::integral_constant<int, PARTS>());
      }
      if constexpr (k == 0) with(t);
      if constexpr (k + 1 < SUB) {
        read_operands<T, S, A, B>(tile_a(t), tile_b(t), wm, wn, wk * S::BK + 16 * (k + 1), lane, o[(k + 1) & 1]);
      } else if (t + 1 < steps) {
        meet(t + 1);
        read_operands<T, S, A, B>(tile_a(t + 1), tile_b(t + 1), wm, wn, wk * S::BK, lane, o[(k + 1) & 1]);
      }
      multiply_operands<T, S>(o[k & 1], sum);
      repeat<S::FM * S::FN>([&](auto) {  // one read of LDS, one product
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
      });
    });
  }
}

// Passes the wave's squares through LDS and gives them out eight columns of a row at a time, so that memory
// is read and written along rows: use(rows, columns, values) of BATCH chunks of the workgroup's tile.  The
// shares of the contraction are added in order.
template <typename S, int BATCH, typename F>
__device__ inline void give_out(char* lds, const f32x16 (*sum)[S::FN], int wm, int wn, int wk, int lane, F use) {
  constexpr int CHUNKS = S::FN * 4, STRIDE = S::kOutRow, BLOCK = 32 * STRIDE, EACH = 32 * CHUNKS / 64;
  const int wave = (wk * S::WM + wm) * S::WN + wn;
  float* own = reinterpret_cast<float*>(lds) + wave * BLOCK;
  repeat<S::FM>([&](auto number) {
    constexpr int i = decltype(number)::value;
#pragma unroll
    for (int j = 0; j < S::FN; ++j)
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        f32x4 v;
#pragma unroll
        for (int q = 0; q < 4; ++q) v[q] = sum[i][j][4 * b + q];
        *reinterpret_cast<f32x4*>(own + (lane & 31) * STRIDE + 32 * j + 8 * b + 4 * (lane / 32)) = v;
      }
    if constexpr (S::WK == 1) {
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int first = 0; first < EACH; first += BATCH) {
        int r[BATCH], c[BATCH];
        float v[BATCH][8];
#pragma unroll
        for (int n = 0; n < BATCH; ++n) {
          const int x = (first + n) * 64 + lane, row = x / CHUNKS, column = x % CHUNKS * 8;
#pragma unroll
          for (int q = 0; q < 8; ++q) v[n][q] = own[row * STRIDE + column + q];
          r[n] = (wm * S::FM + i) * 32 + row;
          c[n] = wn * S::FN * 32 + column;
        }
        use(r, c, v);
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
    } else {
      static_assert(S::WK == 1 || (S::FM == 1 && S::WM == 1 && S::WN == 1), "shares of one wave's rows");
      __syncthreads();
      for (int x = int(threadIdx.x); x < 32 * CHUNKS; x += S::NT) {
        int r[1] = {x / CHUNKS}, c[1] = {x % CHUNKS * 8};
        float v[1][8];
#pragma unroll
        for (int q = 0; q < 8; ++q) v[0][q] = 0.0f;
#pragma unroll
        for (int w = 0; w < S::WK; ++w)
#pragma unroll
          for (int q = 0; q < 8; ++q) v[0][q] += reinterpret_cast<const float*>(lds)[w * BLOCK + r[0] * STRIDE + c[0] + q];
        use(r, c, v);
      }
    }
  });
}

// The same without LDS: the halves of the wave exchange what makes eight columns of a lane's row whole.
template <typename S, int BATCH, typename F>
__device__ inline void hand_out(const f32x16 (*sum)[S::FN], int wm, int wn, int lane, F use) {
  const int half = lane / 32;
  repeat<S::FM * 2 * S::FN / BATCH>([&](auto number) {
    constexpr int first = decltype(number)::value * BATCH;
    int r[BATCH], c[BATCH];
    float v[BATCH][8];
#pragma unroll
    for (int n = 0; n < BATCH; ++n) {
      const int i = (first + n) / (2 * S::FN), j = (first + n) / 2 % S::FN, b = (first + n) % 2 * 2;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const unsigned x = __builtin_bit_cast(unsigned, float(sum[i][j][4 * b + q]));
        const unsigned y = __builtin_bit_cast(unsigned, float(sum[i][j][4 * b + 4 + q]));
        const auto both = __builtin_amdgcn_permlane32_swap(x, y, false, false);
        v[n][q] = __builtin_bit_cast(float, unsigned(both[0]));
        v[n][4 + q] = __builtin_bit_cast(float, unsigned(both[1]));
      }
      r[n] = (wm * S::FM + i) * 32 + (lane & 31);
      c[n] = (wn * S::FN + j) * 32 + 8 * (b + half);
    }
    use(r, c, v);
  });
}

// v[q] = sum of a(k) b(k, q) over k < K in fp32, for results that are not finite; q < most exist.  Sums that have all become
// NaN stay so, and the rest is left out.  One step at a time: two took registers that the kernels' own loops need.
template <typename A, typename B>
__device__ void exact_dots(A a, B b, int K, int most, float* v) {
#pragma unroll
  for (int q = 0; q < 8; ++q) v[q] = 0.0f;
#pragma unroll 1
  for (int k = 0; k < K; ++k) {
    const float x = a(k);
    bool open = false;
#pragma unroll
    for (int q = 0; q < 8; ++q)
      if (q < most) {
        v[q] = fmaf(x, b(k, q), v[q]);
        open |= v[q] == v[q];
      }
    if (!open) break;
  }
}
__device__ inline bool any_not_finite(const float* v) {
  float worst = 0.0f;  // 0 v is NaN for infinities and NaN
#pragma unroll
  for (int q = 0; q < 8; ++q) worst += 0.0f * v[q];
  return worst != 0.0f;
}

// Consecutive tiles run on one XCD, which has an L2 of its own: workgroups go to the eight XCDs in turn.
__device__ inline int64_t tile_of_group() {
  const unsigned n = gridDim.x, b = blockIdx.x, x = b & 7;
  return int64_t(x) * (n / 8) + (x < n % 8 ? x : n % 8) + b / 8;
}

// Rows and columns of tiles: four rows of tiles go together through the columns, so that the 32 or 64 tiles that run on
// an XCD at a time share few rows and columns.
struct Place {
  int64_t row;
  int column;
};
__device__ inline Place place_of(int64_t tile, int64_t rows, unsigned columns) {
  const int64_t band = tile / (4 * int64_t(columns)), left = rows - 4 * band;
  const int high = left < 4 ? int(left) : 4;
  const unsigned in = unsigned(tile - band * 4 * columns);
  return {4 * band + in % high, int(in / high)};
}

// A row's number in memory, -1 for one that an order names outside of the rows
__device__ inline int64_t row_at(const int32_t* order, int64_t i, int64_t rows) {
  if (!order) return i;
  const int64_t r = order[i];
  return r >= 0 && r < rows ? r : -1;
}

// Sums over the rows of each group in shares: where those of a group's shares begin, of which only groups of several have
// any, and how many there are.
__device__ inline int64_t part_of(int64_t begin, int64_t share) { return 2 * begin / share; }
inline int64_t part_count(int64_t rows, int64_t share) { return share < rows ? 2 * rows / share + 1 : 0; }

inline int64_t up(int64_t bytes) { return (bytes + 255) / 256 * 256; }

// ---- the two kinds of product ----------------------------------------------------
// out[i, n] = sum over k of a[i, k] b_g[k, n], g the group of row i.  Rows behind the last group have no
// weight: a sum of zero and no bias.
template <typename T>
struct RowProduct {
  const T* a;
  int64_t a_row;
  const T* b;
  int64_t b_group, b_row;  // b[g][k][n], or b[g][n][k] where `b_across` is false
  bool b_across;
  int K, N;
  int64_t rows, groups;
  bool grouped;            // false: one weight for all rows
  const int32_t* order;
  const int64_t* offsets;
  // epilogue
  const T* bias;           // [groups][N] or null
  const T* residual;       // [rows][N] or null
  T* kept;                 // a row's sum and bias, or null
  T* out;
  int activation;
  Dropout dropout;
  unsigned tiles_n;
  int parts, part_steps;   // parts of the contraction, and steps of each where there are several
  float* part;             // their sums, [parts][rows][N], rows in the order
};

// out_g[m, n] = sum over the group's rows i of a[i, m] b[i, n], and column sums of one of the two
template <typename T>
struct WeightProduct {
  const T *a, *b;
  int64_t a_row, b_row;
  int M, N;
  int64_t rows, groups;
  bool grouped;
  const int32_t* order;
  const int64_t* offsets;
  T* out;          // [groups][M][N]
  T* sums;         // [groups][M] or [groups][N], or null
  bool sums_of_a;
  int64_t share;   // rows of one workgroup
  float* part;     // sums of the shares of groups with several, [2 rows / share + 1][M][N]
  float* sums_part;
  unsigned tiles_m, tiles_n;
  bool spread;     // the slots' tiles over the XCDs
};

// Bytes of device memory that a product takes beside its operands, whatever their addresses are, and the product
template <typename T>
int64_t row_bytes(const RowProduct<T>& p);
template <typename T>
int launch_rows(RowProduct<T> p, void* work, hipStream_t s);
template <typename T>
int64_t weight_bytes(WeightProduct<T> p);
template <typename T>
int launch_weights(WeightProduct<T> p, void* work, hipStream_t s);

}  // namespace linear
}  // namespace ye3t
