// Attention of the atoms of each structure over the structure's atoms.
//
//   s_ij = scale q_i . k_j;  s <- cap tanh(s / cap);  s <- s - slope_h |r_i - r_j|
//   p_ij = softmax over the visible keys j of i's structure,  o_i = sum_j p_ij v_j
//
// Gradient, with D_i = sum_j p_ij (go_i . v_j):
//
//   dz_ij = p_ij (go_i . v_j - D_i)                     of the biased score
//   ds_ij = dz_ij (1 - tanh^2)                          of the scaled product
//   dq_i = scale sum_j ds_ij k_j,  dk_j = scale sum_i ds_ij q_i,  dv_j = sum_i p_ij go_i
//   dslope_h = -sum_ij dz_ij |r_i - r_j|,  dr_i = -slope sum_j dz_ij (r_i - r_j) / |r_i - r_j|  (and its negative to r_j)
//
// Query heads that share a key head are rows of one problem: row r of a key
// head is token r / G of query head r % G of its group.  A wave owns 32 rows
// (32 keys in the key-side gradient) and takes the other axis in tiles that the
// workgroup stages in LDS.  All products run on the 32 x 32 matrix
// instructions, bf16 x bf16 -> fp32 or fp32 x fp32 -> fp32, transposed so that
// a lane holds one row's (key's) values: lane l has column l % 32 and, in
// register 4 b + j, line 8 b + 4 (l / 32) + j.  Softmax statistics are then a
// lane's own but for one exchange between the two half waves, and the same
// registers are the operand of the next product, whose contraction order is
// chosen to fit them.
//
// Scores, the running maximum and sum, and every sum over keys or rows are
// fp32.  bf16 calls round p and ds to bf16 for the matrix instruction (at most
// 2^-8 relative each, as the inputs are) and each output once.
#pragma once

#include <type_traits>

#include "rows.h"

namespace ye3t {
namespace attention {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

constexpr double kLog2eExact = 1.4426950408889634;
constexpr float kLog2e = float(kLog2eExact);
constexpr float kLn2 = 0.6931471805599453f;
// Atoms whose squared distance is below the smallest normal float are at one place: the
// reciprocal root takes no subnormal value.
constexpr float kLeastSquare = 1.17549435e-38f;
// A squared distance past the largest float is infinite, and so is the distance that scores are lowered
// by: such atoms do not see each other.  Gradients take the distance as square times
// reciprocal root, which has to be a number.
constexpr float kMostSquare = 3.40282347e38f;

struct Problem {
  int64_t queries, keys, structures;
  int heads, key_heads, group, group_shift, D;  // group_shift: -1 where group is no power of two
  bool direct;  // rows, heads and width are whole aligned chunks of 16 bytes
  const void *q, *k, *v;
  int64_t q_row, q_head, k_row, k_head, v_row, v_head;
  const int64_t *offsets, *key_offsets;
  float scale, cap;
  float to_log2, to_bend, from_bend;  // of scores: scale in units of log2; the same of 2 / cap; cap in units of log2
  const float *slopes, *positions, *key_positions;
  const uint8_t* key_mask;
};

// 16 bytes of a lane as matrix operand: 8 bf16 or 4 fp32 values
template <typename T>
struct Operand;
template <>
struct Operand<__bf16> {
  typedef bf16x8 type;
};
template <>
struct Operand<float> {
  typedef f32x4 type;
};
template <typename T>
using Op = typename Operand<T>::type;

// c += a b over the 2 kChunk contraction slots of one operand: slot
// (half wave, element)
__device__ inline void mma(bf16x8 a, bf16x8 b, f32x16& c) {
  c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ inline void mma(f32x4 a, f32x4 b, f32x16& c) {
#pragma unroll
  for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[j], c, 0, 0, 0);
}

__device__ inline f32x16 zeros() {
  f32x16 z;
#pragma unroll
  for (int i = 0; i < 16; ++i) z[i] = 0.0f;
  return z;
}

// The same value; with FRESH unknown to the compiler, so that addresses made from it in
// a loop are formed there, a few operations a tile, instead of being held in
// registers.  For short structures, a tile or two a wave, where more waves count
// for more: 2 000 molecules of 21 atoms, fp32, gradients 205 -> 182 us; structures of 480 atoms
// 658 -> 698.
template <bool FRESH>
__device__ inline unsigned anew(unsigned v) {
  if (FRESH) asm volatile("" : "+v"(v));
  return v;
}

// A tile of lines in LDS: DP values each without padding, because the loads that
// go straight to LDS write a wave's 64 chunks of 16 bytes one after the other.  Chunk c
// of line l lies at place c ^ turn(l) of its line.  LDS serves 256 bytes a cycle from 64
// banks: 16 lanes of a 16 byte read, which are one chunk of 16 lines, or 32 of a
// transposing one, four chunks of four lines; turn() puts either into different banks (with
// turns that repeat after eight lines 44 % of the LDS cycles were conflicts).
template <typename T, int DP>
__device__ inline int turn(int line) {
  constexpr int BYTES = DP * int(sizeof(T)), PER = BYTES >= 256 ? 1 : 256 / BYTES;  // lines in 256 bytes
  return (line & 3) / PER * 4 | (line >> 2 & 3);
}

// Contraction over the width: chunk u of line `line` holds values
// 2 kChunk u + kChunk half ...
template <typename T, int DP>
__device__ inline Op<T> line_chunk(const T* tile, int line, int u, int half) {
  return *reinterpret_cast<const Op<T>*>(tile + line * DP + ((2 * u + half) ^ turn<T, DP>(line)) * kChunk<T>);
}

// Contraction over 32 lines of a tile, the transposed operand: column `column`
// + lane % 32 of the lines that registers 2 kChunk s / 2 ... of an accumulator
// hold (bf16: lines 16 s + 4 half + 0..3 and + 8; fp32: lines 8 s + 4 half + 0..3).
// bf16: the transposing LDS read, where lane l of a block of 16 gives the address
// of four values of line l / 4, columns 4 (l % 4) .. + 3, and gets four lines of
// column l.  Every lane of the wave takes part.
template <int DP>
__device__ inline bf16x8 column_chunk(const __bf16* tile, int s, int column, unsigned lane) {
  typedef short s16x4 __attribute__((ext_vector_type(4)));
  typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
  const int line = int(lane / 32 * 4 + (lane & 15) / 4);  // turn() repeats 16 lines on
  const int chunk = column / 8 + int((lane & 16) / 8 + (lane & 3) / 2);
  const __bf16* at = tile + (16 * s + line) * DP + 4 * int(lane & 1);
  const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(at + (chunk ^ turn<__bf16, DP>(line)) * 8));
  const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(at + 8 * DP + (chunk ^ turn<__bf16, DP>(line + 8)) * 8));
  typedef short s16x8 __attribute__((ext_vector_type(8)));
  const s16x8 both = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
  return __builtin_bit_cast(bf16x8, both);
}
template <int DP>
__device__ inline f32x4 column_chunk(const float* tile, int s, int column, unsigned lane) {
  // turn() of line 8 s + 4 half + j, with what the lane adds to it apart from what s and j do: four
  // addresses serve all of a tile
  const int half = int(lane / 32), at = int(lane & 31), own = at / 4 ^ half;
  f32x4 r;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int flip = (DP == 32 ? j / 2 : j & 1) * 4 + 2 * (s & 1), across = DP == 32 ? 0 : column / 32 ^ j / 2;
    const float* from = tile + 4 * half * DP + (own ^ flip) * 4 + (at & 3);
    r[j] = from[(8 * s + j) * DP + 32 * across];
  }
  return r;
}
// and the accumulator's registers as the other operand
__device__ inline void register_chunk(const f32x16& p, int s, bf16x8& r) {
#pragma unroll
  for (int j = 0; j < 8; ++j) r[j] = __bf16(p[8 * s + j]);
}
__device__ inline void register_chunk(const f32x16& p, int s, f32x4& r) {
#pragma unroll
  for (int j = 0; j < 4; ++j) r[j] = p[4 * s + j];
}
template <typename T>
constexpr int kLineChunks = 32 / (2 * kChunk<T>);

// Keeps what follows from being started before what precedes.  Left alone, the
// compiler reads all operands of a tile from LDS first, which takes more
// registers than the products leave.
__device__ inline void in_turn() { __builtin_amdgcn_sched_barrier(0); }

// use(i, load(i)) for i < N with the loads kept DEPTH steps ahead.
template <int N, int DEPTH = 2, typename Load, typename Use>
__device__ inline void in_flight(Load load, Use use) {
  decltype(load(0)) held[DEPTH + 1];
#pragma unroll
  for (int i = 0; i < DEPTH && i < N; ++i) held[i] = load(i);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (i + DEPTH < N) held[(i + DEPTH) % (DEPTH + 1)] = load(i + DEPTH);
    use(i, held[i % (DEPTH + 1)]);
    in_turn();
  }
}
template <typename T>
struct Two {
  Op<T> a, b;
};
template <typename T>
struct Three {
  Op<T> a, b, c;
};

// An operand of a wave's own 32 lines, kept in LDS instead of registers: rows of 128 in
// bf16 then leave room for two waves a SIMD.  Only the wave itself reads it.
template <typename T, int DP>
__device__ inline void keep_lines(T* tile, const Op<T>* r, int lane) {
#pragma unroll
  for (int u = 0; u < DP / (2 * kChunk<T>); ++u)
    *reinterpret_cast<Op<T>*>(tile + (lane & 31) * DP + ((2 * u + lane / 32) ^ turn<T, DP>(lane & 31)) * kChunk<T>) = r[u];
}
template <typename T, int DP, int NW>
constexpr bool kKeepLines = sizeof(T) == 2 && DP == 128 && NW == 4;

// tanh in the form the kernels use it: t = 1 - 2 r with r = 1 / (exp(2 x) + 1), and
// 1 - t^2 = 4 (r - r^2).  r is good to 2e-7 of 1, and capped scores to 2e-7 of the cap: for caps up to
// kLargestRoughCap 2e-4, a twentieth of the rounding of their weights to bf16.  Larger
// caps and fp32 calls (FINE) take t from its odd series for small x, for a relative error
// of t of a few ulp (the first term left out is 4e-3 x^13).
// No branches: a lane's choice between two short formulas costs less than leaving one out.
// `exponent` is 2 x in units of log2.
struct Bend {
  float t, r;
};
template <bool FINE>
__device__ inline Bend bend_of(float exponent) {
  const float r = __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(exponent) + 1.0f);
  Bend b = {1.0f - 2.0f * r, r};
  if (FINE) {
    const float x = exponent * (0.5f * kLn2), y = x * x;
    const float series =
        x + x * y * (-0.333333333f + y * (0.133333333f + y * (-0.0539682540f + y * (0.0218694885f + y * -0.00886323552f))));
    b.t = y < 0.09f ? series : b.t;
  }
  return b;
}

// How scores are capped: not at all, or by which form of tanh.  96 structures of 480 atoms, 8
// heads of 64, bf16, distances and mask, forward and gradients: 849 us rough, 999 fine.
enum Cap { kNoCap, kRoughCap, kFineCap };
constexpr float kLargestRoughCap = 1024.0f;

// The largest d with bound(d) <= slot, bound rising, bound(0) <= slot: 64 probes a round.
template <typename F>
__device__ inline int64_t find_owner(int64_t count, int64_t slot, F bound) {
  int64_t lo = 0, hi = count;
  const int lane = threadIdx.x & 63;
  while (hi - lo > 1) {
    const int64_t step = (hi - lo + 63) / 64;
    const int64_t at = lo + lane * step;
    const uint64_t yes = __ballot(at < hi && bound(at) <= slot);
    const int k = 63 - __clzll(static_cast<long long>(yes | 1));
    lo += k * step;
    hi = lo + step < hi ? lo + step : hi;
  }
  return lo;
}

// The rows or keys of a structure; offsets out of range are clamped, so that no
// access leaves the arrays whatever they hold.
struct Span {
  int64_t begin;
  int length;
};
__device__ inline int64_t clamped(int64_t v, int64_t most) { return v < 0 ? 0 : v > most ? most : v; }
__device__ inline Span span_of(const int64_t* offsets, int64_t d, int64_t most) {
  const int64_t a = clamped(offsets[d], most), b = clamped(offsets[d + 1], most);
  return {a, b > a ? int(b - a) : 0};
}

// Work items of `tile` rows over structures of any lengths without a table of
// them: structure d's items start at floor(offset_d G / tile) + d, which leaves
// room for each; an item past its structure's rows has nothing to do.
struct Item {
  int64_t structure;
  int64_t first;  // row in the structure
};
__device__ inline Item item_of(const int64_t* offsets, int64_t structures, int64_t most, int group, int tile,
                               int64_t slot) {
  auto bound = [&](int64_t d) { return clamped(offsets[d], most) * group / tile + d; };
  const int64_t d = find_owner(structures, slot, bound);
  return {d, (slot - bound(d)) * tile};
}
inline int64_t item_count(int64_t rows, int64_t structures, int tile) { return rows / tile + structures; }

// ---- loads of a tile ---------------------------------------------------------
__device__ __align__(16) const uint32_t kZeros[4] = {0, 0, 0, 0};

// LINES x DP values of `T` by NT threads into a tile, while another tile is used.  Where
// every chunk is 16 whole aligned bytes (`direct`) memory is loaded straight to LDS
// without passing registers; otherwise chunk by chunk through them.  address(line): the
// line's first value, or null for a line of zeros.  arrived() waits for the loads of this wave.
template <typename T, int DP, int LINES, int NT, bool FRESH, typename F>
__device__ inline void load_tile(T* tile, int D, bool direct, F address) {
  constexpr int ROW = DP / kChunk<T>, SLOTS = LINES * ROW;
  const int wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) >> 6), thread = int(anew<FRESH>(threadIdx.x) & 255);
  auto each = [&](auto use) {
#pragma unroll
    for (int n = 0; n < (SLOTS + NT - 1) / NT; ++n) {
      if (SLOTS % NT != 0 && n * NT + 64 * wave >= SLOTS) continue;  // 64 divides SLOTS
      const int x = n * NT + thread, line = x / ROW, c = (x % ROW ^ turn<T, DP>(line)) * kChunk<T>;
      const T* p = address(line);
      use(n, x, c, p && c < D ? p + c : nullptr);
    }
  };
  if (direct) {
    each([&](int n, int, int, const T* p) {
      __builtin_amdgcn_global_load_lds(
          (const __attribute__((address_space(1))) void*)(p ? p : reinterpret_cast<const T*>(kZeros)),
          (__attribute__((address_space(3))) void*)(tile + (n * NT + 64 * wave) * kChunk<T>), 16, 0, 0);
    });
  } else {
    each([&](int, int x, int c, const T* p) {
      const Chunk<T, kChunk<T>> v = p ? Chunk<T, kChunk<T>>::load(p, D - c) : Chunk<T, kChunk<T>>::zero();
      Op<T> a;
#pragma unroll
      for (int q = 0; q < kChunk<T>; ++q) a[q] = v.v[q];
      *reinterpret_cast<Op<T>*>(tile + x * kChunk<T>) = a;
    });
  }
}
__device__ inline void arrived() { __builtin_amdgcn_s_waitcnt(0x0f70); }  // vmcnt(0)

// A row or key as matrix operand, straight from memory: chunks of this lane's half
template <typename T, int DP>
__device__ inline void line_operand(const T* p, int D, int half, Op<T>* r) {
#pragma unroll
  for (int u = 0; u < DP / (2 * kChunk<T>); ++u) {
    const int c = (2 * u + half) * kChunk<T>;
    const Chunk<T, kChunk<T>> a = p && c < D ? Chunk<T, kChunk<T>>::load(p + c, D - c) : Chunk<T, kChunk<T>>::zero();
#pragma unroll
    for (int q = 0; q < kChunk<T>; ++q) r[u][q] = a.v[q];
  }
}

// Values of lines 8 b + 4 half + j, column lane % 32, to memory: line = value of
// the width, the lane's row at `p` (null: none).
template <typename T, int DP>
__device__ inline void store_columns(T* p, int D, int half, const f32x16* acc, float factor) {
  if (!p) return;
#pragma unroll
  for (int t = 0; t < DP / 32; ++t) {
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      const int c = 32 * t + 8 * b + 4 * half;
      Chunk<T, 4> a;
#pragma unroll
      for (int j = 0; j < 4; ++j) a.v[j] = T(acc[t][4 * b + j] * factor);
      if (c < D) a.store(p + c, D - c);
    }
  }
}

__device__ inline float other_half(float v) { return __shfl_xor(v, 32); }

// key: x, y, z, and what its scores are raised by: 0, or -infinity where it is
// not seen
template <bool BIAS>
__device__ inline f32x4 key_place(const Problem& p, int64_t key, bool seen) {
  f32x4 r = {0.0f, 0.0f, 0.0f, seen ? 0.0f : -INFINITY};
  if (BIAS && seen) {
    const float* at = (p.key_positions ? p.key_positions : p.positions) + 3 * key;
    r[0] = at[0];
    r[1] = at[1];
    r[2] = at[2];
  }
  return r;
}

// The keys of a structure in tiles of KT <= 64.  take() makes one ready for the
// workgroup; with two buffers the next one's loads run meanwhile.  One buffer where a
// workgroup is one wave: more of them fit a compute unit's LDS, and they hide each other's
// loads (one row against 9 000 atoms in each of 24 structures 150 -> 120 us).  Whether a key is seen is read a tile ahead of its
// rows; masked keys have rows of zeros, whatever they hold.
template <typename T, int DP, int KT, int NT, int BUFFERS, bool FRESH, bool BIAS>
struct KeyTiles {
  const Problem& p;
  const Span key;
  const T *kbase, *vbase;
  T *ktiles, *vtiles;
  f32x4* places;
  f32x4 place;
  uint8_t mask;  // of this lane's key in the tile after the one begun last, as it was read
  bool any = false;  // a key of the tiles begun so far is seen: the same in all lanes and waves

  __device__ static inline int buffer(int tile) { return BUFFERS == 2 ? tile & 1 : 0; }
  __device__ inline const T* keys(int tile) const { return ktiles + buffer(tile) * KT * DP; }
  __device__ inline const T* values(int tile) const { return vtiles + buffer(tile) * KT * DP; }
  __device__ inline const f32x4* places_of(int tile) const { return places + buffer(tile) * KT; }

  __device__ inline bool exists(int tile) const {
    return (int(threadIdx.x) & 63) < KT && tile * KT + (int(threadIdx.x) & 63) < key.length;
  }
  __device__ inline void look(int tile) {
    mask = 1;
    if (p.key_mask && exists(tile)) mask = p.key_mask[key.begin + tile * KT + (int(threadIdx.x) & 63)];
  }
  __device__ inline void start(int tile) {
    look(tile);
    if (BUFFERS == 2) begin(tile);
  }
  // Nothing here uses what it loads: a wait would be for the tile's rows too.
  __device__ inline void begin(int tile) {
    const bool seen = exists(tile) && mask;
    const uint64_t all = __ballot(seen);
    any |= all != 0;
    const int64_t first = key.begin + int64_t(tile) * KT;
    load_tile<T, DP, KT, NT, FRESH>(ktiles + buffer(tile) * KT * DP, p.D, p.direct,
                             [&](int line) { return all >> line & 1 ? kbase + (first + line) * p.k_row : nullptr; });
    load_tile<T, DP, KT, NT, FRESH>(vtiles + buffer(tile) * KT * DP, p.D, p.direct,
                             [&](int line) { return all >> line & 1 ? vbase + (first + line) * p.v_row : nullptr; });
    if (int(threadIdx.x) < KT) place = key_place<BIAS>(p, first + threadIdx.x, seen);
    look(tile + 1);
  }
  __device__ inline void take(int tile, int tiles) {
    if (BUFFERS == 1) {
      __syncthreads();  // the last tile has been used
      begin(tile);
    }
    if (int(threadIdx.x) < KT) places[buffer(tile) * KT + threadIdx.x] = place;
    arrived();
    __syncthreads();
    if (BUFFERS == 2 && tile + 1 < tiles) begin(tile + 1);
  }
};

struct Row {
  int64_t token;
  int head;
  bool exists;
};
__device__ inline Row row_of(const Problem& p, int64_t begin, int64_t row, int64_t rows, int key_head) {
  Row r;
  r.exists = row < rows;
  const uint32_t x = r.exists ? uint32_t(row) : 0u;
  const uint32_t token = p.group_shift >= 0 ? x >> p.group_shift : x / uint32_t(p.group);
  r.token = begin + token;
  r.head = key_head * p.group + int(x - token * uint32_t(p.group));
  return r;
}

struct Gradient {
  const void *out, *adjoint;  // [queries, heads, D]
  bool direct;                // the adjoint's rows are whole aligned chunks of 16 bytes
  const float* log_sums;      // [queries, heads]
  float* along;               // D_i, [queries, heads]
  void *dq, *dk, *dv;         // [queries, heads, D], [keys, key_heads, D]
  float* row_part;            // [queries, heads, 4]: to the position and the slope
  float* key_part;            // [keys, key_heads, 4]
  float* sum_part;            // [key_parts, 2, keys, key_heads, D]: dk and dv of the parts of the row axis
};

// Scores in units of log2 as the forward takes them, and the derivative of the
// bend, over 4 (slant_scale()); the distance is subtracted by the caller.
struct Score {
  float s, slant;
};
template <Cap CAP>
__device__ inline Score score_of(const Problem& p, float product) {
  if (CAP != kNoCap) {
    const Bend b = bend_of<CAP == kFineCap>(product * p.to_bend);
    return {p.from_bend * b.t, b.r - b.r * b.r};
  }
  return {product * p.to_log2, 1.0f};
}
template <Cap CAP>
__host__ __device__ constexpr float slant_scale() {
  return CAP != kNoCap ? 4.0f : 1.0f;
}

// Waves a SIMD that the register budget is set for: spills cost more than a wave gains.
template <typename T, int DP, int NW>
constexpr int kForwardWaves =
    DP == 32 ? (NW == 1 ? 4 : 3) : DP == 64 ? (sizeof(T) == 4 && NW == 1 ? 2 : 3) : sizeof(T) == 2 ? 2 : 1;
template <typename T, int DP, int NW>
constexpr int kGradientWaves = DP == 32 ? (NW == 1 ? 3 : 2) : DP == 64 || kKeepLines<T, DP, NW> ? 2 : 1;

inline int64_t up(int64_t bytes) { return (bytes + 255) / 256 * 256; }

// Waves of a workgroup: one where the mean structure has rows for one only, four
// otherwise.  2 000 molecules of 21 atoms with forces 48 + 173 us by one, 88 + 419 by four; one
// row against 9 000 atoms in each of 24 structures 106 and 153; 96 structures of 480 atoms 250 +
// 744 by one, 206 + 645 by four, 40 of 1 000 in fp32 1 307 and 971.
inline int waves_for(int64_t rows, int64_t structures) {
  const int64_t mean = structures > 0 ? (rows + structures - 1) / structures : 0;
  return mean <= 32 ? 1 : 4;
}

// Parts of the key axis: where the rows alone give less than four workgroups
// a compute unit, as many as make eight, each with two tiles of 32 keys or more on
// average, 64 at most (a lane each where they are joined).  24 structures of 9 000
// atoms, one row each, 16 heads of 128 over 4 key heads, bf16, before the parts were
// joined a lane each: 120 us, 136 by twice as many.
inline int parts_for(int64_t items, int key_heads, int64_t keys, int64_t structures) {
  const int64_t groups = items * key_heads;
  if (groups >= 1024 || structures == 0) return 1;
  int64_t parts = 2048 / groups;
  const int64_t tiles = keys / structures / 64;
  if (parts > tiles) parts = tiles;
  return int(parts < 1 ? 1 : parts > 64 ? 64 : parts);
}

struct ForwardPlan {
  int waves, parts;
  int64_t items, part_bytes, bytes;
};
inline ForwardPlan forward_plan(const ye3t_attention_args& a) {
  ForwardPlan f{};
  const int64_t group = a.heads / a.key_heads;
  f.waves = waves_for(a.queries * group, a.structures);
  f.items = item_count(a.queries * group, a.structures, 32 * f.waves);
  f.parts = parts_for(f.items, int(a.key_heads), a.keys, a.structures);
  if (f.parts > 1) {
    f.part_bytes = up(f.parts * a.queries * a.heads * a.head_width * 4);
    f.bytes = f.part_bytes + up(f.parts * a.queries * a.heads * 8);
  }
  return f;
}

// workgroups that share the sum over atoms of a slope's gradient
constexpr int kSlopeGroups = 64;

struct AdjointPlan {
  int row_waves, key_waves, key_parts;
  int64_t row_items, key_items, along_bytes, row_bytes, key_bytes, slope_bytes, sum_bytes, bytes;
};
inline AdjointPlan adjoint_plan(const ye3t_attention_args& a, bool forces) {
  AdjointPlan f{};
  const int64_t group = a.heads / a.key_heads;
  f.row_waves = waves_for(a.queries * group, a.structures);
  f.key_waves = waves_for(a.keys, a.structures);
  f.row_items = item_count(a.queries * group, a.structures, 32 * f.row_waves);
  f.key_items = item_count(a.keys, a.structures, 32 * f.key_waves);
  f.along_bytes = up(a.queries * a.heads * 4);
  f.key_parts = 1;
  if (forces) {
    f.row_bytes = up(a.queries * a.heads * 16);
    f.key_bytes = up(a.keys * a.key_heads * 16);
    f.slope_bytes = up(kSlopeGroups * a.heads * 4);
  } else if (a.structures > 0) {
    // Keys that give less than two workgroups a compute unit: the row axis in parts of
    // eight tiles or more on average, summed by attention_key_join_kernel.
    const int64_t groups = f.key_items * a.key_heads, tiles = a.queries * group / a.structures / 256;
    const int64_t parts = groups < 512 ? 1024 / groups : 1;
    f.key_parts = int(parts < tiles ? (parts < 16 ? parts : 16) : tiles < 1 ? 1 : tiles < 16 ? tiles : 16);
    if (f.key_parts > 1) f.sum_bytes = up(f.key_parts * 2 * a.keys * a.key_heads * a.head_width * 4);
  }
  f.bytes = f.along_bytes + f.row_bytes + f.key_bytes + f.slope_bytes + f.sum_bytes + 256;
  return f;
}

inline Problem problem_of(const ye3t_attention_args& a) {
  Problem p{};
  p.queries = a.queries;
  p.keys = a.keys;
  p.structures = a.structures;
  p.heads = int(a.heads);
  p.key_heads = int(a.key_heads);
  p.group = int(a.heads / a.key_heads);
  p.group_shift = -1;
  for (int k = 0; k < 16; ++k)
    if (p.group == 1 << k) p.group_shift = k;
  p.D = int(a.head_width);
  const int64_t chunk = a.dtype == YE3T_F32 ? kChunk<float> : kChunk<__bf16>;
  const uintptr_t bases = reinterpret_cast<uintptr_t>(a.query) | reinterpret_cast<uintptr_t>(a.key) |
                          reinterpret_cast<uintptr_t>(a.value);
  p.direct = a.head_width % chunk == 0 && bases % 16 == 0 && a.query_row_stride % chunk == 0 &&
             a.query_head_stride % chunk == 0 && a.key_row_stride % chunk == 0 && a.key_head_stride % chunk == 0 &&
             a.value_row_stride % chunk == 0 && a.value_head_stride % chunk == 0;
  p.q = a.query;
  p.k = a.key;
  p.v = a.value;
  p.q_row = a.query_row_stride;
  p.q_head = a.query_head_stride;
  p.k_row = a.key_row_stride;
  p.k_head = a.key_head_stride;
  p.v_row = a.value_row_stride;
  p.v_head = a.value_head_stride;
  p.offsets = a.offsets;
  p.key_offsets = a.key_offsets ? a.key_offsets : a.offsets;
  p.scale = float(a.scale);
  p.to_log2 = float(a.scale * kLog2eExact);
  if (a.cap > 0.0) {
    // Held to what fp32 has room for: scores below 1e-30 are equal, and 1e30 caps none below 3e26.
    const double cap = a.cap < 1e-30 ? 1e-30 : a.cap > 1e30 ? 1e30 : a.cap, to_bend = 2.0 * kLog2eExact * a.scale / cap;
    p.cap = float(cap);
    p.to_bend = to_bend > 1e38 ? 1e38f : to_bend < -1e38 ? -1e38f : float(to_bend);
    p.from_bend = float(cap * kLog2eExact);
  }
  p.slopes = a.slopes;
  p.positions = a.positions;
  p.key_positions = a.key_positions;
  p.key_mask = a.key_mask;
  return p;
}

inline int check_attention(const ye3t_attention_args& a) {
  YE3T_REQUIRE(a.queries >= 0 && a.keys >= 0 && a.structures >= 0, "atom and structure counts must not be negative");
  YE3T_REQUIRE(a.heads >= 1 && a.key_heads >= 1 && a.heads % a.key_heads == 0,
               "heads must be a positive multiple of key_heads");
  YE3T_REQUIRE(a.head_width >= 1, "head_width must be positive");
  if (a.head_width > 128) return set_error(YE3T_EUNSUPPORTED, "head_width %lld is above 128", (long long)a.head_width);
  if (a.dtype != YE3T_F32 && a.dtype != YE3T_BF16)
    return set_error(YE3T_EDTYPE, "unsupported dtype %d; expected float32 or bfloat16", a.dtype);
  // Rows, keys and tiles of one structure are counted in 32 bits.  The first row past the last tile,
  // and the tile looked at ahead of it, are at most 255 on.
  constexpr int64_t most = (int64_t(1) << 31) - 256;
  YE3T_REQUIRE(a.heads <= 65535 && a.queries <= most / a.heads && a.keys <= most / a.heads &&
                   a.structures < (int64_t(1) << 24),
               "at most 2^31 - 256 rows (atoms times heads), 65535 heads and 2^24 - 1 structures");
  YE3T_REQUIRE(a.cap >= 0.0, "cap must not be negative");
  // arrays without values may be null
  YE3T_REQUIRE(a.queries == 0 || (a.slopes == nullptr) == (a.positions == nullptr), "slopes and positions come together");
  YE3T_REQUIRE(!a.slopes || a.keys == 0 || a.key_positions || (!a.key_offsets && a.queries == a.keys),
               "keys of their own need key_positions");
  YE3T_REQUIRE(a.key_offsets || a.queries == a.keys, "keys of their own need key_offsets");
  return YE3T_OK;
}

inline int check_pointers(const ye3t_attention_args& a) {
  YE3T_REQUIRE(a.structures == 0 || a.offsets, "attention needs the structures' offsets");
  YE3T_REQUIRE((a.queries == 0 || a.query) && (a.keys == 0 || (a.key && a.value)), "attention needs query, key and value");
  return YE3T_OK;
}

// Calls f.template operator()<T, DP>() for the call's type and width.
template <typename F>
int with_width(int dtype, int64_t D, F f) {
  if (dtype == YE3T_F32)
    return D <= 32 ? f.template operator()<float, 32>()
                   : D <= 64 ? f.template operator()<float, 64>() : f.template operator()<float, 128>();
  return D <= 32 ? f.template operator()<__bf16, 32>()
                 : D <= 64 ? f.template operator()<__bf16, 64>() : f.template operator()<__bf16, 128>();
}

// Calls f with the call's Cap as a type; fp32 calls are fine ones.
template <typename T, typename F>
int with_cap(const Problem& p, F f) {
  if (p.cap <= 0.0f) return f(std::integral_constant<Cap, kNoCap>());
  if constexpr (sizeof(T) == 2)
    if (p.cap <= kLargestRoughCap) return f(std::integral_constant<Cap, kRoughCap>());
  return f(std::integral_constant<Cap, kFineCap>());
}

// The gradient's two sides (attention_rows.hip, attention_keys.hip)
int launch_row_gradient(int dtype, const AdjointPlan& f, const Problem& p, const Gradient& g, bool forces,
                        hipStream_t s);
int launch_key_gradient(int dtype, const AdjointPlan& f, const Problem& p, const Gradient& g, bool forces,
                        hipStream_t s);

}  // namespace attention
}  // namespace ye3t
