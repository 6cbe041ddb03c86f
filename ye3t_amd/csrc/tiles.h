// Tiles of matrix operands in LDS, and work items over packed groups of rows.
#pragma once

#include "rows.h"

namespace ye3t {
namespace tiles {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

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

__device__ inline f32x16 zeros() {
  f32x16 z;
#pragma unroll
  for (int i = 0; i < 16; ++i) z[i] = 0.0f;
  return z;
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

// Keeps what follows from being started before what precedes.  Left alone, the
// compiler reads all operands of a tile from LDS first, which takes more
// registers than the products leave.
__device__ inline void in_turn() { __builtin_amdgcn_sched_barrier(0); }

__device__ __align__(16) const uint32_t kZeros[8] = {0, 0, 0, 0, 0, 0, 0, 0};

__device__ inline void arrived() { __builtin_amdgcn_s_waitcnt(0x0f70); }  // vmcnt(0)


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

}  // namespace tiles
}  // namespace ye3t
