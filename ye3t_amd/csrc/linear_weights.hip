// The gradient to weights and biases: products over the rows of each group.
//
// A workgroup owns a tile of one weight over a share of its group's rows; both operands run across the contraction
// and are turned by the reads of LDS.  Groups of several shares leave their sums in fp32 in a workspace, and a second
// kernel adds them in order: no atomics, equal calls give equal bits.  The bias's gradient is summed from the tiles in
// LDS.  Bound by the matrix instructions: 16 384 rows, 1 024 x 4 096, bf16, 142 us (967 TFLOP/s), with the bias 168; fp32,
// 1 024 x 1 024, 215 us (160 TFLOP/s), half of the cycles matrix and a third vector instructions that split the values.
#include "linear.h"

namespace ye3t {
namespace linear {
namespace {

template <typename T, typename S, bool DIRECT>
__global__ __launch_bounds__(S::NT, S::kPerSimd) void weight_product_kernel(const WeightProduct<T> p) {
  typedef Tile<T, S::TM, S::KT, true> A;
  typedef Tile<T, S::TN, S::KT, true> B;
  static_assert(S::TM == S::TN, "either operand's columns can be summed");
  constexpr int STEP = A::kBytes + B::kBytes;
  constexpr int LDS = S::BUFFERS * STEP > S::kOutBytes || DIRECT ? S::BUFFERS * STEP : S::kOutBytes;
  __shared__ __align__(256) char lds[LDS];
  const int lane = int(threadIdx.x) & 63, wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) >> 6);
  const int wn = wave % S::WN, wm = wave / S::WN % S::WM, wk = wave / (S::WN * S::WM);

  const int64_t tiles = int64_t(p.tiles_m) * p.tiles_n;
  int64_t slot, tile;
  if (p.spread) {  // every XCD takes its part of each slot's tiles
    const int64_t per = (tiles + 7) / 8;
    slot = blockIdx.x / 8 / per;
    tile = (blockIdx.x & 7) * per + blockIdx.x / 8 % per;
    if (tile >= tiles) return;
  } else {
    const int64_t x = p.grouped ? int64_t(blockIdx.x) : tile_of_group();
    slot = x / tiles;
    tile = x % tiles;
  }
  const int tile_m = int(tile / p.tiles_n), tile_n = int(tile % p.tiles_n);
  const int m0 = tile_m * S::TM, n0 = tile_n * S::TN;
  int64_t group = 0, begin = 0, first = slot * p.share, length = p.rows;
  if (p.grouped) {
    auto bound = [&](int64_t d) { return clamped(p.offsets[d], p.rows) / p.share + d; };
    group = find_owner(p.groups, slot, bound);
    first = (slot - bound(group)) * p.share;
    begin = clamped(p.offsets[group], p.rows);
    length = clamped(p.offsets[group + 1], p.rows) - begin;
  }
  if (first && first >= length) return;  // the first share of a group without rows writes its zeros
  const int64_t row0 = begin + first;
  const int64_t left = length - first;
  const int live = int(left < 0 ? 0 : left < p.share ? left : p.share);

  auto tile_a = [&](int t) { return reinterpret_cast<__bf16*>(lds + t % S::BUFFERS * STEP); };
  auto tile_b = [&](int t) { return reinterpret_cast<__bf16*>(lds + t % S::BUFFERS * STEP + A::kBytes); };
  f32x16 sum[S::FM][S::FN];
#pragma unroll
  for (int i = 0; i < S::FM; ++i)
#pragma unroll
    for (int j = 0; j < S::FN; ++j) sum[i][j] = zeros();
  // column sums of one operand, by the workgroups of its first tile of the other
  const bool summing = p.sums && (p.sums_of_a ? tile_n == 0 : tile_m == 0);
  constexpr int ACROSS = S::TM / 8, DOWN = S::NT / ACROSS;
  float column[8];
#pragma unroll
  for (int q = 0; q < 8; ++q) column[q] = 0.0f;
  auto add_columns = [&](int t) {
    if (!summing) return;
    const __bf16* from = p.sums_of_a ? tile_a(t) : tile_b(t);
    const int c = int(threadIdx.x) % ACROSS;
    for (int k = int(threadIdx.x) / ACROSS; k < S::KT; k += DOWN) {
      float v[8];
#pragma unroll
      for (int q = 0; q < 8; ++q) v[q] = 0.0f;
#pragma unroll
      for (int n = kParts<T> - 1; n >= 0; --n) {
        const __bf16* at = from + n * A::kValues + k * S::TM + (c ^ turn<__bf16, S::TM>(k)) * 8;
        const bf16x8 part = *reinterpret_cast<const bf16x8*>(at);
#pragma unroll
        for (int q = 0; q < 8; ++q) v[q] += float(part[q]);
      }
#pragma unroll
      for (int q = 0; q < 8; ++q) column[q] += v[q];
    }
  };

  const int steps = (live + S::KT - 1) / S::KT;
  // rows of this thread's chunks, the same for both operands, of the tile that is loaded next; -1: none
  constexpr int EACH = (A::kChunks + S::NT - 1) / S::NT;
  int64_t row[EACH];
  auto look = [&](int t) {
#pragma unroll
    for (int n = 0; n < EACH; ++n) {
      const int k = t * S::KT + A::line_of(n * S::NT + int(threadIdx.x));
      row[n] = k < live ? row_at(p.order, row0 + k, p.rows) : -1;
    }
  };
  look(0);
  if constexpr (DIRECT) {
    // Columns past the weight's repeat others: their results go nowhere.
    DirectLoads<S::TM, S::KT, true, S::NT> a;
    DirectLoads<S::TN, S::KT, true, S::NT> b;
    static_assert(decltype(a)::kEach == EACH, "both operands' chunks are of the same rows");
    auto load = [&](int t, auto part, auto parts) {
      constexpr int P = decltype(part)::value, OF = decltype(parts)::value;
#pragma unroll
      for (int n = EACH * P / OF; n < EACH * (P + 1) / OF; ++n) {
        const int c = a.column_of(n);
        a.load(tile_a(t), n, wave, row[n] < 0 ? a.none() : p.a + row[n] * p.a_row + (m0 + c < p.M ? m0 + c : 0));
        b.load(tile_b(t), n, wave, row[n] < 0 ? b.none() : p.b + row[n] * p.b_row + (n0 + c < p.N ? n0 + c : 0));
      }
      if (P + 1 == OF) look(t + 1);
    };
    multiply_direct<S, A, B, 2 * EACH, false>(steps, 0, tile_a, tile_b, wm, wn, wk, lane, load, add_columns, sum);
  } else {
    Loads<T, S::TM, S::KT, true, S::NT> a;
    Loads<T, S::TN, S::KT, true, S::NT> b;
    const bool whole_columns = m0 + S::TM <= p.M && n0 + S::TN <= p.N;
    auto load = [&](int t) {
      const T *a_from[EACH], *b_from[EACH];
#pragma unroll
      for (int n = 0; n < EACH; ++n) {
        const int64_t r = row[n] < 0 ? 0 : row[n];
        a_from[n] = p.a + r * p.a_row + m0 + a.column_of(n);
        b_from[n] = p.b + r * p.b_row + n0 + b.column_of(n);
      }
      if ((t + 1) * S::KT <= live && whole_columns) {
        a.load(a_from);
        b.load(b_from);
      } else {
        auto a_left = [&](int n) { return row[n] < 0 ? 0 : p.M - m0 - a.column_of(n); };
        auto b_left = [&](int n) { return row[n] < 0 ? 0 : p.N - n0 - b.column_of(n); };
        if (p.M % 8 == 0 && p.N % 8 == 0) {
          a.load_chunks(a_from, a_left);
          b.load_chunks(b_from, b_left);
        } else {
          a.load(a_from, a_left);
          b.load(b_from, b_left);
        }
      }
      look(t + 1);
    };
    if (steps) load(0);
    for (int t = 0; t < steps; ++t) {
      if (S::BUFFERS == 1 && t) __syncthreads();  // the last tile has been used
      a.put(tile_a(t));
      b.put(tile_b(t));
      if (t + 1 < steps) load(t + 1);
      __syncthreads();
      multiply_tiles<T, S, A, B>(tile_a(t), tile_b(t), wm, wn, wk, lane, sum);
      add_columns(t);
    }
  }
  __syncthreads();

  const bool whole = length <= p.share;
  const int64_t part = part_of(begin, p.share) + first / p.share;
  if (summing) {
    float* held = reinterpret_cast<float*>(lds);
    static_assert(DOWN * S::TM * 4 <= LDS, "column sums fit the tiles' memory");
#pragma unroll
    for (int q = 0; q < 8; ++q)
      held[int(threadIdx.x) / ACROSS * S::TM + int(threadIdx.x) % ACROSS * 8 + q] = column[q];
    __syncthreads();
    const int c = int(threadIdx.x), at = (p.sums_of_a ? m0 : n0) + c, most = p.sums_of_a ? p.M : p.N;
    if (c < S::TM && at < most) {
      float s = 0.0f;
#pragma unroll
      for (int k = 0; k < DOWN; ++k) s += held[k * S::TM + c];
      if (kParts<T> == 3 && 0.0f * s != 0.0f) {  // not finite: again from the values themselves
        const T* v = p.sums_of_a ? p.a : p.b;
        const int64_t step = p.sums_of_a ? p.a_row : p.b_row;
        float again[8];
        exact_dots(
            [](int64_t) { return 1.0f; },
            [&](int64_t k, int) {
              const int64_t r = row_at(p.order, row0 + k, p.rows);
              return r < 0 ? 0.0f : float(v[r * step + at]);
            },
            live, 1, again);
        s = again[0];
      }
      if (whole) p.sums[group * most + at] = T(s);
      else p.sums_part[part * most + at] = s;
    }
    __syncthreads();
  }
  auto finish = [&](const auto& r, const auto& c, auto& v) {
    constexpr int EACH = sizeof(v) / sizeof(v[0]);
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
      const int m = m0 + r[e], n = n0 + c[e], most = p.N - n;
      if (m >= p.M || most <= 0) continue;
      if (kParts<T> == 3 && any_not_finite(v[e])) {
        auto value = [&](const T* from, int64_t step, int at, int64_t k) {
          const int64_t i = row_at(p.order, row0 + k, p.rows);
          return i < 0 ? 0.0f : float(from[i * step + at]);
        };
        exact_dots([&](int64_t k) { return value(p.a, p.a_row, m, k); },
                   [&](int64_t k, int q) { return value(p.b, p.b_row, n + q, k); }, live, most, v[e]);
      }
      if (whole) {
        Chunk<T, 8> out;
#pragma unroll
        for (int q = 0; q < 8; ++q) out.v[q] = T(v[e][q]);
        out.store(p.out + (group * p.M + m) * p.N + n, most);
      } else {
        Chunk<float, 8> out;
#pragma unroll
        for (int q = 0; q < 8; ++q) out.v[q] = v[e][q];
        out.store(p.part + (part * p.M + m) * p.N + n, most);
      }
    }
  };
  if constexpr (DIRECT) hand_out<S, 2 * S::FN>(sum, wm, wn, lane, finish);
  else give_out<S, S::FN>(lds, sum, wm, wn, wk, lane, finish);
}

struct SharePlan {
  int tile;
  int64_t share, slots, part_bytes, sums_bytes, bytes;
};

// Adds the sums of the shares of each group that has several, in order; the workgroups behind those of the
// products add the column sums.
constexpr int kJoinThreads = 256;

template <typename T>
__global__ __launch_bounds__(kJoinThreads) void weight_join_kernel(const WeightProduct<T> p, unsigned product_groups) {
  const bool columns = blockIdx.x >= product_groups;
  const int64_t size = columns ? (p.sums_of_a ? p.M : p.N) : int64_t(p.M) * p.N;
  const float* part = columns ? p.sums_part : p.part;
  T* out = columns ? p.sums : p.out;
  const int64_t at = (int64_t(columns ? blockIdx.x - product_groups : blockIdx.x) * kJoinThreads + threadIdx.x) * 8;
  for (int64_t g = blockIdx.y; g < (p.grouped ? p.groups : 1); g += gridDim.y) {
    const int64_t begin = p.grouped ? clamped(p.offsets[g], p.rows) : 0;
    const int64_t length = (p.grouped ? clamped(p.offsets[g + 1], p.rows) : p.rows) - begin;
    if (length <= p.share || at >= size) continue;
    const float* from = part + part_of(begin, p.share) * size + at;
    const int shares = int((length + p.share - 1) / p.share);
    float s[8];
#pragma unroll
    for (int q = 0; q < 8; ++q) s[q] = 0.0f;
#pragma unroll 4
    for (int k = 0; k < shares; ++k) {
      const Chunk<float, 8> v = Chunk<float, 8>::load(from + k * size, size - at < 8 ? int(size - at) : 8);
#pragma unroll
      for (int q = 0; q < 8; ++q) s[q] += v.v[q];
    }
    Chunk<T, 8> o;
#pragma unroll
    for (int q = 0; q < 8; ++q) o.v[q] = T(s[q]);
    o.store(out + g * size + at, size - at < 8 ? int(size - at) : 8);
  }
}

template <typename T>
struct Shapes;
template <>
struct Shapes<__bf16> {
  typedef Shape<2, 2, 1, 2, 2, 64, 2, 2> Large;
  typedef Shape<2, 2, 1, 1, 1, 64, 2, 4> Middle;
  typedef Shape<2, 4, 1, 4, 2, 64, 2, 2> Square;
};
template <>
struct Shapes<float> {
  typedef Shape<2, 2, 1, 2, 2, 32, 1, 2> Large;
  typedef Shape<2, 2, 1, 1, 1, 32, 1, 3> Middle;
};

// Whether every chunk of eight values of both operands is whole and aligned
template <typename T>
bool direct(const WeightProduct<T>& p) {
  return (reinterpret_cast<uintptr_t>(p.a) | reinterpret_cast<uintptr_t>(p.b)) % 16 == 0 && p.M % 8 == 0 &&
         p.N % 8 == 0 && p.a_row % 8 == 0 && p.b_row % 8 == 0;
}

// Shares of the rows and the tile of the weight that a workgroup owns: the largest tile that gives the card
// enough workgroups with shares of kLeastShare rows, 256 of 256 x 256 (direct loads), 512 of 128 x 128.  Tiles of 64 x 64
// also where those of 128 x 128 would be a quarter empty.  fp32: 2 000 rows, 512 x 512, 21 us by 64 x 64, 26 by 128 x
// 128; 200 003 rows, 161 x 96, 118 and 127; 16 384 rows, 1 024 x 1 024, 286 and 215; bf16, by 256 x 256 57,
// by 128 x 128 58, and with 4 096 columns 142 and 183.
constexpr int64_t kLeastShare = 256;
enum WeightTile { kMiddleTile = 64, kLargeTile = 128, kSquareTile = 256 };
inline WeightTile tile_for(int64_t rows, int64_t groups, int64_t M, int64_t N, bool direct) {
  auto whole = [&](int64_t t) { return ((M + t - 1) / t) * ((N + t - 1) / t); };
  const int64_t shares = rows / kLeastShare + groups;
  if (direct && M >= 512 && N >= 512 && whole(256) * shares >= 256) return kSquareTile;
  return whole(128) * shares < 512 || whole(128) * 16 > whole(64) * 5 ? kMiddleTile : kLargeTile;
}

// Workgroups that the shares make: 256 of 256 x 256, which each fill a compute unit, else 512 of 128 x 128 and 1 024 of
// 64 x 64; 2 048 of either where there are groups, whose lengths differ (fp32, eight species, 16 384 rows, 1 024 x
// 2 048: 652 us, by 512 workgroups 900).
SharePlan share_plan(int64_t rows, int64_t groups, bool grouped, int64_t M, int64_t N, bool direct) {
  SharePlan f{};
  f.tile = tile_for(rows, groups, M, N, direct);
  const int64_t t = f.tile, tiles = ((M + t - 1) / t) * ((N + t - 1) / t);
  const int64_t most = t == kSquareTile ? 256 : grouped ? 2048 : t == kLargeTile ? 512 : 1024;
  const int64_t parts = tiles == 0 ? most : tiles < most ? most / tiles : 1;
  f.share = (rows + parts - 1) / parts;
  if (f.share < kLeastShare) f.share = kLeastShare;
  if (f.share > (1 << 30)) f.share = 1 << 30;
  f.slots = part_count(rows, f.share);
  f.part_bytes = up(f.slots * M * N * 4);
  f.sums_bytes = up(f.slots * (M > N ? M : N) * 4);
  f.bytes = f.part_bytes + f.sums_bytes;
  return f;
}

template <typename T>
SharePlan share_plan(const WeightProduct<T>& p) {
  return share_plan(p.rows, p.grouped ? p.groups : 1, p.grouped, p.M, p.N, sizeof(T) == 2 && direct(p));
}
template <typename T, typename S, bool DIRECT = false>
int launch_shaped(WeightProduct<T> p, hipStream_t s) {
  p.tiles_m = p.M ? unsigned((p.M + S::TM - 1) / S::TM) : 1;  // no rows or columns: there may be sums
  p.tiles_n = p.N ? unsigned((p.N + S::TN - 1) / S::TN) : 1;
  const int64_t slots = p.grouped ? p.rows / p.share + p.groups : (p.rows + p.share - 1) / p.share;
  // The slots of groups are full, in part or empty, and workgroups go to the XCDs in turn: a slot's tiles are shared by all
  // of them.  Eight species, 16 384 rows, 2 048 x 1 024, bf16: 138 us, 202 with runs of slots on one XCD.
  const int64_t tiles = int64_t(p.tiles_m) * p.tiles_n;
  p.spread = p.grouped && tiles >= 8;
  const int64_t groups = (slots ? slots : 1) * (p.spread ? (tiles + 7) / 8 * 8 : tiles);
  if (!fits_grid(groups, S::NT))
    return set_error(YE3T_EUNSUPPORTED, "weights of %d x %d for %lld species are too many for one launch", p.M, p.N,
                     (long long)p.groups);
  hipLaunchKernelGGL((weight_product_kernel<T, S, DIRECT>), dim3(unsigned(groups)), dim3(S::NT), 0, s, p);
  return check_launch("weight_product_kernel");
}

}  // namespace

template <typename T>
int64_t weight_bytes(WeightProduct<T> p) {
  const int64_t groups = p.grouped ? p.groups : 1;
  const int64_t some = share_plan(p.rows, groups, p.grouped, p.M, p.N, false).bytes;
  const int64_t direct = share_plan(p.rows, groups, p.grouped, p.M, p.N, sizeof(T) == 2).bytes;
  return some > direct ? some : direct;
}
template int64_t weight_bytes(WeightProduct<float>);
template int64_t weight_bytes(WeightProduct<__bf16>);

template <typename T>
int launch_weights(WeightProduct<T> p, void* work, hipStream_t s) {
  const int64_t groups = p.grouped ? p.groups : 1;
  if (groups == 0 || ((p.M == 0 || p.N == 0) && !p.sums)) return YE3T_OK;
  const SharePlan f = share_plan(p);
  p.share = f.share;
  p.part = static_cast<float*>(work);
  p.sums_part = reinterpret_cast<float*>(static_cast<char*>(work) + f.part_bytes);
  int rc = YE3T_OK;
  if constexpr (sizeof(T) == 2) {
    if (f.tile == kSquareTile) rc = launch_shaped<T, typename Shapes<T>::Square, true>(p, s);
    else if (f.tile == kMiddleTile) rc = launch_shaped<T, typename Shapes<T>::Middle>(p, s);
    else if (direct(p)) rc = launch_shaped<T, typename Shapes<T>::Large, true>(p, s);
    else rc = launch_shaped<T, typename Shapes<T>::Large>(p, s);
  } else {
    rc = f.tile == kLargeTile ? launch_shaped<T, typename Shapes<T>::Large>(p, s)
                              : launch_shaped<T, typename Shapes<T>::Middle>(p, s);
  }
  if (rc) return rc;
  if (p.rows <= p.share) return YE3T_OK;
  const int64_t per = kJoinThreads * 8, product = (int64_t(p.M) * p.N + per - 1) / per;
  const int64_t column = p.sums ? ((p.sums_of_a ? p.M : p.N) + per - 1) / per : 0;
  if (!fits_grid(product + column, kJoinThreads))
    return set_error(YE3T_EUNSUPPORTED, "a weight of %d x %d is too large for one launch", p.M, p.N);
  hipLaunchKernelGGL((weight_join_kernel<T>), dim3(unsigned(product + column), unsigned(groups < 65535 ? groups : 65535)),
                     dim3(kJoinThreads), 0, s, p, unsigned(product));
  return check_launch("weight_join_kernel");
}
template int launch_weights<float>(WeightProduct<float>, void*, hipStream_t);
template int launch_weights<__bf16>(WeightProduct<__bf16>, void*, hipStream_t);

}  // namespace linear
}  // namespace ye3t
