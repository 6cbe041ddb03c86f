// Rows times weights: the forward product and the gradient to the rows.
//
// A workgroup owns a tile of one group's rows and the weight's columns.  The rows' operand runs along the contraction;
// the weight's runs along or across it, as it lies in memory.  Long products are bound by the matrix instructions (bf16
// 1 000 to 1 200 TFLOP/s; fp32 160 to 190 TFLOP/s of fp32 work, the library's fp32 product 153), short ones by the rows' reads and
// writes (200 003 x 161 x 96, fp32, 90 us for 205 MB: few steps of loads that are waited for), and few
// rows by the latency of one step of loads after the other.
#include "linear.h"

namespace ye3t {
namespace linear {
namespace {

// What follows the sums: some chunks of a lane, row (-1: none) and column of each.  What they need is loaded together.
template <typename T, int EACH>
__device__ inline void epilogue(const RowProduct<T>& p, const T* weight, const T* bias, uint64_t seed, int K,
                                const int64_t (&row)[EACH], const int (&n)[EACH], float (&v)[EACH][8]) {
  int64_t at[EACH];
  int left[EACH];
  Chunk<T, 8> offset[EACH], more[EACH];
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
    left[e] = row[e] < 0 ? 0 : p.N - n[e];
    at[e] = row[e] * p.N + n[e];
    if (left[e] <= 0) continue;
    if (bias) offset[e] = Chunk<T, 8>::load(bias + n[e], left[e]);
    if (p.residual) more[e] = Chunk<T, 8>::load(p.residual + at[e], left[e]);
  }
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
    if (left[e] <= 0) continue;
    if (kParts<T> == 3 && any_not_finite(v[e])) {
      const T* x = p.a + row[e] * p.a_row;
      const int64_t k_step = p.b_across ? p.b_row : 1, n_step = p.b_across ? 1 : p.b_row;
      const T* w = weight + n[e] * n_step;
      exact_dots([&](int64_t k) { return float(x[k]); },
                 [&](int64_t k, int q) { return float(w[k * k_step + q * n_step]); }, K, left[e], v[e]);
    }
    if (bias) {
#pragma unroll
      for (int q = 0; q < 8; ++q) v[e][q] += float(offset[e].v[q]);
    }
    Chunk<T, 8> out;
    if (p.kept) {
#pragma unroll
      for (int q = 0; q < 8; ++q) out.v[q] = T(v[e][q]);
      out.store(p.kept + at[e], left[e]);
    }
    if (p.activation != kNone) activate(p.activation, v[e]);
    if (p.dropout.below) drop(p.dropout, seed, row[e], uint32_t(n[e]) / 8, v[e]);
    if (p.residual) {
#pragma unroll
      for (int q = 0; q < 8; ++q) v[e][q] += float(more[e].v[q]);
    }
#pragma unroll
    for (int q = 0; q < 8; ++q) out.v[q] = T(v[e][q]);
    out.store(p.out + at[e], left[e]);
  }
}

template <typename T, typename S, bool ACROSS, bool DIRECT>
__global__ __launch_bounds__(S::NT, S::kPerSimd) void row_product_kernel(const RowProduct<T> p) {
  typedef Tile<T, S::TM, S::KT, false> A;
  typedef Tile<T, S::TN, S::KT, ACROSS> B;
  constexpr int STEP = A::kBytes + B::kBytes;
  constexpr int LDS = S::BUFFERS * STEP > S::kOutBytes || DIRECT ? S::BUFFERS * STEP : S::kOutBytes;
  __shared__ __align__(256) char lds[LDS];
  const int lane = int(threadIdx.x) & 63, wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) >> 6);
  const int wn = wave % S::WN, wm = wave / S::WN % S::WM, wk = wave / (S::WN * S::WM);

  const Place place = place_of(tile_of_group(), gridDim.x / p.tiles_n, p.tiles_n);
  const int64_t slot = place.row;
  const int n0 = place.column * S::TN;
  int64_t group = 0, begin = 0, first = slot * S::TM, length = p.rows;
  int K = p.K;
  if (p.grouped) {
    const Item item = item_of(p.offsets, p.groups + 1, p.rows, 1, S::TM, slot);
    group = item.structure;
    first = item.first;
    begin = clamped(p.offsets[group], p.rows);
    const int64_t end = group < p.groups ? clamped(p.offsets[group + 1], p.rows) : p.rows;
    length = end - begin;
    if (group == p.groups) K = 0;  // rows behind the last group
  }
  if (first >= length) return;
  const int64_t row0 = begin + first;
  const int live = length - first < S::TM ? int(length - first) : S::TM;
  const T* weight = p.b + group * p.b_group;

  f32x16 sum[S::FM][S::FN];
#pragma unroll
  for (int i = 0; i < S::FM; ++i)
#pragma unroll
    for (int j = 0; j < S::FN; ++j) sum[i][j] = zeros();
  int steps = (K + S::KT - 1) / S::KT, begin_step = 0;
  if constexpr (S::WK > 1) {
    if (p.parts > 1) {  // this workgroup's part of the contraction
      begin_step = int(blockIdx.y) * p.part_steps;
      steps = steps - begin_step < p.part_steps ? (steps > begin_step ? steps - begin_step : 0) : p.part_steps;
    }
  }
  auto tile_a = [&](int t) { return reinterpret_cast<__bf16*>(lds + t % S::BUFFERS * STEP); };
  auto tile_b = [&](int t) { return reinterpret_cast<__bf16*>(lds + t % S::BUFFERS * STEP + A::kBytes); };
  // Lines past the tile's rows or columns repeat others: their results go nowhere.  Past the contraction there are
  // zeros in both operands.
  typedef LoadsOf<T, S::TM, S::KT, false, S::NT, DIRECT> LoadsA;
  typedef LoadsOf<T, S::TN, S::KT, ACROSS, S::NT, DIRECT> LoadsB;
  LoadsA a;
  LoadsB b;
  const T *a_from[LoadsA::kEach], *b_from[LoadsB::kEach];  // of the next tile
  const int64_t b_step = ACROSS ? S::KT * p.b_row : S::KT;
#pragma unroll
  for (int n = 0; n < LoadsA::kEach; ++n) {
    const int line = a.line_of(n);
    const int64_t row = row_at(p.order, row0 + (line < live ? line : 0), p.rows);
    a_from[n] = p.a + (row < 0 ? 0 : row) * p.a_row + a.column_of(n) + begin_step * S::KT;
  }
#pragma unroll
  for (int n = 0; n < LoadsB::kEach; ++n) {
    const int line = b.line_of(n), c = b.column_of(n);
    b_from[n] = (ACROSS ? weight + line * p.b_row + (n0 + c < p.N ? n0 + c : 0)
                        : weight + (n0 + line < p.N ? n0 + line : 0) * p.b_row + c) + begin_step * b_step;
  }
  if constexpr (DIRECT) {
    auto load = [&](int t, auto part, auto parts) {
      auto each = [&](auto& loads, __bf16* tile, const T** from, int64_t step, auto exists) {
        constexpr int EACH = std::remove_reference_t<decltype(loads)>::kEach;
        constexpr int P = decltype(part)::value, OF = decltype(parts)::value;
#pragma unroll
        for (int n = EACH * P / OF; n < EACH * (P + 1) / OF; ++n) {
          loads.load(tile, n, wave, exists(n) ? from[n] : loads.none());
          from[n] += step;
        }
      };
      const int k0 = t * S::KT;
      if (k0 + S::KT <= K) {
        each(a, tile_a(t), a_from, S::KT, [](int) { return true; });
        each(b, tile_b(t), b_from, b_step, [](int) { return true; });
      } else {
        each(a, tile_a(t), a_from, S::KT, [&](int n) { return k0 + a.column_of(n) < K; });
        each(b, tile_b(t), b_from, b_step,
             [&](int n) { return k0 + (ACROSS ? b.line_of(n) : b.column_of(n)) < K; });
      }
    };
    multiply_direct<S, A, B, LoadsA::kEach + LoadsB::kEach, false>(steps, 0, tile_a, tile_b, wm, wn, wk, lane, load,
                                                                   [](int) {}, sum);
  } else {
    const bool whole = !ACROSS || n0 + S::TN <= p.N;  // no chunk of b has columns past the last
    const bool chunks = K % 8 == 0 && (!ACROSS || p.N % 8 == 0);  // every chunk is there or not
    auto load = [&](int k0) {
      if (k0 + S::KT <= K && whole) {
        a.load(a_from);
        b.load(b_from);
      } else {
        auto a_left = [&](int n) { return K - k0 - a.column_of(n); };
        auto b_left = [&](int n) {
          return !ACROSS ? K - k0 - b.column_of(n) : k0 + b.line_of(n) < K ? p.N - n0 - b.column_of(n) : 0;
        };
        if (chunks) {
          a.load_chunks(a_from, a_left);
          b.load_chunks(b_from, b_left);
        } else {
          a.load(a_from, a_left);
          b.load(b_from, b_left);
        }
      }
#pragma unroll
      for (int n = 0; n < LoadsA::kEach; ++n) a_from[n] += S::KT;
#pragma unroll
      for (int n = 0; n < LoadsB::kEach; ++n) b_from[n] += b_step;
    };
    if (steps) load(begin_step * S::KT);
    for (int t = 0; t < steps; ++t) {
      if (S::BUFFERS == 1 && t) __syncthreads();  // the last tile has been used
      a.put(tile_a(t));
      b.put(tile_b(t));
      if (t + 1 < steps) load((begin_step + t + 1) * S::KT);
      __syncthreads();
      multiply_tiles<T, S, A, B>(tile_a(t), tile_b(t), wm, wn, wk, lane, sum);
    }
    __syncthreads();
  }

  if constexpr (S::WK > 1) {
    if (p.parts > 1) {
      give_out<S, 1>(lds, sum, wm, wn, wk, lane, [&](const auto& r, const auto& c, auto& v) {
        const int left = p.N - n0 - c[0];
        if (r[0] >= live || left <= 0) return;
        Chunk<float, 8> out;
#pragma unroll
        for (int q = 0; q < 8; ++q) out.v[q] = v[0][q];
        out.store(p.part + (blockIdx.y * p.rows + row0 + r[0]) * p.N + n0 + c[0], left);
      });
      return;
    }
  }
  const uint64_t seed = p.dropout.below ? seed_of(p.dropout) : 0;
  const T* bias = p.bias && !(p.grouped && group == p.groups) ? p.bias + group * p.N : nullptr;
  auto finish = [&](const auto& r, const auto& c, auto& v) {
    constexpr int EACH = sizeof(v) / sizeof(v[0]);
    int64_t row[EACH];
    int n[EACH];
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
      row[e] = r[e] < live ? row_at(p.order, row0 + r[e], p.rows) : -1;
      n[e] = n0 + c[e];
    }
    epilogue(p, weight, bias, seed, K, row, n, v);
  };
  if constexpr (DIRECT) hand_out<S, 2 * S::FN>(sum, wm, wn, lane, finish);
  else give_out<S, sizeof(T) == 4 ? S::FN : 2 * S::FN>(lds, sum, wm, wn, wk, lane, finish);
}

// The same with tiles of direct loads that fill a compute unit: a workgroup goes through several, and the first loads
// of the next run while the results of one are finished and written.  16 384 x 1 024 x 4 096: 132 to 145 us (1 036 to
// 948 TFLOP/s from card to card), by a workgroup a tile 14 % more; with a bias and gelu 186, the preactivation kept too
// 205, among a training step's other kernels 211 to 219.  Bound by the matrix instructions: at 8 192^3 they run 66 % of the
// cycles, at a clock that falls with their share.
template <typename S, bool ACROSS>
__global__ __launch_bounds__(S::NT, S::kPerSimd) void row_product_rounds_kernel(const RowProduct<__bf16> p,
                                                                                int64_t items) {
  typedef __bf16 T;
  typedef Tile<T, S::TM, S::KT, false> A;
  typedef Tile<T, S::TN, S::KT, ACROSS> B;
  typedef DirectLoads<S::TM, S::KT, false, S::NT> LoadsA;
  typedef DirectLoads<S::TN, S::KT, ACROSS, S::NT> LoadsB;
  constexpr int STEP = A::kBytes + B::kBytes;
  static_assert(S::BUFFERS == 2 && S::WK == 1, "two buffers");
  __shared__ __align__(256) char lds[2 * STEP];
  const int lane = int(threadIdx.x) & 63, wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) >> 6);
  const int wn = wave % S::WN, wm = wave / S::WN;
  auto tile_a = [&](int t) { return reinterpret_cast<T*>(lds + (t & 1) * STEP); };
  auto tile_b = [&](int t) { return reinterpret_cast<T*>(lds + (t & 1) * STEP + A::kBytes); };

  // This XCD's share of the tiles, and its workgroups that take them in turn
  const int64_t all = items * p.tiles_n;
  const unsigned x = blockIdx.x & 7, n = gridDim.x;
  const int64_t begin = x * (all / 8) + (x < all % 8 ? x : all % 8), end = begin + all / 8 + (x < all % 8);
  const unsigned workers = n / 8 + (x < n % 8);
  int64_t next = begin + blockIdx.x / 8;

  struct At {
    int64_t row0, group;
    int live, n0, K;
  };
  auto advance = [&](At& at) {
    for (; next < end; next += workers) {
      const Place place = place_of(next, items, p.tiles_n);
      int64_t group = 0, first = place.row * S::TM, from = 0, length = p.rows;
      int K = p.K;
      if (p.grouped) {
        const Item item = item_of(p.offsets, p.groups + 1, p.rows, 1, S::TM, place.row);
        group = item.structure;
        first = item.first;
        from = clamped(p.offsets[group], p.rows);
        length = (group < p.groups ? clamped(p.offsets[group + 1], p.rows) : p.rows) - from;
        if (group == p.groups) K = 0;  // rows behind the last group
      }
      if (first >= length) continue;
      const int live = length - first < S::TM ? int(length - first) : S::TM;
      at = {from + first, group, live, place.column * S::TN, K};
      next += workers;
      return true;
    }
    return false;
  };

  const T *a_from[LoadsA::kEach], *b_from[LoadsB::kEach];
  const int64_t b_step = ACROSS ? S::KT * p.b_row : S::KT;
  At at;
  auto load = [&](int t, auto part, auto parts) {
    auto each = [&](auto loads, T* tile, const T** from, int64_t step, auto exists) {
      constexpr int EACH = decltype(loads)::kEach, P = decltype(part)::value, OF = decltype(parts)::value;
#pragma unroll
      for (int k = EACH * P / OF; k < EACH * (P + 1) / OF; ++k) {
        loads.load(tile, k, wave, exists(k) ? from[k] : loads.none());
        from[k] += step;
      }
    };
    const int k0 = t * S::KT;
    if (k0 + S::KT <= at.K) {
      each(LoadsA(), tile_a(t), a_from, S::KT, [](int) { return true; });
      each(LoadsB(), tile_b(t), b_from, b_step, [](int) { return true; });
    } else {
      each(LoadsA(), tile_a(t), a_from, S::KT, [&](int k) { return k0 + LoadsA::column_of(k) < at.K; });
      each(LoadsB(), tile_b(t), b_from, b_step,
           [&](int k) { return k0 + (ACROSS ? LoadsB::line_of(k) : LoadsB::column_of(k)) < at.K; });
    }
  };
  auto start = [&] {
#pragma unroll
    for (int k = 0; k < LoadsA::kEach; ++k) {
      const int line = LoadsA::line_of(k);
      const int64_t row = row_at(p.order, at.row0 + (line < at.live ? line : 0), p.rows);
      a_from[k] = p.a + (row < 0 ? 0 : row) * p.a_row + LoadsA::column_of(k);
    }
    const T* weight = p.b + at.group * p.b_group;
#pragma unroll
    for (int k = 0; k < LoadsB::kEach; ++k) {
      const int line = LoadsB::line_of(k), c = LoadsB::column_of(k);
      b_from[k] = ACROSS ? weight + line * p.b_row + (at.n0 + c < p.N ? at.n0 + c : 0)
                         : weight + (at.n0 + line < p.N ? at.n0 + line : 0) * p.b_row + c;
    }
    if (at.K > 0) load(0, std::integral_constant<int, 0>(), std::integral_constant<int, 1>());
    asm volatile("" ::: "memory");  // the loads stay before what follows
  };

  const uint64_t seed = p.dropout.below ? seed_of(p.dropout) : 0;
  if (!advance(at)) return;
  start();
  int behind = 0;
  for (;;) {
    f32x16 sum[S::FM][S::FN];
#pragma unroll
    for (int i = 0; i < S::FM; ++i)
#pragma unroll
      for (int j = 0; j < S::FN; ++j) sum[i][j] = zeros();
    multiply_direct<S, A, B, LoadsA::kEach + LoadsB::kEach, true>((at.K + S::KT - 1) / S::KT, behind, tile_a, tile_b, wm,
                                                                  wn, 0, lane, load, [](int) {}, sum);
    const At done = at;
    // every wave has read its last operands before the next tile's loads take their place
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    const bool more = advance(at);
    if (more) start();
    const T* bias = p.bias && !(p.grouped && done.group == p.groups) ? p.bias + done.group * p.N : nullptr;
    hand_out<S, S::FN>(sum, wm, wn, lane, [&](const auto& r, const auto& c, auto& v) {
      constexpr int EACH = sizeof(v) / sizeof(v[0]);
      int64_t row[EACH];
      int column[EACH];
#pragma unroll
      for (int e = 0; e < EACH; ++e) {
        row[e] = r[e] < done.live ? row_at(p.order, done.row0 + r[e], p.rows) : -1;
        column[e] = done.n0 + c[e];
      }
      epilogue(p, p.b, bias, seed, done.K, row, column, v);
    });
    if (!more) return;
    // A whole tile's results are a store for every eight columns of 64 rows, in two outputs or one: 32 or 16, the counts
    // that multiply_direct waits by.
    static_assert(S::FM * S::FN * 2 == 16, "multiply_direct knows the stores of a tile");
    const bool whole = done.live == S::TM && done.n0 + S::TN <= p.N && !p.order;
    behind = whole ? (p.kept ? 2 : 1) * S::FM * S::FN * 2 : 0;
  }
}

// Adds the parts of the contraction in order and goes on as the product's own epilogue.  A lane a chunk of eight columns.
constexpr int kJoinThreads = 256;
template <typename T>
__global__ __launch_bounds__(kJoinThreads) void row_join_kernel(const RowProduct<T> p, int chunks) {
  const int64_t x = int64_t(blockIdx.x) * kJoinThreads + threadIdx.x, i = x / chunks;
  if (i >= p.rows) return;
  int64_t row[1] = {row_at(p.order, i, p.rows)}, group = 0;
  int n[1] = {int(x - i * chunks) * 8};
  if (p.grouped) {  // the group of row i: the number of offsets behind the first that are not above it
    int64_t lo = 0, hi = p.groups;
    while (lo < hi) {
      const int64_t mid = (lo + hi) >> 1;
      if (p.offsets[mid + 1] <= i) lo = mid + 1;
      else hi = mid;
    }
    group = lo;
  }
  const bool none = p.grouped && group == p.groups;
  const int left = p.N - n[0];
  float v[1][8];
#pragma unroll
  for (int q = 0; q < 8; ++q) v[0][q] = 0.0f;
#pragma unroll 4
  for (int k = 0; k < p.parts; ++k) {
    const Chunk<float, 8> a = Chunk<float, 8>::load(p.part + (k * p.rows + i) * p.N + n[0], left);
#pragma unroll
    for (int q = 0; q < 8; ++q) v[0][q] += a.v[q];
  }
  epilogue(p, p.b + group * p.b_group, p.bias && !none ? p.bias + group * p.N : nullptr,
           p.dropout.below ? seed_of(p.dropout) : 0, none ? 0 : p.K, row, n, v);
}

template <typename T, typename S, bool DIRECT = false>
int launch_shaped(RowProduct<T> p, hipStream_t s) {
  const int64_t items = p.grouped ? item_count(p.rows, p.groups + 1, S::TM) : (p.rows + S::TM - 1) / S::TM;
  p.tiles_n = unsigned((p.N + S::TN - 1) / S::TN);
  if (!fits_grid(items * p.tiles_n, S::NT))
    return set_error(YE3T_EUNSUPPORTED, "%lld rows of %d columns are too many for one launch", (long long)p.rows, p.N);
  hipLaunchKernelGGL((p.b_across ? row_product_kernel<T, S, true, DIRECT> : row_product_kernel<T, S, false, DIRECT>),
                     dim3(unsigned(items * p.tiles_n), unsigned(p.parts)), dim3(S::NT), 0, s, p);
  if (int rc = check_launch("row_product_kernel")) return rc;
  if (p.parts == 1) return YE3T_OK;
  const int64_t chunks = (p.N + 7) / 8;
  hipLaunchKernelGGL((row_join_kernel<T>), dim3(unsigned((p.rows * chunks + kJoinThreads - 1) / kJoinThreads)),
                     dim3(kJoinThreads), 0, s, p, int(chunks));
  return check_launch("row_join_kernel");
}

constexpr int kComputeUnits = 256;

template <typename S>
int launch_rounds(RowProduct<__bf16> p, hipStream_t s) {
  const int64_t items = p.grouped ? item_count(p.rows, p.groups + 1, S::TM) : (p.rows + S::TM - 1) / S::TM;
  p.tiles_n = unsigned((p.N + S::TN - 1) / S::TN);
  const int64_t all = items * p.tiles_n;
  hipLaunchKernelGGL((p.b_across ? row_product_rounds_kernel<S, true> : row_product_rounds_kernel<S, false>),
                     dim3(unsigned(all < kComputeUnits ? all : kComputeUnits)), dim3(S::NT), 0, s, p, items);
  return check_launch("row_product_rounds_kernel");
}

template <typename T>
struct Shapes;
template <>
struct Shapes<__bf16> {
  typedef Shape<2, 2, 1, 2, 2, 64, 2, 2> Large;
  typedef Shape<2, 2, 1, 1, 1, 64, 2, 4> Middle;
  typedef Shape<1, 1, 8, 1, 1, 64, 1, 2> Few;
  typedef Shape<2, 4, 1, 4, 2, 64, 2, 2> Square;
  typedef Shape<2, 2, 1, 2, 2, 32, 3, 3> Direct;
};
template <>
struct Shapes<float> {
  typedef Shape<2, 2, 1, 2, 2, 32, 1, 3> Large;
  typedef Shape<2, 2, 1, 2, 1, 32, 1, 3> Tall;
  typedef Shape<2, 2, 1, 1, 1, 32, 1, 3> Middle;
  typedef Shape<1, 1, 8, 1, 1, 16, 1, 4> Few;
};

// Whether every chunk of eight values of both operands is whole and aligned
template <typename T>
bool direct(const RowProduct<T>& p) {
  return (reinterpret_cast<uintptr_t>(p.a) | reinterpret_cast<uintptr_t>(p.b)) % 16 == 0 && p.K % 8 == 0 &&
         p.a_row % 8 == 0 && p.b_row % 8 == 0 && p.b_group % 8 == 0 && (!p.b_across || p.N % 8 == 0);
}

// Which shape a product takes, and in how many parts of the contraction
enum Kind { kFew, kMiddle, kTall, kLarge, kDirect, kSquare };
struct Choice {
  Kind kind;
  int parts, part_steps;
};
template <typename T>
Choice choice_of(const RowProduct<T>& p, bool direct) {
  auto tiles = [&](int64_t t) { return ((p.rows + t - 1) / t + (p.grouped ? p.groups : 0)) * ((p.N + t - 1) / t); };
  if (direct && p.rows > 64) {
    // Direct loads: tiles of 256 x 256 read half of what those of 128 x 128 do, but one workgroup fills a compute unit
    // and nothing hides how it begins and ends, nor a last round that is not full.  65 536 x 2 048 x 2 048: 609 us, by
    // tiles of 128 x 128 767; 40 000 x 512 x 1 024 76 and 64; 40 000 x 2 048 x 512 (1.2 rounds) 116 and 104.
    const int64_t wide = tiles(256);
    if (p.K >= 1024 && wide * 4 >= (wide + 255) / 256 * 256 * 3) return {kSquare, 1, 0};
    if (tiles(128) >= 256) return {kDirect, 1, 0};
  }
  // Tiles of 128 x 128 where they give every compute unit one, of 64 x 64 where those do, else of 32 x 32 with the
  // contraction shared by eight waves, and by several workgroups where it is long and they are few.  fp32: tiles of
  // 128 x 64 where the contraction is short, for more workgroups that hide each other's loads, or where 128
  // columns leave much of the last tile empty.  200 003 x 161 x 96: 90 us, by 128 x 128 97; 60 000 x 512 x 192: 105
  // and 126; 16 384 x 1 024 x 1 024: 252 and 227; 30 011 x 128 x 128 by 89 species: 23, by 64 x 64 21.
  if constexpr (sizeof(T) == 4) {
    const int64_t tall = ((p.rows + 127) / 128 + (p.grouped ? p.groups : 0)) * ((p.N + 63) / 64);
    const bool empty = (p.N + 127) / 128 * 128 * 5 > (p.N + 63) / 64 * 64 * 6;
    if (p.rows > 64 && (p.K < 256 || empty)) {
      if (tall >= 1024) return {kTall, 1, 0};
      if (tiles(64) >= 256) return {kMiddle, 1, 0};
    }
  }
  if (p.rows > 64 && tiles(128) >= 256) return {kLarge, 1, 0};
  if (p.rows > 32 && tiles(64) >= 256) return {kMiddle, 1, 0};
  const int64_t groups = ((p.rows + 31) / 32 + (p.grouped ? p.groups : 0)) * ((p.N + 31) / 32);
  const int steps = (p.K + Shapes<T>::Few::KT - 1) / Shapes<T>::Few::KT;
  const int least = 2 * Shapes<T>::Few::KT < 512 ? 512 : 2 * Shapes<T>::Few::KT;  // of the contraction, for a part
  // as many workgroups as run at a time; 64 x 4 096 x 4 096 with the join: bf16 14 us (one part), by twice as many 18; fp32
  // 34 (two parts), by half as many 37, by twice as many 36
  const int64_t most = sizeof(T) == 4 ? 512 : 256;
  int parts = p.K / least;
  if (parts < 2 || groups > most / 2) return {kFew, 1, 0};
  if (parts > most / groups) parts = int(most / groups);
  const int each = (steps + parts - 1) / parts;
  return {kFew, (steps + each - 1) / each, each};
}

}  // namespace

template <typename T>
int64_t row_bytes(const RowProduct<T>& p) {
  if (p.rows == 0 || p.N == 0) return 0;
  const Choice c = choice_of(p, false);  // direct or not, it is the last choice that has parts
  return c.parts > 1 ? up(c.parts * p.rows * p.N * 4) : 0;
}

template <typename T>
int launch_rows(RowProduct<T> p, void* work, hipStream_t s) {
  if (p.rows == 0 || p.N == 0) return YE3T_OK;
  const Choice c = choice_of(p, sizeof(T) == 2 && direct(p));
  p.parts = c.parts;
  p.part_steps = c.part_steps;
  p.part = static_cast<float*>(work);
  if constexpr (sizeof(T) == 2) {
    if (c.kind == kSquare) return launch_rounds<typename Shapes<T>::Square>(p, s);
    if (c.kind == kDirect) return launch_shaped<T, typename Shapes<T>::Direct, true>(p, s);
  }
  if constexpr (sizeof(T) == 4) {
    if (c.kind == kTall) return launch_shaped<T, typename Shapes<T>::Tall>(p, s);
  }
  if (c.kind == kLarge) return launch_shaped<T, typename Shapes<T>::Large>(p, s);
  if (c.kind == kMiddle) return launch_shaped<T, typename Shapes<T>::Middle>(p, s);
  return launch_shaped<T, typename Shapes<T>::Few>(p, s);
}
template int64_t row_bytes(const RowProduct<float>&);
template int64_t row_bytes(const RowProduct<__bf16>&);
template int launch_rows<float>(RowProduct<float>, void*, hipStream_t);
template int launch_rows<__bf16>(RowProduct<__bf16>, void*, hipStream_t);

}  // namespace linear
}  // namespace ye3t
