// Rows times weights: the forward product and the gradient to the rows.
#include "linear.h"

namespace ye3t {
namespace linear {
namespace {

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
  const int steps = (K + S::KT - 1) / S::KT;
  auto tile_a = [&](int t) { return reinterpret_cast<__bf16*>(lds + t % S::BUFFERS * STEP); };
  auto tile_b = [&](int t) { return reinterpret_cast<__bf16*>(lds + t % S::BUFFERS * STEP + A::kBytes); };
  if constexpr (DIRECT) {
    // Lines past the tile's rows or columns repeat others: their results go nowhere.  Past the contraction there
    // are zeros.
    DirectLoads<S::TM, S::KT, false, S::NT> a;
    DirectLoads<S::TN, S::KT, ACROSS, S::NT> b;
    const T *a_from[decltype(a)::kEach], *b_from[decltype(b)::kEach];  // of the next tile
#pragma unroll
    for (int n = 0; n < decltype(a)::kEach; ++n) {
      const int line = a.line_of(n);
      const int64_t row = row_at(p.order, row0 + (line < live ? line : 0), p.rows);
      a_from[n] = p.a + (row < 0 ? 0 : row) * p.a_row + a.column_of(n);
    }
#pragma unroll
    for (int n = 0; n < decltype(b)::kEach; ++n) {
      const int line = b.line_of(n), c = b.column_of(n);
      b_from[n] = ACROSS ? weight + line * p.b_row + (n0 + c < p.N ? n0 + c : 0)
                         : weight + (n0 + line < p.N ? n0 + line : 0) * p.b_row + c;
    }
    const int64_t b_step = ACROSS ? S::KT * p.b_row : S::KT;
    auto load = [&](int t, auto part, auto parts) {
      auto each = [&](auto& loads, __bf16* tile, const T** from, int64_t step, auto exists) {
        constexpr int EACH = std::remove_reference_t<decltype(loads)>::kEach, P = decltype(part)::value, OF = decltype(parts)::value;
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
        each(b, tile_b(t), b_from, b_step, [&](int n) { return k0 + (ACROSS ? b.line_of(n) : b.column_of(n)) < K; });
      }
    };
    multiply_direct<S, A, B, decltype(a)::kEach + decltype(b)::kEach>(steps, tile_a, tile_b, wm, wn, wk, lane, load,
                                                                      [](int) {}, sum);
  } else {
    Loads<T, S::TM, S::KT, false, S::NT> a;
    Loads<T, S::TN, S::KT, ACROSS, S::NT> b;
    const T* a_line[decltype(a)::kEach];
#pragma unroll
    for (int n = 0; n < decltype(a)::kEach; ++n) {
      const int line = A::line_of(n * S::NT + int(threadIdx.x));
      const int64_t row = line < live ? row_at(p.order, row0 + line, p.rows) : -1;
      a_line[n] = row >= 0 ? p.a + row * p.a_row : nullptr;
    }
    auto load = [&](int k0) {
      a.load([&](int, int c, int n) { return a_line[n] ? a_line[n] + k0 + c : nullptr; }, [&](int c) { return K - k0 - c; });
      if (ACROSS)
        b.load([&](int k, int c, int) { return k0 + k < K ? weight + int64_t(k0 + k) * p.b_row + n0 + c : nullptr; },
               [&](int c) { return p.N - n0 - c; });
      else
        b.load([&](int n, int c, int) { return n0 + n < p.N ? weight + int64_t(n0 + n) * p.b_row + k0 + c : nullptr; },
               [&](int c) { return K - k0 - c; });
    };
    if (steps) load(0);
    for (int t = 0; t < steps; ++t) {
      if (S::BUFFERS == 1 && t) __syncthreads();  // the last tile has been used
      a.put(tile_a(t));
      b.put(tile_b(t));
      if (t + 1 < steps) load((t + 1) * S::KT);
      __syncthreads();
      multiply_tiles<T, S, A, B>(tile_a(t), tile_b(t), wm, wn, wk, lane, sum);
    }
    __syncthreads();
  }

  const uint64_t seed = p.dropout.below ? seed_of(p.dropout) : 0;
  auto finish = [&](int r, int c, float* v) {
    const int n = n0 + c, left = p.N - n;
    if (r >= live || left <= 0) return;
    const int64_t row = row_at(p.order, row0 + r, p.rows);
    if (row < 0) return;
    if (kParts<T> == 3 && any_not_finite(v)) {
      for (int q = 0; q < 8 && q < left; ++q) {
        const int64_t k_step = ACROSS ? p.b_row : 1, n_step = ACROSS ? 1 : p.b_row;
        const T *x = p.a + row * p.a_row, *w = weight + (n + q) * n_step;
        v[q] = exact_dot([&](int64_t k) { return float(x[k]); }, [&](int64_t k) { return float(w[k * k_step]); }, K);
      }
    }
    if (p.bias && !(p.grouped && group == p.groups)) {
      const Chunk<T, 8> bias = Chunk<T, 8>::load(p.bias + group * p.N + n, left);
#pragma unroll
      for (int q = 0; q < 8; ++q) v[q] += float(bias.v[q]);
    }
    const int64_t at = row * p.N + n;
    Chunk<T, 8> out;
    if (p.kept) {
#pragma unroll
      for (int q = 0; q < 8; ++q) out.v[q] = T(v[q]);
      out.store(p.kept + at, left);
    }
    if (p.activation != kNone) {
#pragma unroll
      for (int q = 0; q < 8; ++q) v[q] = activated(p.activation, v[q]);
    }
    if (p.dropout.below) drop(p.dropout, seed, row, uint32_t(n) / 8, v);
    if (p.residual) {
      const Chunk<T, 8> more = Chunk<T, 8>::load(p.residual + at, left);
#pragma unroll
      for (int q = 0; q < 8; ++q) v[q] += float(more.v[q]);
    }
#pragma unroll
    for (int q = 0; q < 8; ++q) out.v[q] = T(v[q]);
    out.store(p.out + at, left);
  };
  if constexpr (DIRECT) hand_out<S>(sum, wm, wn, lane, finish);
  else give_out<S>(lds, sum, wm, wn, wk, lane, finish);
}

template <typename T, typename S, bool DIRECT = false>
int launch_shaped(RowProduct<T> p, hipStream_t s) {
  const int64_t items = p.grouped ? item_count(p.rows, p.groups + 1, S::TM) : (p.rows + S::TM - 1) / S::TM;
  p.tiles_n = unsigned((p.N + S::TN - 1) / S::TN);
  if (!fits_grid(items * p.tiles_n, S::NT))
    return set_error(YE3T_EUNSUPPORTED, "%lld rows of %d columns are too many for one launch", (long long)p.rows, p.N);
  hipLaunchKernelGGL((p.b_across ? row_product_kernel<T, S, true, DIRECT> : row_product_kernel<T, S, false, DIRECT>),
                     dim3(unsigned(items * p.tiles_n)), dim3(S::NT), 0, s, p);
  return check_launch("row_product_kernel");
}

template <typename T>
struct Shapes;
template <>
struct Shapes<__bf16> {
  typedef Shape<2, 2, 1, 2, 2, 64, 2, 2> Large;
  typedef Shape<2, 2, 1, 1, 1, 64, 2, 4> Middle;
  typedef Shape<1, 1, 8, 1, 1, 64, 1, 2> Few;
  typedef Shape<2, 4, 1, 4, 2, 64, 2, 2> Square;
};
template <>
struct Shapes<float> {
  typedef Shape<2, 2, 1, 2, 2, 32, 1, 2> Large;
  typedef Shape<2, 2, 1, 1, 1, 32, 1, 3> Middle;
  typedef Shape<1, 1, 8, 1, 1, 32, 1, 2> Few;
};

// Whether every chunk of eight values of both operands is whole and aligned
template <typename T>
bool direct(const RowProduct<T>& p) {
  return (reinterpret_cast<uintptr_t>(p.a) | reinterpret_cast<uintptr_t>(p.b)) % 16 == 0 && p.K % 8 == 0 &&
         p.a_row % 8 == 0 && p.b_row % 8 == 0 && p.b_group % 8 == 0 && (!p.b_across || p.N % 8 == 0);
}

}  // namespace

template <typename T>
int launch_rows(RowProduct<T> p, hipStream_t s) {
  if (p.rows == 0 || p.N == 0) return YE3T_OK;
  auto tiles = [&](int64_t t) { return ((p.rows + t - 1) / t + (p.grouped ? p.groups : 0)) * ((p.N + t - 1) / t); };
  if constexpr (sizeof(T) == 2) {
    // Direct loads: tiles of 256 x 256 halve what is read, but one workgroup fills a compute unit, and nothing hides how
    // it begins and ends.  40 000 x 512 x 1 024: 74 us, by tiles of 128 x 128 63; 16 384 x 1 024 x 4 096: 150 and 163.
    if (direct(p) && p.K >= 1024 && p.rows > 64 && tiles(256) >= 256)
      return launch_shaped<T, typename Shapes<T>::Square, true>(p, s);
    if (direct(p) && p.rows > 64 && tiles(128) >= 256) return launch_shaped<T, typename Shapes<T>::Large, true>(p, s);
  }
  // tiles of 128 x 128 where they give every compute unit one, of 64 x 64 where those do, else of 32 x 32 with the
  // contraction shared by eight waves
  if (p.rows > 64 && tiles(128) >= 256) return launch_shaped<T, typename Shapes<T>::Large>(p, s);
  if (p.rows > 32 && tiles(64) >= 256) return launch_shaped<T, typename Shapes<T>::Middle>(p, s);
  return launch_shaped<T, typename Shapes<T>::Few>(p, s);
}
template int launch_rows<float>(RowProduct<float>, hipStream_t);
template int launch_rows<__bf16>(RowProduct<__bf16>, hipStream_t);

}  // namespace linear
}  // namespace ye3t
