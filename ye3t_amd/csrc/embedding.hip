// Rows of a table by token, scaled, and the table's gradient by sorted tokens.
//
//   out[i] = s T[t_i],   dT[v] = s (sum of g[i] over the i with t_i = v)
//
// The forward is a copy.  The gradient sorts the positions by token (stable
// counting passes over eight bits each), cuts the sorted positions into equal
// shares whatever the tokens' frequencies are, and sums each share in order in
// registers; a token that crosses a share's end leaves partial sums that are
// added in the shares' order.  No atomics: the sums depend on the tokens and
// sizes alone.  Sums are fp32 (fp64 for fp64 rows), scaled and rounded once.
#include "rows.h"
#include "sort.h"

namespace ye3t {
namespace {

constexpr int kThreads = 256;

// A lane a chunk of 16 bytes of an output row, four chunks a lane in flight.
// Tokens outside the table give rows of zeros.  Bound by the writes: 200 000 x 128
// fp32 18 us, 5.6 TB/s.
template <typename T, typename Index>
__global__ __launch_bounds__(kThreads) void embedding_kernel(const Index* __restrict__ tokens, int64_t N,
                                                             const T* __restrict__ table, int64_t row_stride,
                                                             int64_t vocabulary, int W, int chunks,
                                                             typename Wide<T>::type scale, T* __restrict__ out) {
  constexpr int V = kChunk<T>, STEPS = 4;
  const int64_t all = N * chunks;
  for (int64_t x0 = int64_t(blockIdx.x) * (kThreads * STEPS); x0 < all; x0 += int64_t(gridDim.x) * (kThreads * STEPS)) {
    Chunk<T, V> v[STEPS];
    int64_t row[STEPS];
    int c[STEPS];
#pragma unroll
    for (int k = 0; k < STEPS; ++k) {
      const int64_t x = x0 + k * kThreads + threadIdx.x;
      row[k] = all <= INT32_MAX ? int64_t(uint32_t(x) / uint32_t(chunks)) : x / chunks;
      c[k] = int(x - row[k] * chunks) * V;
      v[k] = Chunk<T, V>::zero();
      if (x < all) {
        const int64_t t = token_at(tokens, row[k], vocabulary);
        if (t >= 0) v[k] = Chunk<T, V>::load(table + t * row_stride + c[k], W - c[k]);
      }
    }
#pragma unroll
    for (int k = 0; k < STEPS; ++k) {
      if (x0 + k * kThreads + threadIdx.x < all) {
#pragma unroll
        for (int q = 0; q < V; ++q) v[k].v[q] = T(typename Wide<T>::type(v[k].v[q]) * scale);
        v[k].store(out + row[k] * W + c[k], W - c[k]);
      }
    }
  }
}

// ---- sums over the sorted positions -------------------------------------------
// Rows of tokens that do not occur: a workgroup looks 64 of them up in the
// sorted positions and clears those that are missing.
template <typename T>
__device__ inline void clear_missing(const Pair* __restrict__ sorted, int64_t N, int64_t vocabulary, int W,
                                     int64_t group, T* __restrict__ table) {
  constexpr int V = kChunk<T>;
  const int64_t v0 = group * 64;
  const int lane = threadIdx.x & 63;
  const int64_t v = v0 + lane;
  int64_t lo = 0, hi = v < vocabulary ? N : 0;
  while (lo < hi) {
    const int64_t mid = (lo + hi) >> 1;
    if (int64_t(sorted[mid].token) < v) lo = mid + 1;
    else hi = mid;
  }
  const bool missing = v < vocabulary && !(lo < N && int64_t(sorted[lo].token) == v);
  const uint64_t rows = __ballot(missing);  // the same in every wave
  if (rows == 0) return;
  const Chunk<T, V> zero = Chunk<T, V>::zero();
  const uint32_t chunks = uint32_t(W + V - 1) / V;
  for (uint32_t i = threadIdx.x; i < 64 * chunks; i += kThreads) {
    const uint32_t r = i / chunks;
    const int c = int(i - r * chunks) * V;
    if (rows >> r & 1) zero.store(table + (v0 + r) * W + c, W - c);
  }
}

// A worker is L lanes with a share of `share` sorted positions and a column
// chunk of 16 bytes a lane (grid axis y over the columns that L lanes do not
// hold).  Tokens that lie in the share go to the table.  The sum of a token that began
// before the share, or fills it and goes on, goes to `heads`, that of one that begins in it and goes on to
// `tails`; `ends` keeps the shares' first and last token for the kernel that joins them.
// Bound by the adjoint's read: 200 000 x 128 fp32 by 8 tokens 25 us for 102 MB, the
// whole gradient 52 us (sort 11, join 16).
template <typename T, int L>
__global__ __launch_bounds__(kThreads) void embedding_sum_kernel(
    const Pair* __restrict__ sorted, int64_t N, int64_t share, int64_t workers, const T* __restrict__ adjoint,
    int64_t vocabulary, int W, typename Wide<T>::type scale, int64_t clearing, T* __restrict__ table,
    typename Wide<T>::type* __restrict__ heads, typename Wide<T>::type* __restrict__ tails,
    uint32_t* __restrict__ ends) {
  typedef typename Wide<T>::type Real;
  constexpr int V = kChunk<T>, AHEAD = 8;
  if (int64_t(gridDim.x) - blockIdx.x <= clearing) {  // the last workgroups
    if (blockIdx.y == 0) clear_missing(sorted, N, vocabulary, W, int64_t(gridDim.x) - 1 - blockIdx.x, table);
    return;
  }
  const int lane = int(threadIdx.x) % L;
  const int64_t worker = int64_t(blockIdx.x) * (kThreads / L) + int(threadIdx.x) / L;
  const int c = (int(blockIdx.y) * L + lane) * V;
  if (worker >= workers || c >= W) return;
  const int64_t begin = worker * share, end = begin + share < N ? begin + share : N;
  Real sum[V];
#pragma unroll
  for (int q = 0; q < V; ++q) sum[q] = Real(0);
  const uint32_t first = sorted[begin].token;
  uint32_t now = first;
  bool head = begin > 0 && sorted[begin - 1].token == first;  // began before
  auto flush = [&](bool goes_on) {
    if (head || goes_on) {
      Real* to = (head || now == first ? heads : tails) + worker * W + c;
#pragma unroll
      for (int q = 0; q < V; ++q)
        if (c + q < W) to[q] = sum[q];
    } else if (int64_t(now) < vocabulary) {
      Chunk<T, V> a;
#pragma unroll
      for (int q = 0; q < V; ++q) a.v[q] = T(sum[q] * scale);
      a.store(table + int64_t(now) * W + c, W - c);
    }
    head = false;
  };
  for (int64_t p0 = begin; p0 < end; p0 += AHEAD) {
    Chunk<T, V> g[AHEAD];
    uint32_t token[AHEAD];
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const Pair p = sorted[p0 + k < end ? p0 + k : end - 1];
      token[k] = p.token;
      g[k] = Chunk<T, V>::load(adjoint + int64_t(p.position) * W + c, W - c);
    }
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      if (p0 + k >= end) break;
      if (token[k] != now) {
        flush(false);
        now = token[k];
#pragma unroll
        for (int q = 0; q < V; ++q) sum[q] = Real(0);
      }
#pragma unroll
      for (int q = 0; q < V; ++q) sum[q] += Real(g[k].v[q]);
    }
  }
  flush(end < N && sorted[end].token == now);
  if (lane == 0 && blockIdx.y == 0) {
    ends[2 * worker] = first;
    ends[2 * worker + 1] = now;
  }
}

// Joins a token that crosses the ends of shares: the workgroups of the share where it
// begins add the sums of the shares that it goes on in, found by bisection (the shares'
// first tokens do not fall).  Eight rows of lanes take the shares in turn, eight loads
// of each in flight, and are added in order.  Grid axis y takes columns in steps of 32: 2 600
// shares of one token, 128 columns, took 330 us by one load a lane and all columns in
// one workgroup.
constexpr int kJoinColumns = 32, kJoinGroups = 8;

template <typename T>
__global__ __launch_bounds__(kThreads) void embedding_join_kernel(
    const uint32_t* __restrict__ ends, int64_t workers, const typename Wide<T>::type* __restrict__ heads,
    const typename Wide<T>::type* __restrict__ tails, int64_t vocabulary, int W, typename Wide<T>::type scale,
    T* __restrict__ table) {
  typedef typename Wide<T>::type Real;
  constexpr int COLS = kJoinColumns, ROWS = kThreads / COLS, AHEAD = 8;
  __shared__ Real sums[ROWS][COLS + 1];
  const int64_t w = blockIdx.x;
  const int col = int(threadIdx.x) % COLS, row = int(threadIdx.x) / COLS;
  const uint32_t first = ends[2 * w], token = ends[2 * w + 1];
  if (w + 1 == workers || ends[2 * w + 2] != token || int64_t(token) >= vocabulary) return;  // ends here
  if (first == token && w > 0 && ends[2 * w - 1] == token) return;                           // does not begin here
  int64_t until = w + 2, hi = workers;
  while (until < hi) {
    const int64_t mid = (until + hi) >> 1;
    if (ends[2 * mid] == token) until = mid + 1;
    else hi = mid;
  }
  for (int c0 = int(blockIdx.y) * COLS; c0 < W; c0 += int(gridDim.y) * COLS) {
    const int c = c0 + col;
    Real s = Real(0);
    if (c < W) {
      if (row == 0) s = (first == token ? heads : tails)[w * W + c];
      for (int64_t k0 = w + 1 + row; k0 < until; k0 += AHEAD * ROWS) {
        Real v[AHEAD];
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) v[k] = k0 + k * ROWS < until ? heads[(k0 + k * ROWS) * W + c] : Real(0);
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) s += v[k];
      }
    }
    sums[row][col] = s;
    __syncthreads();
    if (row == 0 && c < W) {
      Real t = Real(0);
#pragma unroll
      for (int r = 0; r < ROWS; ++r) t += sums[r][col];
      table[int64_t(token) * W + c] = T(t * scale);
    }
    __syncthreads();
  }
}

struct GradientPlan {
  SortPlan sort;
  int L, columns;
  int64_t share, workers;
  int64_t partial_bytes, bytes;
};

// Sums: lanes enough for a row (256 at most), and shares that give the card about two waves a
// SIMD, of 16 positions or more.  Eight rows of a lane are in flight at a time, and
// every further share is one more end to join: 200 000 x 128 fp32 by 8 tokens, sums
// and join 26 + 16 us; 43 + 9 by one wave a SIMD.
GradientPlan gradient_plan(int64_t N, int64_t vocabulary, int64_t width, int size) {
  GradientPlan p{};
  p.sort = sort_plan(N, vocabulary);
  const int V = 16 / size;
  const int64_t chunks = (width + V - 1) / V;
  p.L = 4;
  while (p.L < kThreads && p.L < chunks) p.L *= 2;
  p.columns = int((chunks + p.L - 1) / p.L);
  const int64_t most = int64_t(256) * 4 * 2 * 64 / p.L;
  p.share = (N + most - 1) / most;
  if (p.share < 16) p.share = 16;
  p.workers = (N + p.share - 1) / p.share;
  auto up = [](int64_t b) { return (b + 255) / 256 * 256; };
  p.partial_bytes = up(p.workers * width * (size == 8 ? 8 : 4));
  p.bytes = p.sort.bytes + 2 * p.partial_bytes + up(p.workers * 8 + 1);
  return p;
}

template <typename T, typename Index>
int gradient_as(const T* adjoint, const Index* tokens, int64_t N, int64_t vocabulary, int64_t width, double scale,
                T* table, char* work, hipStream_t s) {
  typedef typename Wide<T>::type Real;
  const GradientPlan p = gradient_plan(N, vocabulary, width, int(sizeof(T)));
  Real* heads = reinterpret_cast<Real*>(work + p.sort.bytes);
  Real* tails = reinterpret_cast<Real*>(work + p.sort.bytes + p.partial_bytes);
  uint32_t* ends = reinterpret_cast<uint32_t*>(work + p.sort.bytes + 2 * p.partial_bytes);
  Pair* sorted = nullptr;
  if (int rc = sort_tokens(p.sort, tokens, N, vocabulary, work, &sorted, s)) return rc;
  const int W = int(width);
  const auto sum = p.L == 4     ? embedding_sum_kernel<T, 4>
                   : p.L == 8   ? embedding_sum_kernel<T, 8>
                   : p.L == 16  ? embedding_sum_kernel<T, 16>
                   : p.L == 32  ? embedding_sum_kernel<T, 32>
                   : p.L == 64  ? embedding_sum_kernel<T, 64>
                   : p.L == 128 ? embedding_sum_kernel<T, 128>
                                : embedding_sum_kernel<T, 256>;
  const int64_t per = kThreads / p.L, clearing = (vocabulary + 63) / 64;
  if (!fits_grid((p.workers + per - 1) / per + clearing, kThreads))
    return set_error(YE3T_EUNSUPPORTED, "a table of %lld rows is too large for one launch", (long long)vocabulary);
  hipLaunchKernelGGL(sum, dim3(unsigned((p.workers + per - 1) / per + clearing), unsigned(p.columns)), dim3(kThreads),
                     0, s, sorted, N, p.share, p.workers, adjoint, vocabulary, W, Real(scale), clearing, table, heads,
                     tails, ends);
  if (int rc = check_launch("embedding_sum_kernel")) return rc;
  if (p.workers < 2) return YE3T_OK;
  const int64_t columns = (width + kJoinColumns - 1) / kJoinColumns;
  hipLaunchKernelGGL((embedding_join_kernel<T>), dim3(unsigned(p.workers), unsigned(columns < kJoinGroups ? columns : kJoinGroups)),
                     dim3(kThreads), 0, s, ends, p.workers,
                     heads, tails, vocabulary, W, Real(scale), table);
  return check_launch("embedding_join_kernel");
}

template <typename T, typename Index>
int forward_as(const Index* tokens, int64_t N, const T* table, int64_t stride, int64_t vocabulary, int64_t width,
               double scale, T* out, hipStream_t s) {
  const int64_t chunks = (width + kChunk<T> - 1) / kChunk<T>;
  int64_t groups = (N * chunks + 4 * kThreads - 1) / (4 * kThreads);
  if (groups > (1 << 20)) groups = 1 << 20;
  hipLaunchKernelGGL((embedding_kernel<T, Index>), dim3(unsigned(groups)), dim3(kThreads), 0, s, tokens, N, table,
                     stride, vocabulary, int(width), int(chunks), typename Wide<T>::type(scale), out);
  return check_launch("embedding_kernel");
}

int check_embedding(int dtype, int token_bytes, int64_t N, int64_t vocabulary, int64_t width) {
  YE3T_REQUIRE(N >= 0 && vocabulary >= 0 && width >= 1, "token, row and column counts must not be negative");
  YE3T_REQUIRE(token_bytes == 4 || token_bytes == 8, "tokens must be int32 or int64");
  YE3T_REQUIRE(width <= (1 << 24), "rows of more than 2^24 values are not supported");
  YE3T_REQUIRE(N < (int64_t(1) << 31) && vocabulary < (int64_t(1) << 31), "at most 2^31 - 1 tokens and rows");
  if (dtype != YE3T_F32 && dtype != YE3T_F64 && dtype != YE3T_BF16)
    return set_error(YE3T_EDTYPE, "unsupported dtype %d; expected float32, float64 or bfloat16", dtype);
  return YE3T_OK;
}

inline int size_of(int dtype) { return dtype == YE3T_F64 ? 8 : dtype == YE3T_F32 ? 4 : 2; }

// calls f with a null pointer of the storage type
template <typename F>
int with_type(int dtype, F f) {
  if (dtype == YE3T_F64) return f(static_cast<double*>(nullptr));
  if (dtype == YE3T_F32) return f(static_cast<float*>(nullptr));
  return f(static_cast<__bf16*>(nullptr));
}

}  // namespace
}  // namespace ye3t

using namespace ye3t;

extern "C" {

int ye3t_hip_embedding(int dtype, const void* tokens, int token_bytes, int64_t token_count, const void* table,
                       int64_t row_stride, int64_t vocabulary, int64_t width, double scale, void* out,
                       ye3t_stream_t stream) {
  clear_error();
  if (int rc = check_embedding(dtype, token_bytes, token_count, vocabulary, width)) return rc;
  if (token_count == 0) return YE3T_OK;
  YE3T_REQUIRE(tokens && out && (table || vocabulary == 0), "the embedding needs tokens, a table and an output");
  YE3T_REQUIRE(row_stride >= 0, "row_stride must not be negative");
  const hipStream_t s = as_stream(stream);
  return with_type(dtype, [&](auto* type) {
    typedef std::remove_pointer_t<decltype(type)> T;
    const T* t = static_cast<const T*>(table);
    return token_bytes == 4 ? forward_as(static_cast<const int32_t*>(tokens), token_count, t, row_stride, vocabulary,
                                         width, scale, static_cast<T*>(out), s)
                            : forward_as(static_cast<const int64_t*>(tokens), token_count, t, row_stride, vocabulary,
                                         width, scale, static_cast<T*>(out), s);
  });
}

int64_t ye3t_hip_embedding_adjoint_workspace_bytes(int dtype, int64_t token_count, int64_t vocabulary, int64_t width) {
  clear_error();
  if (check_embedding(dtype, 4, token_count, vocabulary, width)) return -1;
  return gradient_plan(token_count, vocabulary, width, size_of(dtype)).bytes;
}

int ye3t_hip_embedding_adjoint(int dtype, const void* adjoint, const void* tokens, int token_bytes, int64_t token_count,
                               int64_t vocabulary, int64_t width, double scale, void* table_adjoint, void* workspace,
                               int64_t workspace_bytes, ye3t_stream_t stream) {
  clear_error();
  if (int rc = check_embedding(dtype, token_bytes, token_count, vocabulary, width)) return rc;
  if (vocabulary == 0) return YE3T_OK;
  YE3T_REQUIRE(table_adjoint && (token_count == 0 || (adjoint && tokens)),
               "the gradient needs the rows' adjoint, the tokens and an output");
  YE3T_REQUIRE(workspace && workspace_bytes >= gradient_plan(token_count, vocabulary, width, size_of(dtype)).bytes,
               "the workspace is smaller than ye3t_hip_embedding_adjoint_workspace_bytes");
  const hipStream_t s = as_stream(stream);
  return with_type(dtype, [&](auto* type) {
    typedef std::remove_pointer_t<decltype(type)> T;
    const T* g = static_cast<const T*>(adjoint);
    T* to = static_cast<T*>(table_adjoint);
    char* work = static_cast<char*>(workspace);
    return token_bytes == 4
               ? gradient_as(g, static_cast<const int32_t*>(tokens), token_count, vocabulary, width, scale, to, work, s)
               : gradient_as(g, static_cast<const int64_t*>(tokens), token_count, vocabulary, width, scale, to, work, s);
  });
}

}  // extern "C"
